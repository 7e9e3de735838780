"""csrc/extents.h (do rows of one tensor lie over rows of another?) against a look at every byte."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("extents")
    (d / "x.cc").write_text('''#include "extents.h"
using namespace llmops;
static Extent of(const int64_t* a) { return Extent(reinterpret_cast<const void*>(a[0]), a[1], a[2], a[3], a[4], a[5]); }
extern "C" int two(const int64_t* a, const int64_t* b) { return apart(of(a), of(b)); }
extern "C" int one(const int64_t* a) { return rows_apart(of(a)); }
extern "C" int nested(const int64_t* a) { return of(a).nested(); }
''')
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "llama.cl_amd", "csrc"), "-o", str(d / "x.so"), str(d / "x.cc")],
                   check=True)
    return ctypes.CDLL(str(d / "x.so"))


def _rows(a):
    base, n0, s0, n1, s1, width = a
    return [range(base + i * s0 + j * s1, base + i * s0 + j * s1 + width) for i in range(n0) for j in range(n1)]


def _arg(a):
    return (ctypes.c_int64 * 6)(*a)


def _draw(rng, negative):
    step = lambda: rng.choice([0, rng.randint(0, 12), rng.randint(0, 60)]) * (rng.choice([1, 1, -1]) if negative else 1)  # noqa: E731
    return [rng.randint(1000, 1100), rng.randint(1, 4), step(), rng.randint(1, 4), step(), rng.randint(1, 12)]


@pytest.mark.parametrize("negative", [False, True])
def test_against_every_byte(lib, negative):
    rng = random.Random(1)
    seen = {}
    for _ in range(20000):
        a, b = _draw(rng, negative), _draw(rng, negative)
        rows = _rows(a)
        alone = sum(map(len, rows)) == len(set().union(*rows))
        assert lib.one(_arg(a)) == alone, a
        bytes_a, bytes_b = set().union(*rows), set().union(*_rows(b))
        far = max(bytes_a) < min(bytes_b) or max(bytes_b) < min(bytes_a)
        want = not (bytes_a & bytes_b)
        got = lib.two(_arg(a), _arg(b))
        if lib.nested(_arg(a)) or far:
            assert got == want, (a, b)
        else:
            assert not got
        seen[(alone, want, far)] = seen.get((alone, want, far), 0) + 1
    assert min(seen.get(k, 0) for k in ((True, True, False), (True, False, False), (True, True, True), (False, False, False))) > 20, seen


def test_strides_that_pass_64_bits(lib):
    far = (1 << 62) + 5
    assert lib.one(_arg([4096, 8, far, 8, far, 100])) == 0
    assert lib.one(_arg([4096, 8, far, 1 << 20, 128, 100])) == 1
    assert lib.two(_arg([4096, 2, far, 2, 200, 100]), _arg([4196, 2, far, 2, 200, 100])) == 1
    assert lib.two(_arg([4096, 2, far, 2, 200, 100]), _arg([4195, 2, far, 2, 200, 100])) == 0
