// fc_Q4A, attention_rope2 and the ops of several requests as the Python module calls them, in native code: the argument checks, the
// output and the call of the C entry.  A small call is shorter than the Python around it (one row of a 4096 x 4096 product: 5.4 us on the
// device, 10.9 us per call through ctypes and 5.2 us so; one token of attention over 2048 rows of halves 21.2 and 14.1).
//
// These are shortcuts for the ordinary case and decide nothing: whatever is not ordinary -- a tensor subclass, vmap, a mode
// that intercepts calls, a stream under capture, a workspace that is missing or too small, any argument that a check
// would refuse -- returns NotImplemented with nothing done, and the Python function takes the call, workspace policy and
// error messages included.  (torch.jit.trace does not stop them: neither way can it record more than the output's
// allocation.)  Nothing is kept between calls but the addresses of the C entries.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/llmops_hip.h"

namespace {

decltype(&llmops_fc_Q4A_workspace_bytes) fc_workspace_bytes;
decltype(&llmops_fc_Q4A) fc;
decltype(&llmops_attention_workspace_bytes) attention_workspace_bytes;
decltype(&llmops_attention_rope) attention;
decltype(&llmops_last_error) last_error;
decltype(&llmops_attention_prefix_workspace_bytes) prefix_workspace_bytes;
decltype(&llmops_attention_rope_prefix) attention_prefix;
decltype(&llmops_lora_workspace_bytes) lora_workspace_bytes;
decltype(&llmops_lora_add) lora;
decltype(&llmops_verify_drafts_workspace_bytes) verify_workspace_bytes;
decltype(&llmops_verify_drafts) verify;
decltype(&llmops_cache_write_q4) write_q4;
decltype(&llmops_cache_read_q4) read_q4;
decltype(&llmops_attention_q4_workspace_bytes) q4_workspace_bytes;
decltype(&llmops_attention_rope_q4) attention_q4;
decltype(&llmops_token_logprobs_workspace_bytes) logprobs_workspace_bytes;
decltype(&llmops_token_logprobs) logprobs;

// a plain tensor with memory of its own on the HIP device
bool plain_strided(PyObject* o, at::ScalarType type, int64_t dims) {
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet kWrapped({K::Python, K::PythonTLSSnapshot, K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Batched,
                                            K::Functionalize, K::Conjugate, K::Negative, K::ZeroTensor});
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == type && t.dim() == dims &&
           !t.key_set().has_any(kWrapped) && t.has_storage();
}
// .. and dense
bool plain(PyObject* o, at::ScalarType type, int64_t dims) { return plain_strided(o, type, dims) && THPVariable_Unpack(o).is_contiguous(); }
// fp32 [B, L, C], dense in C
bool plain_rows(PyObject* o) {
    if (!plain_strided(o, at::kFloat, 3)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.stride(2) == 1 && t.numel() > 0;
}
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
// all on the current device
bool all_here(std::initializer_list<PyObject*> all) {
    const int here = c10::hip::current_device();
    for (PyObject* o : all)
        if (o != Py_None && THPVariable_Unpack(o).get_device() != here) return false;
    return true;
}
at::Tensor scratch(const at::Tensor& like, size_t bytes) { return at::empty({(int64_t)(bytes > 0 ? bytes : 1)}, like.options().dtype(at::kByte).requires_grad(false)); }
void* address(PyObject* o) { return o == Py_None ? nullptr : THPVariable_Unpack(o).data_ptr(); }
bool whole(PyObject* o, int64_t& v) {
    int over = 0;
    if (!PyLong_CheckExact(o)) return false;
    v = PyLong_AsLongLongAndOverflow(o, &over);
    return over == 0;
}

// nothing between this call and the device: no Python mode, no functorch level, no capture on the stream
bool direct() {
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet kModes({K::Python, K::PythonTLSSnapshot, K::FuncTorchDynamicLayerFrontMode, K::FuncTorchDynamicLayerBackMode,
                                          K::FuncTorchVmapMode, K::Batched, K::Functionalize});
    return !at::impl::torch_function_mode_enabled() && !c10::impl::tls_local_dispatch_key_set().included_.has_any(kModes) &&
           c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None;
}

// the module's workspace of this family on this device and stream, undefined if there is none of `bytes`
at::Tensor workspace(PyObject* held, const char* kind, const at::Tensor& t, hipStream_t stream, size_t bytes) {
    PyObject* key = Py_BuildValue("(ssiK)", kind, "cuda", (int)t.get_device(), (unsigned long long)(uintptr_t)stream);
    if (key == nullptr) {
        PyErr_Clear();
        return {};
    }
    PyObject* ws = PyDict_Check(held) ? PyDict_GetItem(held, key) : nullptr;  // (borrowed)
    Py_DECREF(key);
    if (ws == nullptr || !THPVariable_CheckExact(ws)) return {};
    const at::Tensor& w = THPVariable_Unpack(ws);
    return (size_t)w.numel() >= bytes ? w : at::Tensor();
}

hipStream_t current_stream(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

PyObject* refused() {
    const char* what = last_error();
    PyErr_SetString(PyExc_RuntimeError, what);
    return nullptr;
}

PyObject* not_ordinary() { Py_RETURN_NOTIMPLEMENTED; }

// fc_Q4A(workspaces, input, weiq, N)
PyObject* call_fc(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !PyLong_CheckExact(args[3]) || !plain(args[1], at::kFloat, 3) || !plain(args[2], at::kChar, 3) || !direct())
        return not_ordinary();
    const at::Tensor &x = THPVariable_Unpack(args[1]), &w = THPVariable_Unpack(args[2]);
    int overflow = 0;
    const int64_t N = PyLong_AsLongLongAndOverflow(args[3], &overflow);
    const int64_t B = x.size(0), M = x.size(1), K = x.size(2), Ng = w.size(0), Kg = w.size(1), blk = w.size(2);
    const int g = blk == 640 ? 32 : blk == 2176 ? 128 : 0;
    if (overflow || g == 0 || N <= 0 || B <= 0 || M <= 0 || K <= 0) return not_ordinary();
    const hipStream_t st = current_stream(x);
    const at::Tensor ws = workspace(args[0], "fc", x, st, fc_workspace_bytes(B * M, K, Ng, Kg, g));
    if (!ws.defined()) return not_ordinary();
    at::Tensor y = at::empty({B, M, N}, x.options().requires_grad(false));
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;  // (a launch can wait for room in the queue)
        rc = fc(static_cast<const float*>(x.data_ptr()), B * M, K, static_cast<const int8_t*>(w.data_ptr()), Ng, Kg, g, N,
                static_cast<float*>(y.data_ptr()), ws.data_ptr(), (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// attention_rope2(workspaces, q, k, v, inv_freq, kv_cache, kvc_slots, position_id, layer_id)
PyObject* call_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9 || !plain(args[1], at::kFloat, 3) || !plain(args[2], at::kFloat, 3) || !plain(args[3], at::kFloat, 3) ||
        !plain(args[4], at::kFloat, 1) || !(plain(args[5], at::kFloat, 5) || plain(args[5], at::kHalf, 5)) || !plain(args[6], at::kInt, 1) ||
        !PyLong_CheckExact(args[7]) || !PyLong_CheckExact(args[8]) || !direct())
        return not_ordinary();
    const at::Tensor &q = THPVariable_Unpack(args[1]), &k = THPVariable_Unpack(args[2]), &v = THPVariable_Unpack(args[3]),
                     &f = THPVariable_Unpack(args[4]), &c = THPVariable_Unpack(args[5]), &slots = THPVariable_Unpack(args[6]);
    const int64_t B = q.size(0), qL = q.size(1), planes = c.size(0), H = c.size(2), maxlen = c.size(3), S = c.size(4);
    int over[2] = {0, 0};
    const long position = PyLong_AsLongAndOverflow(args[7], &over[0]), layer = PyLong_AsLongAndOverflow(args[8], &over[1]);
    if (over[0] || over[1] || position != (int)position || layer != (int)layer || c.size(1) != B || B <= 0 || qL <= 0 || q.size(2) != H * S ||
        k.sizes() != q.sizes() || v.sizes() != q.sizes() || slots.size(0) != qL)
        return not_ordinary();
    const hipStream_t st = current_stream(q);
    const at::Tensor ws = workspace(args[0], "attn", q, st, attention_workspace_bytes(B, qL, H, S, maxlen));
    if (!ws.defined()) return not_ordinary();
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = attention(static_cast<float*>(q.data_ptr()), static_cast<float*>(k.data_ptr()), static_cast<const float*>(v.data_ptr()), B, qL, H, S,
                       static_cast<const float*>(f.data_ptr()), f.size(0), c.data_ptr(), c.scalar_type() == at::kFloat ? 0 : 1, planes, maxlen,
                       static_cast<const int32_t*>(slots.data_ptr()), (int)position, (int)layer, ws.data_ptr(), (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// attention_rope_prefix(q, k, v, inv_freq, prefix_cache, prefix_len, kv_cache, lengths, layer_id, q_lens)
PyObject* call_attention_prefix(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t prefix_len = 0, layer = 0;
    if (n != 10 || !plain_rows(args[0]) || !plain_rows(args[1]) || !plain_rows(args[2]) || !plain(args[3], at::kFloat, 1) ||
        !whole(args[5], prefix_len) || !(plain(args[6], at::kFloat, 5) || plain(args[6], at::kHalf, 5)) || !plain(args[7], at::kInt, 1) || !whole(args[8], layer) ||
        !(args[9] == Py_None || plain(args[9], at::kInt, 1)) || !direct())
        return not_ordinary();
    const at::Tensor &q = THPVariable_Unpack(args[0]), &k = THPVariable_Unpack(args[1]), &v = THPVariable_Unpack(args[2]), &f = THPVariable_Unpack(args[3]),
                     &c = THPVariable_Unpack(args[6]), &len = THPVariable_Unpack(args[7]);
    const bool prefixed = args[4] != Py_None;
    if (prefixed && !plain(args[4], c.scalar_type(), 5)) return not_ordinary();
    if (!all_here({args[0], args[1], args[2], args[3], args[4], args[6], args[7], args[9]})) return not_ordinary();
    const int64_t B = q.size(0), qL = q.size(1), planes = c.size(0), Hkv = c.size(2), maxlen = c.size(3), S = c.size(4);
    int64_t pplanes = 0, pmax = 0;
    if (prefixed) {
        const at::Tensor& p = THPVariable_Unpack(args[4]);
        if (p.size(1) != 1 || p.size(2) != Hkv || p.size(4) != S) return not_ordinary();
        pplanes = p.size(0), pmax = p.size(3);
    }
    if (S <= 0 || Hkv <= 0 || q.size(2) % S != 0 || c.size(1) != B || len.size(0) != B || k.size(0) != B || k.size(1) != qL || k.size(2) != Hkv * S ||
        k.sizes() != v.sizes() || layer != (int)layer || prefix_len < 0 || prefix_len > pmax || (args[9] != Py_None && THPVariable_Unpack(args[9]).size(0) != B))
        return not_ordinary();
    const int64_t H = q.size(2) / S;
    const hipStream_t st = current_stream(q);
    at::Tensor out = at::empty({B, qL, H * S}, q.options().requires_grad(false));
    const size_t bytes = prefix_workspace_bytes(B, qL, H, Hkv, S, prefix_len, maxlen);
    const at::Tensor ws = scratch(q, bytes);
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = attention_prefix(static_cast<const float*>(q.data_ptr()), stride_of(q, 0), stride_of(q, 1), static_cast<const float*>(k.data_ptr()), stride_of(k, 0),
                              stride_of(k, 1), static_cast<const float*>(v.data_ptr()), stride_of(v, 0), stride_of(v, 1), B, qL, H, Hkv, S,
                              static_cast<const float*>(f.data_ptr()), f.size(0), address(args[4]), pplanes, pmax, prefix_len, c.data_ptr(),
                              c.scalar_type() == at::kFloat ? 0 : 1, planes, maxlen, static_cast<const int32_t*>(len.data_ptr()),
                              static_cast<const int32_t*>(address(args[9])), (int)layer, static_cast<float*>(out.data_ptr()), ws.data_ptr(), (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// lora_add(y, x, lora_A, lora_B, adapters, scales), the result in a new tensor
PyObject* call_lora(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !plain_rows(args[0]) || !plain_rows(args[1]) || !THPVariable_CheckExact(args[2]) || !plain(args[4], at::kInt, 1) ||
        !plain(args[5], at::kFloat, 1) || !direct())
        return not_ordinary();
    const at::ScalarType type = THPVariable_Unpack(args[2]).scalar_type();
    const int dtype = type == at::kFloat ? LLMOPS_F32 : type == at::kHalf ? LLMOPS_F16 : type == at::kBFloat16 ? LLMOPS_BF16 : -1;
    if (dtype < 0 || !plain(args[2], type, 3) || !plain(args[3], type, 3) || !all_here({args[0], args[1], args[2], args[3], args[4], args[5]})) return not_ordinary();
    const at::Tensor &y = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[1]), &A = THPVariable_Unpack(args[2]), &W = THPVariable_Unpack(args[3]),
                     &ids = THPVariable_Unpack(args[4]), &scales = THPVariable_Unpack(args[5]);
    const int64_t B = y.size(0), M = y.size(1), N = y.size(2), K = x.size(2), count = A.size(0), R = A.size(1);
    if (x.size(0) != B || x.size(1) != M || A.size(2) != K || W.size(0) != count || W.size(1) != N || W.size(2) != R || ids.size(0) != B || scales.size(0) != count)
        return not_ordinary();
    const hipStream_t st = current_stream(y);
    at::Tensor out = at::empty({B, M, N}, y.options().requires_grad(false));
    const size_t bytes = lora_workspace_bytes(B, M, N, K, R, count);
    const at::Tensor ws = scratch(y, bytes);
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = lora(static_cast<const float*>(y.data_ptr()), stride_of(y, 0), stride_of(y, 1), static_cast<const float*>(x.data_ptr()), stride_of(x, 0),
                  stride_of(x, 1), B, M, N, K, A.data_ptr(), W.data_ptr(), dtype, R, count, static_cast<const int32_t*>(ids.data_ptr()),
                  static_cast<const float*>(scales.data_ptr()), static_cast<float*>(out.data_ptr()), M * N, N, ws.data_ptr(), (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// verify_drafts(logits, drafts, uniforms, draft_probs, temperature, draft_lens) with drafts int64
PyObject* call_verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !plain(args[0], at::kFloat, 3) || !plain(args[1], at::kLong, 2) || !plain(args[2], at::kFloat, 2) ||
        !(args[3] == Py_None || plain(args[3], at::kFloat, 3)) || !(args[5] == Py_None || plain(args[5], at::kInt, 1)) || !direct())
        return not_ordinary();
    float one = 1.0f;
    const bool rows_have = THPVariable_Check(args[4]);
    if (rows_have ? !plain(args[4], at::kFloat, 1) : !(args[4] == Py_None || PyFloat_CheckExact(args[4]))) return not_ordinary();
    if (PyFloat_CheckExact(args[4])) one = (float)PyFloat_AS_DOUBLE(args[4]);
    if (!all_here({args[0], args[1], args[2], args[3], rows_have ? args[4] : Py_None, args[5]})) return not_ordinary();
    const at::Tensor &z = THPVariable_Unpack(args[0]), &d = THPVariable_Unpack(args[1]), &u = THPVariable_Unpack(args[2]);
    const int64_t B = z.size(0), K = z.size(1) - 1, V = z.size(2);
    if (B <= 0 || K < 0 || V <= 0 || d.size(0) != B || d.size(1) != K || u.size(0) != B || u.size(1) != K + 1) return not_ordinary();
    if (args[3] != Py_None) {
        const at::Tensor& p = THPVariable_Unpack(args[3]);
        if (p.size(0) != B || p.size(1) != K || p.size(2) != V) return not_ordinary();
    }
    if ((rows_have && THPVariable_Unpack(args[4]).size(0) != B) || (args[5] != Py_None && THPVariable_Unpack(args[5]).size(0) != B)) return not_ordinary();
    const hipStream_t st = current_stream(z);
    at::Tensor tokens = at::empty({B, K + 1}, d.options().requires_grad(false)), accepted = at::empty({B}, d.options().dtype(at::kInt).requires_grad(false));
    const size_t bytes = verify_workspace_bytes(B, K, V);
    const at::Tensor ws = scratch(z, bytes);
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = verify(static_cast<const float*>(z.data_ptr()), B, K, V, K > 0 ? static_cast<const int64_t*>(d.data_ptr()) : nullptr,
                    K > 0 ? static_cast<const float*>(address(args[3])) : nullptr, static_cast<const float*>(u.data_ptr()),
                    rows_have ? static_cast<const float*>(address(args[4])) : nullptr, one, static_cast<const int32_t*>(address(args[5])),
                    static_cast<int64_t*>(tokens.data_ptr()), static_cast<int32_t*>(accepted.data_ptr()), ws.data_ptr(), (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    PyObject* first = THPVariable_Wrap(std::move(tokens));
    PyObject* second = THPVariable_Wrap(std::move(accepted));
    PyObject* both = first != nullptr && second != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
    END_HANDLE_TH_ERRORS
}

// int8 [planes, B, Hkv, maxlen, LLMOPS_Q4_ROW_BYTES]
bool q4_cache(PyObject* o) { return plain(o, at::kChar, 5) && THPVariable_Unpack(o).size(4) == LLMOPS_Q4_ROW_BYTES && THPVariable_Unpack(o).numel() > 0; }
bool counts(PyObject* o, int64_t B) { return plain(o, at::kInt, 1) && THPVariable_Unpack(o).size(0) == B; }

// cache_write_q4(k, v, kv_cache, lengths, layer_id, inv_freq, q_lens)
PyObject* call_write_q4(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t layer = 0;
    if (n != 7 || !THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1]) || !q4_cache(args[2]) || !whole(args[4], layer) ||
        !(args[5] == Py_None || (plain(args[5], at::kFloat, 1) && THPVariable_Unpack(args[5]).numel() > 0)) || !direct())
        return not_ordinary();
    const at::Tensor &c = THPVariable_Unpack(args[2]), &first = THPVariable_Unpack(args[0]);
    const int64_t B = c.size(1), Hkv = c.size(2), S = 128;
    const at::ScalarType type = first.scalar_type();
    if ((type != at::kFloat && type != at::kHalf) || layer != (int)layer || !counts(args[3], B) || !(args[6] == Py_None || counts(args[6], B)) || first.dim() < 3)
        return not_ordinary();
    const int64_t L = first.size(1);
    int64_t at[2][3];
    for (int i = 0; i < 2; i++) {
        const int64_t dims = THPVariable_Unpack(args[i]).dim();
        if ((dims != 3 && dims != 4) || !plain_strided(args[i], type, dims)) return not_ordinary();
        const at::Tensor& t = THPVariable_Unpack(args[i]);
        if (t.size(0) != B || t.size(1) != L || L <= 0 || t.stride(-1) != 1 || (dims == 3 ? t.size(2) != Hkv * S : t.size(2) != Hkv || t.size(3) != S)) return not_ordinary();
        at[i][0] = stride_of(t, 0), at[i][1] = stride_of(t, 1), at[i][2] = dims == 3 ? S : stride_of(t, 2);
    }
    if (!all_here({args[0], args[1], args[2], args[3], args[5], args[6]})) return not_ordinary();
    const hipStream_t st = current_stream(c);
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = write_q4(first.data_ptr(), at[0][0], at[0][1], at[0][2], THPVariable_Unpack(args[1]).data_ptr(), at[1][0], at[1][1], at[1][2],
                      type == at::kFloat ? LLMOPS_F32 : LLMOPS_F16, B, L, Hkv, S, static_cast<const float*>(address(args[5])),
                      args[5] == Py_None ? 0 : THPVariable_Unpack(args[5]).size(0), c.data_ptr(), c.size(0), c.size(3),
                      static_cast<const int32_t*>(address(args[3])), static_cast<const int32_t*>(address(args[6])), (int)layer, st);
    }
    if (rc != 0) return refused();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// cache_read_q4(kv_cache, rows, starts, whether to fp32)
PyObject* call_read_q4(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t rows = 0;
    if (n != 4 || !q4_cache(args[0]) || !whole(args[1], rows) || rows <= 0 || !PyBool_Check(args[3]) || !direct()) return not_ordinary();
    const at::Tensor& c = THPVariable_Unpack(args[0]);
    if (!(args[2] == Py_None || counts(args[2], c.size(1))) || !all_here({args[0], args[2]})) return not_ordinary();
    const bool full = args[3] == Py_True;
    const hipStream_t st = current_stream(c);
    at::Tensor out = at::empty({c.size(0), c.size(1), c.size(2), rows, 128}, c.options().dtype(full ? at::kFloat : at::kHalf).requires_grad(false));
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = read_q4(c.data_ptr(), c.size(0), c.size(1), c.size(2), c.size(3), 128, static_cast<const int32_t*>(address(args[2])), rows, out.data_ptr(),
                     full ? LLMOPS_F32 : LLMOPS_F16, st);
    }
    if (rc != 0) return refused();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// attention_rope_q4(q, k, v, inv_freq, kv_cache, lengths, layer_id, q_lens)
PyObject* call_attention_q4(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t layer = 0;
    if (n != 8 || !plain_rows(args[0]) || !plain_rows(args[1]) || !plain_rows(args[2]) || !plain(args[3], at::kFloat, 1) || !q4_cache(args[4]) ||
        !whole(args[6], layer) || !direct())
        return not_ordinary();
    const at::Tensor &q = THPVariable_Unpack(args[0]), &k = THPVariable_Unpack(args[1]), &v = THPVariable_Unpack(args[2]), &f = THPVariable_Unpack(args[3]),
                     &c = THPVariable_Unpack(args[4]);
    const int64_t B = c.size(1), qL = q.size(1), planes = c.size(0), Hkv = c.size(2), maxlen = c.size(3), S = 128;
    if (q.size(0) != B || q.size(2) % S != 0 || k.size(0) != B || k.size(1) != qL || k.size(2) != Hkv * S || k.sizes() != v.sizes() || layer != (int)layer ||
        !counts(args[5], B) || !(args[7] == Py_None || counts(args[7], B)) || !all_here({args[0], args[1], args[2], args[3], args[4], args[5], args[7]}))
        return not_ordinary();
    const int64_t H = q.size(2) / S;
    const hipStream_t st = current_stream(q);
    at::Tensor out = at::empty({B, qL, H * S}, q.options().requires_grad(false));
    const at::Tensor ws = scratch(q, q4_workspace_bytes(B, qL, H, Hkv, S, maxlen));
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = attention_q4(static_cast<const float*>(q.data_ptr()), stride_of(q, 0), stride_of(q, 1), static_cast<const float*>(k.data_ptr()), stride_of(k, 0),
                          stride_of(k, 1), static_cast<const float*>(v.data_ptr()), stride_of(v, 0), stride_of(v, 1), B, qL, H, Hkv, S,
                          static_cast<const float*>(f.data_ptr()), f.size(0), c.data_ptr(), planes, maxlen, static_cast<const int32_t*>(address(args[5])),
                          static_cast<const int32_t*>(address(args[7])), (int)layer, static_cast<float*>(out.data_ptr()), ws.data_ptr(), (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// token_logprobs(logits, tokens, top) with tokens int64
PyObject* call_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int64_t top = 0;
    if (n != 3 || !plain_rows(args[0]) || !plain_strided(args[1], at::kLong, 2) || !whole(args[2], top) || top < 0 || top > 64 || !direct()) return not_ordinary();
    const at::Tensor &z = THPVariable_Unpack(args[0]), &t = THPVariable_Unpack(args[1]);
    const int64_t B = z.size(0), L = z.size(1), V = z.size(2);
    if (t.size(0) != B || t.size(1) != L || !all_here({args[0], args[1]})) return not_ordinary();
    const hipStream_t st = current_stream(z);
    const auto real = z.options().requires_grad(false);
    at::Tensor out[4] = {at::empty({B, L}, real), at::empty({B, L}, real), at::empty({B, L, top}, real.dtype(at::kLong)), at::empty({B, L, top}, real)};
    const at::Tensor ws = scratch(z, logprobs_workspace_bytes(B, L, V, top));
    int rc = 0;
    {
        pybind11::gil_scoped_release others_run;
        rc = logprobs(static_cast<const float*>(z.data_ptr()), stride_of(z, 0), stride_of(z, 1), B, L, V, static_cast<const int64_t*>(t.data_ptr()), stride_of(t, 0),
                      stride_of(t, 1), top, static_cast<float*>(out[0].data_ptr()), static_cast<float*>(out[1].data_ptr()),
                      top > 0 ? static_cast<int64_t*>(out[2].data_ptr()) : nullptr, top > 0 ? static_cast<float*>(out[3].data_ptr()) : nullptr, ws.data_ptr(),
                      (size_t)ws.numel(), st);
    }
    if (rc != 0) return refused();
    PyObject* all = PyTuple_New(4);
    for (int i = 0; all != nullptr && i < 4; i++) {
        PyObject* one = THPVariable_Wrap(std::move(out[i]));
        if (one == nullptr) {
            Py_DECREF(all);
            return nullptr;
        }
        PyTuple_SET_ITEM(all, i, one);
    }
    return all;
    END_HANDLE_TH_ERRORS
}

// bind(addresses of the C entries, in the order of the variables above)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[17];
    if (PyTuple_GET_SIZE(args) != 17) {
        PyErr_SetString(PyExc_TypeError, "bind: the addresses of 17 entries");
        return nullptr;
    }
    for (int j = 0; j < 17; j++) {
        a[j] = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(args, j));
        if (PyErr_Occurred()) return nullptr;
    }
    int i = 0;
    auto take = [&](auto& entry) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>((uintptr_t)a[i++]); };
    take(fc_workspace_bytes), take(fc), take(attention_workspace_bytes), take(attention), take(last_error);
    take(prefix_workspace_bytes), take(attention_prefix), take(lora_workspace_bytes), take(lora), take(verify_workspace_bytes), take(verify);
    take(write_q4), take(read_q4), take(q4_workspace_bytes), take(attention_q4), take(logprobs_workspace_bytes), take(logprobs);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"fc_Q4A", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_fc)), METH_FASTCALL, nullptr},
                         {"attention_rope2", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_attention)), METH_FASTCALL, nullptr},
                         {"attention_rope_prefix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_attention_prefix)), METH_FASTCALL, nullptr},
                         {"lora_add", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_lora)), METH_FASTCALL, nullptr},
                         {"verify_drafts", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_verify)), METH_FASTCALL, nullptr},
                         {"cache_write_q4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_write_q4)), METH_FASTCALL, nullptr},
                         {"cache_read_q4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_read_q4)), METH_FASTCALL, nullptr},
                         {"attention_rope_q4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_attention_q4)), METH_FASTCALL, nullptr},
                         {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_logprobs)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    PyObject* m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddStringConstant(m, "built_for", LLMOPS_BUILT_FOR) != 0) {  // (compared before anything is called)
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
