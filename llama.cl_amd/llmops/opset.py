"""Python-side wrappers the reference keeps next to its model code (the ``llmop_*`` classes and
``KVCache`` of /root/reference/chatllama/main.py:60-219), re-stated over device tensors.

``to_lt`` / ``to_torch`` are identities here because the tensor type at the boundary already is a
``torch.Tensor`` (the reference converts between torch, numpy and its own tensor class,
chatllama/main.py:136-144).
"""
import torch

import llmops


def to_lt(a):
    return a


def to_torch(a):
    return a


class KVCache:
    """Fixed-size ring-buffer KV cache with slot reuse (chatllama/main.py:60-134).

    ``cache`` is [2*layers, batch, heads, max_kv_len, head_size]; ``prepare`` assigns the cache rows
    ("slots") the next ``query_len`` tokens go to, skipping rows that hold the system prompt
    (mask -1) and refusing (returning False) when it would have to overwrite sentence
    ``fail_on_sid``.
    """

    def __init__(self, configs, batch_size, max_kv_len, verbose=False, device="cuda", dtype=torch.float32):
        self.cache = torch.zeros(configs["layer_num"] * 2, batch_size, configs["head_num"], max_kv_len,
                                 configs["head_size"], dtype=dtype, device=device)
        self.device = device
        self.mask = torch.zeros(max_kv_len, dtype=torch.int32)  # host-side bookkeeping
        self.max_kv_len = max_kv_len
        self.position_id_next = 0
        self.position_id = 0
        self.slots = torch.empty(0, dtype=torch.int32, device=device)
        self.cur_slot = 0
        self.cur_kv_len = 0
        self.verbose = verbose

    def size(self):
        return self.cache.numel() * self.cache.element_size()

    def prepare(self, query_len, sentence_id, fail_on_sid):
        assert query_len > 0
        cur_slot = self.cur_slot
        slots = []
        for _ in range(query_len):
            while self.mask[cur_slot] < 0:  # reserved for the system message
                cur_slot = (cur_slot + 1) % self.max_kv_len
            if self.mask[cur_slot] != 0 and self.mask[cur_slot] == fail_on_sid:
                return False
            slots.append(cur_slot)
            cur_slot = (cur_slot + 1) % self.max_kv_len
        self.cur_slot = cur_slot
        for s in slots:
            self.mask[s] = sentence_id
        self.slots = torch.tensor(slots, dtype=torch.int32, device=self.device)
        self.position_id = self.position_id_next
        self.position_id_next = self.position_id + query_len
        self.cur_kv_len = min(self.cur_kv_len + query_len, self.max_kv_len)
        return True


class llmop_fc_q4a:
    """Holds one packed weight and applies fc_Q4A (+ optional bias) -- chatllama/main.py:158-177."""

    def __init__(self, linear=None, weight=None, bias=None, group_k=None, packed=None, N=None):
        if linear is not None:
            weight, bias = linear.weight, linear.bias
        if packed is not None:
            self.weight, self.N = packed, N
        else:
            self.weight = llmops.offline_FC_quant_Q4A(weight.detach(), group_k)
            self.N = weight.shape[0]
        self.bias = bias.detach() if bias is not None else None

    def __call__(self, input, residual=None):
        out = llmops.fc_Q4A(input, self.weight, self.N, residual=residual)
        if self.bias is not None:
            llmops.iadd(out, self.bias)
        return out

    def weight_size(self):
        size = self.weight.numel() * self.weight.element_size()
        if self.bias is not None:
            size += self.bias.numel() * self.bias.element_size()
        return size

    def __repr__(self):
        return f"llmop_fc_q4a(weight: {list(self.weight.shape)})"


class llmop_rmsnorm:
    """chatllama/main.py:179-191"""

    def __init__(self, weight, variance_epsilon):
        self.weight = weight.detach().clone()
        self.eps = variance_epsilon

    def __call__(self, input):
        llmops.rmsnorm(input, self.weight, self.eps)

    def out_of_place(self, input):
        return llmops.rmsnorm_out(input, self.weight, self.eps)

    def __repr__(self):
        return f"llmop_rmsnorm(weight: {list(self.weight.shape)}, eps: {self.eps})"


class llmop_embedding_q8c:
    """chatllama/main.py:206-219"""

    def __init__(self, weight=None, packed=None):
        # packed = (int8 rows, fp32 per-row scales) as embedding_q8c_quant_w returns them
        self.weight, self.scales = packed if packed is not None else llmops.embedding_q8c_quant_w(weight.detach())

    def __call__(self, input_ids):
        output = llmops.empty(*input_ids.shape, self.weight.shape[1], device=input_ids.device)
        llmops.embedding_q8c(output, input_ids, self.weight, self.scales)
        return output

    def __repr__(self):
        return f"llmop_embedding_q8c(weight: {list(self.weight.shape)})"


class PrefixCache:
    """KV cache of a batch whose sequences share a prefix (a system prompt, a document): the prefix's rows once, behind them
    ``max_kv_len`` rows for each sequence (``llmops.attention_rope_prefix``).  The reference keeps the system prompt's rows in the one
    cache of its one chat (mask -1 of chatllama/main.py:60-134); here many chats have them in common.

    ``prefix`` is a cache [2*layers, 1, heads, rows, head_size] whose first ``prefix_len`` rows are filled (``LlamaDecoder.read_prefix``
    makes one; several PrefixCaches may share it).  ``lengths`` (int32 [batch], on the device) counts each sequence's own rows: what a
    model has been given with this cache counts from ``keep`` on; rows that are not kept are overwritten by the next call."""

    def __init__(self, configs, batch_size, max_kv_len, prefix=None, prefix_len=0, device="cuda", dtype=None):
        if dtype is None:
            dtype = torch.float32 if prefix is None else prefix.dtype
        if prefix is not None and (prefix.dtype != dtype or not 0 <= prefix_len <= prefix.shape[3]):
            raise ValueError("the prefix has the cache's type and at least prefix_len rows")
        self.prefix, self.prefix_len = prefix, int(prefix_len)
        self.cache = torch.zeros(configs["layer_num"] * 2, batch_size, configs["head_num"], max_kv_len, configs["head_size"],
                                 dtype=dtype, device=device)
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self.max_kv_len = max_kv_len

    def size(self):
        shared = self.prefix.numel() if self.prefix is not None else 0
        return (self.cache.numel() + shared) * self.cache.element_size()

    def keep(self, tokens):
        """``tokens`` (an int, or int32 [batch] on the device) more rows of each sequence are its own from now on"""
        self.lengths.add_(tokens).clamp_(0, self.max_kv_len)

    def forget(self, sequence, length=0):
        """a sequence ends (or goes back to its first ``length`` rows): a new one may begin behind the prefix"""
        if not 0 <= length <= self.max_kv_len:
            raise ValueError("length outside the cache")
        self.lengths[sequence] = length

    def attend(self, q, k, v, inv_freq, layer_id, q_lens=None):
        return llmops.attention_rope_prefix(q, k, v, inv_freq, self.prefix, self.prefix_len, self.cache, self.lengths, layer_id, q_lens=q_lens)


class Q4Cache(PrefixCache):
    """KV cache of a batch in 4 bits (``llmops.attention_rope_q4``): 80 bytes for a token and head where fp32 takes 512 and fp16 256, on the device
    int8 [2*layers, batch, heads, max_kv_len, 80].  Each sequence has rows of its own from the first on; ``begin`` gives all of them
    the same first rows, of a cache in full width (a system prompt that was read once), which ``forget`` and ``keep`` leave."""

    def __init__(self, configs, batch_size, max_kv_len, device="cuda"):
        if configs["head_size"] != 128:
            raise ValueError("a cache in 4 bits holds heads of 128")
        self.prefix, self.prefix_len, self.begun = None, 0, 0
        self.cache = torch.zeros(configs["layer_num"] * 2, batch_size, configs["head_num"], max_kv_len, llmops.Q4_ROW_BYTES, dtype=torch.int8, device=device)
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)
        # what lengths are held to, on the device: a captured step holds them to the beginning that there is when it is replayed
        self.least, self.most = (torch.full((), n, dtype=torch.int32, device=device) for n in (0, max_kv_len))
        self.max_kv_len = max_kv_len

    def begin(self, full, rows=None):
        """The first ``rows`` rows (None: all) of a cache in full width, [2*layers, 1, heads, rows, 128] in fp32 or fp16 with k rotated
        (``LlamaDecoder.read_prefix``), become every sequence's beginning; what sequences had is forgotten."""
        rows = full.shape[3] if rows is None else int(rows)
        planes, batch = self.cache.shape[:2]
        if full.dim() != 5 or full.shape[:3] != (planes, 1, self.cache.shape[2]) or full.shape[4] != 128 or not 0 <= rows <= min(full.shape[3], self.max_kv_len):
            raise ValueError("a cache of one sequence of the same layers and heads, and rows that both have")
        if full.dtype not in (torch.float32, torch.float16) or full.device != self.cache.device:
            raise ValueError("a cache in fp32 or fp16 on the same device")
        # what cache_write_q4 would refuse is refused before anything changes: its calls write layer after layer
        e = full.element_size()
        if rows and (full.stride(4) != 1 or full.data_ptr() % 16 or any(n > 1 and full.stride(d) * e % 16 for d, n in ((0, planes), (2, full.shape[2]), (3, rows)))):
            raise ValueError("a cache with dense rows, each at 16 bytes")
        if full.untyped_storage().data_ptr() == self.cache.untyped_storage().data_ptr():
            raise ValueError("a cache in memory of its own")
        at = torch.zeros_like(self.lengths)
        for i in range(planes // 2 if rows else 0):
            k, v = (full[2 * i + j, :, :, :rows].transpose(1, 2).expand(batch, -1, -1, -1) for j in (0, 1))
            llmops.cache_write_q4(k, v, self.cache, at, i)
        self.begun = rows
        self.least.fill_(rows)
        self.lengths.fill_(rows)

    def read(self, rows=None, starts=None, dtype=torch.float16):
        """What rows stand for, in full width: [2*layers, batch, heads, rows, 128] (of one sequence: the form that ``PrefixCache`` and ``begin`` take)"""
        return llmops.cache_read_q4(self.cache, self.max_kv_len if rows is None else rows, starts=starts, dtype=dtype)

    def size(self):
        return self.cache.numel()

    def keep(self, tokens):
        """as in ``PrefixCache``; a negative number takes rows back, of a sequence's own: its beginning stays"""
        self.lengths.add_(tokens).clamp_(self.least, self.most)

    def forget(self, sequence, length=0):
        """a sequence ends (or goes back to its first ``length`` rows behind its beginning)"""
        if length < 0:
            raise ValueError("length outside the cache")
        super().forget(sequence, self.begun + length)

    def attend(self, q, k, v, inv_freq, layer_id, q_lens=None):
        return llmops.attention_rope_q4(q, k, v, inv_freq, self.cache, self.lengths, layer_id, q_lens=q_lens)


class LoraAdapters:
    """Low-rank adapters of one projection, by number: y + scale * (x A^T) B^T (``llmops.lora_add``).  ``adapters``: a list of
    (A [r, K], B [N, r], scale) whose ranks may differ (they are padded to the largest), or None where an adapter leaves this
    projection alone."""

    def __init__(self, adapters, device="cuda", dtype=torch.float16):
        some = [a for a in adapters if a is not None]
        if not some:
            raise ValueError("no adapter for this projection")
        K, N = some[0][0].shape[1], some[0][1].shape[0]
        for A, B, _ in some:
            if A.dim() != 2 or B.dim() != 2 or A.shape[1] != K or B.shape[0] != N or B.shape[1] != A.shape[0]:
                raise ValueError("adapters of one projection are A [r, K] and B [N, r] with the same K and N")
        rank = max(A.shape[0] for A, _, _ in some)
        rank += -rank % 8  # (rows of 16 bytes)
        self.A = torch.zeros(len(adapters), rank, K, dtype=dtype, device=device)
        self.B = torch.zeros(len(adapters), N, rank, dtype=dtype, device=device)
        scales = [0.0] * len(adapters)
        for i, a in enumerate(adapters):
            if a is not None:
                self.A[i, :a[0].shape[0]] = a[0].detach().to(self.A)
                self.B[i, :, :a[1].shape[1]] = a[1].detach().to(self.B)
                scales[i] = float(a[2])
        self.scales = torch.tensor(scales, dtype=torch.float32, device=device)

    def __call__(self, y, x, numbers):
        """adds to y in place; numbers int32 [B]: each sequence's adapter, -1 for none"""
        return llmops.lora_add(y, x, self.A, self.B, numbers, self.scales, out=y)

    def __repr__(self):
        return f"LoraAdapters({self.A.shape[0]} of rank {self.A.shape[1]}, {self.A.shape[2]} -> {self.B.shape[1]})"
