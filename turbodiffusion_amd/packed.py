"""Operators for the prompts and adapters of many requests at once (csrc/attn_packed.hip, csrc/lora.hip).

The rows of all requests stand behind one another without padding.  What depends on the lengths alone - which workgroup does
what - is a PLAN, made once per batch on the host and used by every layer: ``AttentionPlan`` for ``packed_attention``,
``AdapterPlan`` for ``lora_add``.  Inference only: inputs that require gradients are refused.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L
from .kernels import call, _f32c
from ._lib import dt_code, ptr, require_gpu, stream_ptr


# torch.cuda.current_device / current_stream without the Python around them: 4 of a small call's 13 us
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _lengths(lens, what):
    if isinstance(lens, torch.Tensor):
        if lens.dim() != 1 or lens.is_floating_point() or lens.dtype == torch.bool:
            raise ValueError(f"{what}: a 1-D tensor or a list of whole numbers, got {lens.dtype} {tuple(lens.shape)}")
        lens = lens.tolist()
    lens = list(lens)
    for n in lens:
        if isinstance(n, bool) or isinstance(n, float) and not math.isfinite(n) or int(n) != n:
            raise ValueError(f"{what}: whole numbers, got {n!r}")
        if not -1 << 63 <= n < 1 << 63:
            raise ValueError(f"{what}: {n} does not fit 64 bits")
    return [int(n) for n in lens]


def _i64_array(values):
    return (ctypes.c_int64 * max(1, len(values)))(*values)


class _Plan:
    """A host-made table of int32 records on ``device``."""

    def _upload(self, host, device):
        self._admitted = {}        # layouts (shapes, strides, types) that passed the checks -> what the C entry takes for them
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"{type(self).__name__}: the operators run on a GPU, got device {device!r}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        with torch.cuda.device(self.device):
            self._stream = torch.cuda.current_stream().cuda_stream
            self.table = host.to(self.device)          # synchronous: complete for every stream

    def _admit(self, key, value):
        if len(self._admitted) >= 256:
            self._admitted.clear()
        self._admitted[key] = value
        return value

    def _launch(self, fn, *held):
        """``fn(stream)`` with the plan's device current; the table and ``held`` (what else the framework keeps for the caller) stay
        allocated while that stream needs them"""
        if _current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._launch(fn, *held)
        stream = _raw_stream(self.device.index)
        if stream != self._stream or held:
            for t in (self.table, *held):
                t.record_stream(torch.cuda.current_stream())
        fn(stream)


def _check_tensors(what, dev, *tensors):
    """GPU tensors on ``dev`` that want no gradient (None: an argument left out)"""
    index, grad = dev.index, torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if t.get_device() != index:
            require_gpu(t)
            raise ValueError(f"{what}: the plan and every tensor must be on one device ({dev}, got {t.device})")
        if grad and t.requires_grad:
            raise RuntimeError(f"{what} is inference only: an input requires gradients (call under torch.no_grad() or detach it)")


def _overlap(a, b):
    """whether two tensors may share memory.  Their ranges may intersect without it: column ranges of one buffer, heads of a fused
    projection.  Seen modulo a stride of either, a tensor is one interval if the strides that are no multiples of it fit into one period;
    two intervals apart there are apart everywhere."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    dims = [[(n, st * t.element_size()) for n, st in zip(t.shape, t.stride()) if n > 1] for t in (a, b)]
    at = a.data_ptr(), b.data_ptr()
    size = [sum((n - 1) * st for n, st in d) + t.element_size() for d, t in zip(dims, (a, b))]
    if at[0] + size[0] <= at[1] or at[1] + size[1] <= at[0]:
        return False
    for period in {st for d in dims for _, st in d if st}:
        wa, wb = (sum((n - 1) * st for n, st in d if st % period) + t.element_size() for d, t in zip(dims, (a, b)))
        gap = (at[1] - at[0]) % period               # from the beginning of a's interval to that of b's, and on to a's next
        if wa <= gap and wb <= period - gap:
            return False
    return True


class AttentionPlan(_Plan):
    """The work of ``packed_attention`` for sequences of ``lens`` query and ``lens_k`` (default: the same) key tokens, in the
    order in which they are packed.  Lengths may be zero.  ``heads`` query heads share ``kv_heads`` (default: as many) key /
    value heads in groups of consecutive heads."""

    def __init__(self, lens, lens_k=None, *, heads, kv_heads=None, head_dim=128, causal=False, device="cuda"):
        self.lens = _lengths(lens, "AttentionPlan lens")
        self.lens_k = self.lens if lens_k is None else _lengths(lens_k, "AttentionPlan lens_k")
        if len(self.lens) != len(self.lens_k):
            raise ValueError(f"AttentionPlan: {len(self.lens)} query and {len(self.lens_k)} key sequences")
        self.heads, self.kv_heads = _lengths([heads, heads if kv_heads is None else kv_heads], "AttentionPlan heads, kv_heads")
        if not 1 <= self.heads < 1 << 31 or self.kv_heads < 1 or self.heads % self.kv_heads:
            raise ValueError(f"AttentionPlan: {heads} heads do not share {kv_heads} key heads evenly")
        if head_dim not in (64, 128):
            raise ValueError(f"AttentionPlan: head_dim = {head_dim} (64 or 128)")
        self.head_dim, self.causal = int(head_dim), bool(causal)
        lq, lk = _i64_array(self.lens), _i64_array(self.lens_k)
        self._counts = (ctypes.c_int64 * 6)()
        args = (lq, lk, len(self.lens), self.heads, self.kv_heads, 1 if self.causal else 0)
        L.call("td_attn_packed_plan", *args, None, 0, self._counts)
        n = self._counts[0] + self._counts[1] + self._counts[2]
        host = torch.zeros(max(1, n), 8, dtype=torch.int32)
        L.call("td_attn_packed_plan", *args, ptr(host), n, self._counts)
        self.tokens, self.tokens_k = self._counts[4], self._counts[5]
        self.ws_floats = self._counts[3] * self.kv_heads * (self.head_dim + 2)
        self._upload(host, device)


def _layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def _packed_strides(t, tokens, heads, head_dim, what):
    if t.shape != (tokens, heads, head_dim):
        raise ValueError(f"packed_attention: {what} is {tuple(t.shape)}, the plan wants ({tokens}, {heads}, {head_dim})")
    ts, hs, ds = t.stride()
    if ds != 1:
        raise ValueError(f"packed_attention: the last dimension of {what} must be contiguous")
    return (ts if tokens > 1 else 0), (hs if heads > 1 else 0)   # a stride that no second element uses is arbitrary


def _attention_layout(plan, q, k, v, scale, bias, out):
    """The checks that depend on shapes, strides, types and scale alone -> (strides as a C array, dtype code, scale, bias range)"""
    H, Hkv, D, dt = plan.heads, plan.kv_heads, plan.head_dim, q.dtype
    if k.dtype != dt or v.dtype != dt or (dt != torch.bfloat16 and dt != torch.float16):
        raise TypeError(f"packed_attention: q, k, v must all be bf16 or all f16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    strides = (*_packed_strides(q, plan.tokens, H, D, "q"), *_packed_strides(k, plan.tokens_k, Hkv, D, "k"),
               *_packed_strides(v, plan.tokens_k, Hkv, D, "v"))
    R = 0
    if bias is not None:
        _f32c(bias, "bias")
        if bias.dim() != 2 or bias.shape[0] != H or bias.shape[1] % 2 == 0:
            raise ValueError(f"packed_attention: bias is {tuple(bias.shape)}, wanted [{H}, 2 R + 1]")
        R = bias.shape[1] // 2
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if not 0.0 < scale < math.inf:
        raise ValueError(f"packed_attention: scale must be positive and finite, got {scale}")
    if out is None:
        strides += (H * D, D)
    else:
        if out.dtype != dt:
            raise TypeError(f"packed_attention: out is {out.dtype}, the inputs {dt}")
        ts, hs = _packed_strides(out, plan.tokens, H, D, "out")
        if not ((H == 1 or hs >= D) and (plan.tokens <= 1 or ts >= (H - 1) * hs + D)
                or (plan.tokens <= 1 or ts >= D) and (H == 1 or hs >= (plan.tokens - 1) * ts + D)):
            raise ValueError("packed_attention: out overlaps itself")
        strides += (ts, hs)
    return _i64_array(strides), dt_code(dt), scale, R


def packed_attention(q, k, v, plan, scale=None, bias=None, out=None):
    """Softmax attention over packed sequences: q [tokens, heads, D], k / v [tokens_k, kv_heads, D] (bf16 | f16, D contiguous, the
    other strides any multiple of 8 elements) -> [tokens, heads, D].

    Row i of a sequence with m queries and n keys stands at position i + n - m: the queries are its last m positions, so one new
    token over the keys kept so far is ``lens`` = 1.  ``plan.causal``: keys at or before that position only.  ``scale``: positive,
    default 1 / sqrt(D).  ``bias``: f32 [heads, 2 R + 1], added to the scaled score by distance key - query clamped to [-R, R]
    (``relative_bias``); finite values past 2.36e38 count as that, and (2 R + 193) heads / kv_heads may not exceed 8192.  A row with
    nothing to attend to is zero.  Scores, maxima and sums are fp32; the weights are rounded to the inputs' type for the second
    product.  A masked key weighs exactly 0, so its VALUE must be finite like any other.
    ``out``: written instead of a new tensor; it may not overlap the inputs.  Any stream, capturable; the plan must outlive a
    captured graph."""
    _check_tensors("packed_attention", plan.device, q, k, v, bias, out)
    if scale is not None and type(scale) is not float:
        scale = float(scale)
    key = (_layout(q), _layout(k), _layout(v), scale, _layout(bias), _layout(out))
    strides, dt, scale_, R = plan._admitted.get(key) or plan._admit(key, _attention_layout(plan, q, k, v, scale, bias, out))
    if out is None:
        out = q.new_empty((plan.tokens, plan.heads, plan.head_dim))
    elif any(_overlap(out, t) for t in (q, k, v, bias) if t is not None):
        raise ValueError("packed_attention: out overlaps an input")
    if plan.tokens == 0:
        return out
    ws = q.new_empty(plan.ws_floats, dtype=torch.float32) if plan.ws_floats else None
    plan._launch(lambda stream: call(
        "td_attn_packed", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), strides, dt, plan.heads, plan.kv_heads, plan.head_dim, scale_,
        plan.causal, None if bias is None else bias.data_ptr(), R, plan.table.data_ptr(), plan._counts, None if ws is None else ws.data_ptr(),
        stream))
    return out


def distance_buckets(rel, num_buckets, max_dist, bidirectional=True):
    """Bucket ids of distances ``rel`` = key - query (T5RelativeEmbedding._relative_position_bucket, umt5.py:289-305): half of a
    direction's buckets hold one distance each, the others widen logarithmically up to ``max_dist``.  Not bidirectional: later
    keys share bucket 0 and earlier ones have all buckets."""
    nb = num_buckets // 2 if bidirectional else num_buckets
    exact = nb // 2
    if bidirectional:
        out = (rel > 0).long() * nb
        rel = rel.abs()
    else:
        out = torch.zeros_like(rel)
        rel = (-rel).clamp(min=0)
    large = exact + (torch.log(rel.float() / exact) / math.log(max_dist / exact) * (nb - exact)).long()
    large = torch.min(large, torch.full_like(large, nb - 1))
    return out + torch.where(rel < exact, rel, large)


def relative_bias(table, max_dist=128, bidirectional=True):
    """The learned relative position bias as ``packed_attention`` reads it: ``table`` [buckets, heads] -> f32 [heads, 2 max_dist + 1],
    entry max_dist + d for key - query = d; every distance beyond max_dist is in its direction's last bucket.  Laid out once
    per layer."""
    if table.dim() != 2:
        raise ValueError(f"relative_bias: table is {tuple(table.shape)}, wanted [buckets, heads]")
    exact = table.shape[0] // (4 if bidirectional else 2)
    if exact < 1 or max_dist <= exact:
        raise ValueError(f"relative_bias: {table.shape[0]} buckets up to distance {max_dist} leave none to widen")
    rel = torch.arange(-max_dist, max_dist + 1, device=table.device)
    return table.detach().float()[distance_buckets(rel, table.shape[0], max_dist, bidirectional)].t().contiguous()


class AdapterBank:
    """Low-rank pairs for ONE projection, laid out once: ``pairs[i]`` = (A [rank, k], B [n, rank]), all bf16 or all f16, ranks of
    1 to 256 that may differ; ``scales[i]`` (default 1) multiplies the update (the usual alpha / rank)."""

    MAX_RANK = 256
    SPARE = 16384          # elements behind the last adapter that a call may read (td_lora_add)

    def __init__(self, pairs, scales=None, device="cuda"):
        pairs = list(pairs)
        if not pairs:
            raise ValueError("AdapterBank: no adapters")
        scales = [1.0] * len(pairs) if scales is None else [float(s) for s in scales]
        if len(scales) != len(pairs):
            raise ValueError(f"AdapterBank: {len(pairs)} adapters, {len(scales)} scales")
        if not torch.tensor(scales, dtype=torch.float32).isfinite().all():
            raise ValueError(f"AdapterBank: scales must be finite in fp32, got {scales}")
        self.dtype = pairs[0][0].dtype
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"AdapterBank: bf16 or f16 adapters, got {self.dtype}")
        self.k, self.n = pairs[0][0].shape[-1], pairs[0][1].shape[0]
        if self.k % 8 or self.n % 8 or not self.k or not self.n:
            raise ValueError(f"AdapterBank: k = {self.k}, n = {self.n} must be positive multiples of 8")
        for i, (a, b) in enumerate(pairs):
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.k or b.shape != (self.n, a.shape[0]):
                raise ValueError(f"AdapterBank: adapter {i} is {tuple(a.shape)} / {tuple(b.shape)}, wanted [rank, {self.k}] / [{self.n}, rank]")
            if a.dtype != self.dtype or b.dtype != self.dtype:
                raise TypeError(f"AdapterBank: adapter {i} is {a.dtype} / {b.dtype}, the first {self.dtype}")
            if not 1 <= a.shape[0] <= self.MAX_RANK:
                raise ValueError(f"AdapterBank: adapter {i} has rank {a.shape[0]} (1 to {self.MAX_RANK})")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"AdapterBank: the operators run on a GPU, got device {device!r}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.ranks = [a.shape[0] for a, _ in pairs]
        r8 = [-(-r // 8) * 8 for r in self.ranks]
        self.max_rank = max(r8)
        self.layout = (self.dtype, self.k, self.n, len(pairs), self.max_rank)
        k32, n32 = -(-self.k // 32) * 32, -(-self.n // 32) * 32
        with torch.cuda.device(self.device):
            self._stream = torch.cuda.current_stream().cuda_stream
            self.data = torch.empty(sum(r * (k32 + n32) for r in r8) + self.SPARE, dtype=self.dtype, device=self.device)
            meta = torch.zeros(len(pairs), 3, dtype=torch.int64)
            off, st = 0, stream_ptr()
            for i, ((a, b), r, r_) in enumerate(zip(pairs, self.ranks, r8)):
                oa, ob = off, off + r_ * k32
                off = ob + n32 * r_
                a, b = (t.detach().to(self.device).contiguous() for t in (a, b))
                call("td_lora_pack", ptr(a), self.k, ptr(b), r, r, self.k, self.n, ptr(self.data[oa:]), ptr(self.data[ob:]), st)
                meta[i, 0], meta[i, 1] = oa, ob
                words = meta[i, 2:].view(torch.int32)
                words[0] = r
                words.view(torch.float32)[1] = scales[i]
            self.meta = meta.to(self.device)
        torch.cuda.current_stream(self.device).synchronize()      # laid out once, complete for every stream

    def __len__(self):
        return len(self.ranks)


class AdapterPlan(_Plan):
    """The work of ``lora_add`` for packed requests of ``lens`` rows, request i with adapter ``ids[i]`` (-1: none)."""

    def __init__(self, lens, ids, device="cuda"):
        self.lens, self.ids = _lengths(lens, "AdapterPlan lens"), _lengths(ids, "AdapterPlan ids")
        if len(self.lens) != len(self.ids):
            raise ValueError(f"AdapterPlan: {len(self.lens)} lengths, {len(self.ids)} adapter ids")
        args = (_i64_array(self.lens), _i64_array(self.ids), len(self.lens))
        self._counts = (ctypes.c_int64 * 6)()
        L.call("td_lora_plan", *args, None, 0, self._counts)
        n = 4 * (self._counts[0] + self._counts[1]) + self._counts[2]
        host = torch.zeros(max(1, n), dtype=torch.int32)
        L.call("td_lora_plan", *args, ptr(host), n, self._counts)
        self.rows = self._counts[2]
        self._upload(host, device)


def _rows(t, rows, cols, what):
    if t.shape != (rows, cols):
        raise ValueError(f"lora_add: {what} is {tuple(t.shape)}, wanted ({rows}, {cols})")
    ld, one = t.stride()
    if one != 1:
        raise ValueError(f"lora_add: the last dimension of {what} must be contiguous")
    return ld if rows > 1 else 0


def _lora_layout(y, x, bank, plan, out):
    """The checks that depend on shapes, strides, types and the bank's sizes alone -> (row strides of y, x, out; workspace; dtype code)"""
    if x.dtype != bank.dtype or y.dtype != bank.dtype:
        raise TypeError(f"lora_add: x is {x.dtype}, y {y.dtype}, the adapters {bank.dtype}")
    if plan._counts[4] > len(bank):
        raise ValueError(f"lora_add: the plan names adapter {plan._counts[4] - 1}, the bank holds {len(bank)}")
    ldx, ldy, ldo = _rows(x, plan.rows, bank.k, "x"), _rows(y, plan.rows, bank.n, "y"), bank.n
    if out is not None:
        if out.dtype != y.dtype:
            raise TypeError(f"lora_add: out is {out.dtype}, y {y.dtype}")
        ldo = _rows(out, plan.rows, bank.n, "out")
        if plan.rows > 1 and ldo < bank.n:
            raise ValueError("lora_add: out overlaps itself")
    floats = ctypes.c_int64()
    L.call("td_lora_workspace", plan._counts, bank.k, bank.n, bank.max_rank, ctypes.byref(floats))
    return ldy, ldx, ldo, floats.value, dt_code(y.dtype)


def lora_add(y, x, bank, plan, out=None):
    """y [rows, n] + the adapters' updates of x [rows, k] (row stride: any multiple of 8 elements) -> [rows, n]: row r of a request
    with adapter i becomes y[r] + scale_i * (x[r] A_i^T) B_i^T, one without stays y[r].  ``y`` is the output of the projection that
    all requests share (``int8_linear``, ``Int8Linear``, a 16-bit GEMM).  ``out``: written instead of a new tensor; ``out=y`` adds
    in place; any other overlap is refused.  x A^T is summed in fp32 and rounded once to the adapters' type (f16: each row times a power
    of two, undone in fp32, so that its size does not matter); scale and sum are fp32, rounded with the result.  Any stream, capturable; bank and plan must outlive a captured graph."""
    dev = plan.device
    _check_tensors("lora_add", dev, y, x, out, bank.data)
    key = (_layout(y), _layout(x), _layout(out), bank.layout)
    ldy, ldx, ldo, floats, dt = plan._admitted.get(key) or plan._admit(key, _lora_layout(y, x, bank, plan, out))
    if out is None:
        out = y.new_empty((plan.rows, bank.n))
    elif _overlap(out, x) or ((out.data_ptr() != y.data_ptr() or ldo != ldy) and _overlap(out, y)):
        raise ValueError("lora_add: out overlaps an input (out=y alone may)")
    if plan.rows == 0:
        return out
    ws = y.new_empty(floats, dtype=torch.float32) if floats else None
    plan._launch(lambda stream: call(
        "td_lora_add", x.data_ptr(), ldx, y.data_ptr(), ldy, out.data_ptr(), ldo, dt, bank.k, bank.n, bank.data.data_ptr(),
        bank.meta.data_ptr(), len(bank), bank.max_rank, plan.table.data_ptr(), plan._counts, None if ws is None else ws.data_ptr(), stream),
        *(() if _raw_stream(dev.index) == bank._stream else (bank.data, bank.meta)))
    return out
