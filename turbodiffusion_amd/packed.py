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
from ._lib import dt_code, ptr, require_gpu


def _lengths(lens, what):
    if isinstance(lens, torch.Tensor):
        if lens.dim() != 1 or lens.is_floating_point() or lens.dtype == torch.bool:
            raise ValueError(f"{what}: a 1-D tensor or a list of whole numbers, got {lens.dtype} {tuple(lens.shape)}")
        lens = lens.tolist()
    lens = list(lens)
    for n in lens:
        if isinstance(n, bool) or int(n) != n:
            raise ValueError(f"{what}: whole numbers, got {n!r}")
    return [int(n) for n in lens]


def _i64_array(values):
    return (ctypes.c_int64 * max(1, len(values)))(*values)


class _Plan:
    """A host-made table of int32 records on ``device``; ``use()`` ties it to the stream a call runs on."""

    def _upload(self, host, device):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"{type(self).__name__}: the operators run on a GPU, got device {device!r}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        with torch.cuda.device(self.device):
            self._stream = torch.cuda.current_stream()
            self.table = host.to(self.device)          # synchronous: complete for every stream

    def use(self):
        s = torch.cuda.current_stream(self.device)
        if s != self._stream:
            self.table.record_stream(s)
        return ctypes.c_void_p(s.cuda_stream)


def _guard(device):
    """launch on ``device`` whatever the current device is"""
    return torch.cuda.device(device)


def _no_grad_inputs(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("inference only: an input requires gradients (call under torch.no_grad() or detach it)")


def _overlap(a, b):
    """whether the memory ranges of two tensors intersect"""
    def span(t):
        n = sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


class AttentionPlan(_Plan):
    """The work of ``packed_attention`` for sequences of ``lens`` query and ``lens_k`` (default: the same) key tokens, in the
    order in which they are packed.  Lengths may be zero.  ``heads`` query heads share ``kv_heads`` (default: as many) key /
    value heads in groups of consecutive heads."""

    def __init__(self, lens, lens_k=None, *, heads, kv_heads=None, head_dim=128, causal=False, device="cuda"):
        self.lens = _lengths(lens, "AttentionPlan lens")
        self.lens_k = self.lens if lens_k is None else _lengths(lens_k, "AttentionPlan lens_k")
        if len(self.lens) != len(self.lens_k):
            raise ValueError(f"AttentionPlan: {len(self.lens)} query and {len(self.lens_k)} key sequences")
        self.heads, self.kv_heads = int(heads), int(heads if kv_heads is None else kv_heads)
        if self.heads < 1 or self.kv_heads < 1 or self.heads % self.kv_heads:
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


def _packed_strides(t, tokens, heads, head_dim, what):
    if t.dim() != 3 or tuple(t.shape) != (tokens, heads, head_dim):
        raise ValueError(f"packed_attention: {what} is {tuple(t.shape)}, the plan wants ({tokens}, {heads}, {head_dim})")
    if t.stride(2) != 1:
        raise ValueError(f"packed_attention: the last dimension of {what} must be contiguous")
    return (t.stride(0) if tokens > 1 else 0), (t.stride(1) if heads > 1 else 0)   # a stride that no second element uses is arbitrary


def packed_attention(q, k, v, plan, scale=None, bias=None, out=None):
    """Softmax attention over packed sequences: q [tokens, heads, D], k / v [tokens_k, kv_heads, D] (bf16 | f16, D contiguous, the
    other strides any multiple of 8 elements) -> [tokens, heads, D].

    Row i of a sequence with m queries and n keys stands at position i + n - m: the queries are its last m positions, so one new
    token over the keys kept so far is ``lens`` = 1.  ``plan.causal``: keys at or before that position only.  ``scale``: positive,
    default 1 / sqrt(D).  ``bias``: f32 [heads, 2 R + 1], added to the scaled score by distance key - query clamped to [-R, R]
    (``relative_bias``).  A row with nothing to attend to is zero.  Scores, maxima and sums are fp32; the weights are rounded to
    the inputs' type for the second product.  A masked key weighs exactly 0, so its VALUE must be finite like any other.
    ``out``: written instead of a new tensor; it may not overlap the inputs.  Any stream, capturable; the plan must outlive a
    captured graph."""
    H, Hkv, D = plan.heads, plan.kv_heads, plan.head_dim
    require_gpu(q, k, v, bias, out)
    _no_grad_inputs(q, k, v, bias)
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"packed_attention: q, k, v must all be bf16 or all f16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    dev = plan.device
    if any(t is not None and t.device != dev for t in (q, k, v, bias, out)):
        raise ValueError(f"packed_attention: the plan and every tensor must be on one device ({dev})")
    qs = _packed_strides(q, plan.tokens, H, D, "q")
    ks = _packed_strides(k, plan.tokens_k, Hkv, D, "k")
    vs = _packed_strides(v, plan.tokens_k, Hkv, D, "v")
    R = 0
    if bias is not None:
        _f32c(bias, "bias")
        if bias.dim() != 2 or bias.shape[0] != H or bias.shape[1] % 2 == 0:
            raise ValueError(f"packed_attention: bias is {tuple(bias.shape)}, wanted [{H}, 2 R + 1]")
        R = bias.shape[1] // 2
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"packed_attention: scale must be positive and finite, got {scale}")
    if out is None:
        out = torch.empty((plan.tokens, H, D), dtype=q.dtype, device=dev)
        os_ = (H * D, D)
    else:
        if out.dtype != q.dtype:
            raise TypeError(f"packed_attention: out is {out.dtype}, the inputs {q.dtype}")
        os_ = _packed_strides(out, plan.tokens, H, D, "out")
        ts, hs = os_
        if not ((H == 1 or hs >= D) and (plan.tokens <= 1 or ts >= (H - 1) * hs + D)
                or (plan.tokens <= 1 or ts >= D) and (H == 1 or hs >= (plan.tokens - 1) * ts + D)):
            raise ValueError("packed_attention: out overlaps itself")
        if any(_overlap(out, t) for t in (q, k, v)):
            raise ValueError("packed_attention: out overlaps an input")
    if plan.tokens == 0:
        return out
    with _guard(dev):
        ws = torch.empty(plan.ws_floats, dtype=torch.float32, device=dev) if plan.ws_floats else None
        call("td_attn_packed", ptr(q), *qs, ptr(k), *ks, ptr(v), *vs, ptr(out), *os_, dt_code(q.dtype), H, Hkv, D, scale,
             1 if plan.causal else 0, ptr(bias), R, ptr(plan.table), plan._counts, ptr(ws), plan.use())
    return out
