"""Attention over packed sequences (csrc/attn_packed.hip) against its formula in 64 bits.

Bound on one output, from the roundings the kernel makes (u = half a step of the 16-bit type, A = sum_j p_j |v_j|, l = sum of
exp(score - max)):
  * the output itself is rounded once:                                  u |o|
  * every weight is rounded to the 16-bit type before the second product: u A, and for f16 (whose steps stop shrinking below
    2^-14) at most 2^-25 for each visible key beside a largest weight of at least 1: 2^-25 sum |v| / l
  * a score's fp32 sum of D products is off by at most (D + 4) 2^-24 scale sum |q k|, which moves weights and their sum: 2 e A;
    a bias b adds two roundings of the sum, 2^-23 (|s| + |b|)
  * exp2 of the hardware, the fp32 sums and the rescales stay below 2^-18 A.
"""
import math

import pytest
import torch

from turbodiffusion_amd import ops
from turbodiffusion_amd._lib import TurboDiffusionAMDError

pytestmark = pytest.mark.gpu


def formula(q, k, v, lens, lens_k, causal, scale=None, bias=None):
    """-> (o, bound without the terms in |o|) in float64, one sequence and head at a time"""
    T, H, D = q.shape
    G = H // k.shape[1] if k.shape[1] else 1
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    for m, n in zip(lens, lens_k):
        if m and n:
            dist = torch.arange(n, device=q.device)[None, :] - (torch.arange(m, device=q.device) + n - m)[:, None]
            for h in range(H):
                Q, K_, V = q[q0:q0 + m, h].double(), k[k0:k0 + n, h // G].double(), v[k0:k0 + n, h // G].double()
                s = (Q @ K_.t().contiguous()) * scale
                e = (D + 4) * 2.0 ** -24 * scale * (Q.abs() @ K_.abs().t().contiguous())
                if bias is not None:
                    R = bias.shape[1] // 2
                    b = bias[h].double()[dist.clamp(-R, R) + R]
                    e = e + 2.0 ** -23 * (s.abs() + torch.where(b.abs() < 1e30, b.abs(), torch.zeros_like(b)))
                    s = s + b
                hide = dist > 0 if causal else torch.zeros_like(dist, dtype=torch.bool)
                s = s.masked_fill(hide, -math.inf)
                mx = s.amax(1, keepdim=True)
                w = torch.exp(s - mx.masked_fill(mx == -math.inf, 0.0))
                w = w.masked_fill(hide, 0.0)
                seen = (w.sum(1, keepdim=True) > 0)
                l = w.sum(1, keepdim=True).clamp_min(1e-300)
                p = w / l
                out[q0:q0 + m, h] = p @ V * seen
                A = p @ V.abs()
                e = torch.where(hide, torch.zeros_like(e), e).nan_to_num(0.0, 0.0, 0.0).amax(1, keepdim=True)
                t = (u + 2 * e + 2.0 ** -18) * A
                if q.dtype == torch.float16:
                    t = t + 2.0 ** -25 * ((~hide).double() @ V.abs()) / l
                tol[q0:q0 + m, h] = t * seen
        q0, k0 = q0 + m, k0 + n
    return out, tol


def check(o, ref, tol):
    u = torch.finfo(o.dtype).eps / 2
    tiny = torch.finfo(o.dtype).smallest_normal * u        # below the smallest normal number steps stop shrinking
    err = (o.double() - ref).abs()
    bad = ~(err <= tol + u * (ref.abs() + tol) + tiny)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {err[bad].max():.3e} at {bad.nonzero()[0].tolist()}"


def make(lens, lens_k, H, Hkv, D, dtype, layout="plain", seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tq, tk = sum(lens), sum(lens_k)

    def r(*s):
        return (torch.randn(*s, generator=g, device="cuda") * std).to(dtype)

    if layout == "fused":            # one projection's output
        assert tq == tk
        x = r(tq, H + 2 * Hkv, D)
        return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    if layout == "heads":            # head-major storage
        return tuple(r(h, t, D).transpose(0, 1) for h, t in ((H, tq), (Hkv, tk), (Hkv, tk)))
    if layout == "padded":           # rows with a tail, another stride for each
        return r(tq, H, D + 8)[:, :, :D], r(tk, Hkv + 1, D)[:, 1:], r(tk, Hkv, D + 64)[:, :, 64:]
    return r(tq, H, D), r(tk, Hkv, D), r(tk, Hkv, D)


LENGTHS = [
    ([1], [1]), ([5], [5]), ([32], [32]), ([33], [33]), ([64], [64]), ([65], [65]), ([127], [127]), ([128], [128]), ([129], [129]),
    ([300], [300]), ([1, 77, 2, 130, 31, 64], [1, 77, 2, 130, 31, 64]), ([0, 40, 0, 3], [0, 40, 0, 3]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(3, 3), (10, 2), (8, 1)])
def test_packed_lengths(dtype, D, causal, heads):
    H, Hkv = heads
    for i, (lens, lens_k) in enumerate(LENGTHS):
        for R in (None, 0, 20):
            q, k, v = make(lens, lens_k, H, Hkv, D, dtype, "fused", seed=i)
            bias = None if R is None else torch.randn(H, 2 * R + 1, device="cuda")
            plan = ops.AttentionPlan(lens, lens_k, heads=H, kv_heads=Hkv, head_dim=D, causal=causal)
            ref, tol = formula(q, k, v, lens, lens_k, causal, bias=bias)
            check(ops.packed_attention(q, k, v, plan, bias=bias), ref, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_queries_and_keys_of_different_lengths(D, causal):
    """a prompt under many video tokens, new tokens behind a past, more queries than keys (causal: rows that see nothing),
    no keys at all, single keys"""
    lens = [200, 3, 90, 1, 7, 1, 260, 40]
    lens_k = [37, 70, 30, 500, 0, 1, 1, 333]
    q, k, v = make(lens, lens_k, 4, 2, D, torch.bfloat16, "padded", seed=3)
    bias = torch.randn(4, 2 * 33 + 1, device="cuda")
    plan = ops.AttentionPlan(lens, lens_k, heads=4, kv_heads=2, head_dim=D, causal=causal)
    for b in (None, bias):
        ref, tol = formula(q, k, v, lens, lens_k, causal, bias=b)
        o = ops.packed_attention(q, k, v, plan, bias=b)
        check(o, ref, tol)
        assert o[294:301].abs().max() == 0                       # the sequence without keys
        if causal:
            assert o[203:203 + 60].abs().max() == 0              # 90 queries over 30 keys: the first 60 stand before any key


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,heads", [(64, (8, 8)), (128, (40, 8)), (128, (5, 1)), (64, (3, 3))])
def test_single_tokens_over_long_pasts(dtype, D, heads):
    """one row (G rows) over a long key range: split over workgroups and joined"""
    H, Hkv = heads
    lens_k = [4097, 1, 255, 20011, 1000, 128]
    lens = [1] * len(lens_k)
    q, k, v = make(lens, lens_k, H, Hkv, D, dtype, seed=5)
    for R in (None, 64):
        bias = None if R is None else torch.randn(H, 2 * R + 1, device="cuda")
        plan = ops.AttentionPlan(lens, lens_k, heads=H, kv_heads=Hkv, head_dim=D, causal=True)
        ref, tol = formula(q, k, v, lens, lens_k, True, bias=bias)
        check(ops.packed_attention(q, k, v, plan, bias=bias), ref, tol)


@pytest.mark.parametrize("longest", [383, 385])
@pytest.mark.parametrize("D", [64, 128])
def test_many_single_tokens(D, longest):
    """more workgroups than the chip holds at a time: short pasts take the tile kernel, one longer past brings all to the other"""
    lens_k = [129 + (37 * i) % 200 for i in range(299)] + [longest]
    lens = [1] * len(lens_k)
    q, k, v = make(lens, lens_k, 4, 1, D, torch.bfloat16, seed=18)
    plan = ops.AttentionPlan(lens, lens_k, heads=4, kv_heads=1, head_dim=D, causal=True)
    assert (plan._counts[1] == 0) == (longest == 383)
    ref, tol = formula(q, k, v, lens, lens_k, True)
    check(ops.packed_attention(q, k, v, plan), ref, tol)


@pytest.mark.parametrize("D", [64, 128])
def test_several_tokens_over_a_long_past_split(D):
    """few workgroups of 128 rows over long keys: their ranges are split too; beside them single tokens, on the same kernel"""
    lens, lens_k = [100, 1, 300, 2], [9000, 5000, 7001, 65]
    q, k, v = make(lens, lens_k, 2, 1, D, torch.bfloat16, seed=7)
    plan = ops.AttentionPlan(lens, lens_k, heads=2, kv_heads=1, head_dim=D, causal=True)
    assert plan.ws_floats > 0
    ref, tol = formula(q, k, v, lens, lens_k, True)
    check(ops.packed_attention(q, k, v, plan), ref, tol)


@pytest.mark.parametrize("D,heads", [(128, (40, 1)), (64, (64, 1)), (64, (300, 2)), (128, (7, 7))])
def test_many_heads_on_one_key_head(D, heads):
    """one token's heads fill a tile and spill into the next; rows walk over heads and tokens in every combination"""
    H, Hkv = heads
    lens, lens_k = [3, 1, 70, 17], [3, 900, 100, 17]
    for layout in ("plain", "padded", "heads"):
        q, k, v = make(lens, lens_k, H, Hkv, D, torch.float16, layout, seed=6)
        for causal in (True, False):
            plan = ops.AttentionPlan(lens, lens_k, heads=H, kv_heads=Hkv, head_dim=D, causal=causal)
            ref, tol = formula(q, k, v, lens, lens_k, causal)
            check(ops.packed_attention(q, k, v, plan), ref, tol)


def test_large_scores_and_growing_maxima():
    """scores of +-200 whose running maximum rises tile after tile; equal scores; a positive scale far from the default"""
    lens = [400, 64]
    q, k, v = make(lens, lens, 2, 2, 128, torch.bfloat16, seed=9)
    ramp = (torch.arange(464, device="cuda") / 40.0).to(torch.bfloat16)
    k = k.clone()
    k[:, :, 0] = ramp[:, None]
    q = q.clone()
    q[:, :, 0] = 8.0
    for scale in (None, 1.0, 0.004):
        for causal in (False, True):
            plan = ops.AttentionPlan(lens, heads=2, head_dim=128, causal=causal)
            ref, tol = formula(q, k, v, lens, lens, causal, scale=scale)
            check(ops.packed_attention(q, k, v, plan, scale=scale), ref, tol)


def test_hidden_keys_and_foreign_rows_do_not_leak():
    """infinite and NaN keys behind a causal mask, garbage rows of a neighbouring sequence and behind the last one"""
    lens = [70, 33, 90]
    q, k, v = make(lens, lens, 2, 2, 64, torch.bfloat16, seed=11)
    plan = ops.AttentionPlan(lens, heads=2, head_dim=64, causal=True)
    base = ops.packed_attention(q, k, v, plan)
    k2, v2 = torch.cat([k, k[:40]]), torch.cat([v, v[:40]])
    k2[70 + 33 + 90:] = float("nan")
    v2[70 + 33 + 90:] = float("inf")
    k2[100:103] = float("nan")           # the last three keys of sequence 1: rows before them must not notice
    o = ops.packed_attention(q, k2[:193], v2[:193], plan)
    keep = [i for i in range(193) if not 100 <= i < 103]
    assert torch.equal(o[keep], base[keep])
    v2[70:103] = float("nan")            # a whole foreign sequence
    o = ops.packed_attention(q, k2[:193], v2[:193], plan)
    assert torch.equal(o[:70], base[:70]) and torch.equal(o[103:], base[103:])


def test_bias_of_the_types_lowest_value_and_of_minus_infinity():
    lens = [50, 20]
    q, k, v = make(lens, lens, 2, 2, 64, torch.float16, seed=13)
    plan = ops.AttentionPlan(lens, heads=2, head_dim=64)
    low = torch.finfo(torch.float32).min
    near = torch.zeros(2, 2 * 3 + 1, device="cuda")
    for hide in (low, -math.inf):
        bias = near.clone()
        bias[:, 0] = hide                # distances <= -3: the far past
        ref, tol = formula(q, k, v, lens, lens, False, bias=bias)
        check(ops.packed_attention(q, k, v, plan, bias=bias), ref, tol)
    all_low = torch.full_like(near, low)                       # equal scores once the lowest value has absorbed them: the mean
    o = ops.packed_attention(q, k, v, plan, bias=all_low)
    mean = torch.stack([v[:50].double().mean(0)] * 50 + [v[50:].double().mean(0)] * 20)
    check(o, mean, torch.full_like(mean, 2.0 ** -11 * 4))      # |v| < 4.5: u A, A <= 4
    none = torch.full_like(near, -math.inf)                    # nothing to attend to
    assert ops.packed_attention(q, k, v, plan, bias=none).abs().max() == 0


@pytest.mark.parametrize("layout", ["plain", "heads", "padded"])
def test_strides_and_out(layout):
    lens = [3, 150, 64]
    q, k, v = make(lens, lens, 4, 2, 128, torch.bfloat16, layout, seed=15)
    plan = ops.AttentionPlan(lens, heads=4, kv_heads=2, head_dim=128, causal=True)
    ref, tol = formula(q, k, v, lens, lens, True)
    check(ops.packed_attention(q, k, v, plan), ref, tol)
    big = torch.full((217 + 6, 6, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[3:220, 1:5, :128]
    assert ops.packed_attention(q, k, v, plan, out=out).data_ptr() == out.data_ptr()
    check(out, ref, tol)
    big[3:220, 1:5, :128] = 7.0
    assert (big == 7.0).all()                                  # nothing around it was written


@pytest.mark.parametrize("heads", [(4, 4), (4, 2)])
@pytest.mark.parametrize("n", [1, 40, 700])
def test_one_token_into_out(heads, n):
    """a token whose stride in q and out is arbitrary, as nothing follows it"""
    H, Hkv = heads
    q, k, v = make([1], [n], H, Hkv, 128, torch.bfloat16, seed=19)
    plan = ops.AttentionPlan([1], [n], heads=H, kv_heads=Hkv, head_dim=128, causal=True)
    ref, tol = formula(q, k, v, [1], [n], True)
    big = torch.full((4, H, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    for out in (big[1:2, :, :128], torch.as_strided(big, (1, H, 128), (8, 136, 1), H * 136)):
        check(ops.packed_attention(q, k, v, plan, out=out), ref, tol)
        out[:] = 7.0
        assert (big == 7.0).all()


def test_key_offsets_past_32_bits():
    """keys and values whose rows lie 128 KB apart: 5 GB between the first and the last"""
    n, H, D = 40000, 2, 64
    store = torch.zeros(n, 65536, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    store[:, :256] = torch.randn(n, 256, generator=g, device="cuda").to(torch.bfloat16)
    k, v = store[:, :128].view(n, H, D), store[:, 128:256].view(n, H, D)
    for lens in ([1], [200]):
        q = torch.randn(lens[0], H, D, generator=g, device="cuda").to(torch.bfloat16)
        plan = ops.AttentionPlan(lens, [n], heads=H, head_dim=D, causal=True)
        ref, tol = formula(q, k, v, lens, [n], True)
        check(ops.packed_attention(q, k, v, plan), ref, tol)


def test_same_bits_every_time_on_any_stream_and_in_graphs():
    lens, lens_k = [1, 300, 1, 20, 150], [9000, 300, 40, 2000, 8000]
    q, k, v = make(lens, lens_k, 4, 2, 128, torch.bfloat16, seed=17)
    plan = ops.AttentionPlan(lens, lens_k, heads=4, kv_heads=2, head_dim=128, causal=True)
    base = ops.packed_attention(q, k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = [ops.packed_attention(q, k, v, plan) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, base) for x in o)
    graphs, outs = [], []
    for _ in range(2):                                         # two graphs, each with its own workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.packed_attention(q, k, v, plan))
        graphs.append(gr)
    for i in range(3):
        v.copy_(v.flip(0))
        base = ops.packed_attention(q, k, v, plan)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], base) and torch.equal(outs[1], base)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(4, 4), (20, 5)])
def test_a_rows_bits_are_its_own(D, heads):
    """scores that outgrow a row's first ones by 2^8 to 2^12: neither what earlier calls left in rows past a sequence's end nor a
    sequence's other rows changes a row's bits"""
    H, Hkv = heads
    lens_k = [57, 39, 33, 31, 86, 63, 53, 92, 33, 100, 128, 90]
    lens = [1, 3, 4, 4, 4, 1, 2, 4, 31, 7, 5, 90]
    q, k, v = make(lens, lens_k, H, Hkv, D, torch.bfloat16, seed=20, std=3.0)
    plan = ops.AttentionPlan(lens, lens_k, heads=H, kv_heads=Hkv, head_dim=D, causal=True)
    first = ops.packed_attention(q, k, v, plan)
    ref, tol = formula(q, k, v, lens, lens_k, True)
    check(first, ref, tol)
    for i in range(10):
        ops.packed_attention(q * 2 ** i, k.roll(1, 0), v, plan)
        assert torch.equal(ops.packed_attention(q, k, v, plan), first)
    end = sum(lens) - 90
    other = q.clone()
    other[end + 40:] *= 100.0
    assert torch.equal(ops.packed_attention(other, k, v, plan)[:end + 40], first[:end + 40])


def test_refusals():
    lens = [5, 9]
    q, k, v = make(lens, lens, 4, 2, 64, torch.bfloat16)
    plan = ops.AttentionPlan(lens, heads=4, kv_heads=2, head_dim=64)
    call = ops.packed_attention
    with pytest.raises(TypeError):
        call(q.float(), k.float(), v.float(), plan)
    with pytest.raises(TypeError):
        call(q, k.half(), v, plan)
    with pytest.raises(ValueError):
        call(q[:13], k, v, plan)
    with pytest.raises(ValueError):
        call(q, k[:, :1], v, plan)
    with pytest.raises(ValueError):
        call(q, k, v.transpose(1, 2).contiguous().transpose(1, 2), plan)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            call(q, k, v, plan, scale=scale)
    with pytest.raises(TurboDiffusionAMDError):
        call(q, k, v, plan, scale=2e38)
    with pytest.raises(ValueError):
        call(q, k, v, plan, bias=torch.zeros(4, 6, device="cuda"))
    with pytest.raises(TypeError):
        call(q, k, v, plan, bias=torch.zeros(4, 7, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(TurboDiffusionAMDError):
        call(q, k, v, plan, bias=torch.zeros(4, 2 * 4000 + 1, device="cuda"))          # more than 32 KB
    with pytest.raises(TurboDiffusionAMDError):                                         # a stride of 68 elements
        call(torch.zeros(14, 4, 68, dtype=torch.bfloat16, device="cuda")[:, :, :64], k, v, plan)
    with pytest.raises(TurboDiffusionAMDError):                                         # 2-byte alignment
        call(torch.zeros(14 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(14, 4, 64), k, v, plan)
    with pytest.raises(ValueError):
        call(q, k, v, plan, out=q)
    with pytest.raises(ValueError):
        call(q, k, v, plan, out=torch.empty(1, 4, 64, dtype=torch.bfloat16, device="cuda").expand(14, 4, 64))
    with pytest.raises(TurboDiffusionAMDError):
        call(q.cpu(), k, v, plan)
    with pytest.raises(RuntimeError):
        call(q.clone().requires_grad_(), k, v, plan)
    with torch.no_grad():
        call(q.clone().requires_grad_(), k, v, plan)
