"""packed_attention where a score is far larger than what separates it from its neighbours (csrc/attn_packed.hip), against the
formula in 64 bits.

Bound on one output (u = half a step of the 16-bit type, p_j the weights, A = sum_j p_j |v_j|):
  * output rounded once, u |o|; weights rounded once, u A (f16 below its normal numbers: 2^-25 sum |v| / l, l = sum of exp(score - max))
  * score j is off by e_j = (D + 4) 2^-24 scale sum |q k| + 2^-23 (|s| + |b|), which moves o by at most sum_j p_j e_j (|v_j| + |o|):
    a key whose weight is 0 in 64 bits too, far below the others, has no part in it
  * exp2, fp32 sums and rescales: 2^-18 A."""
import math

import pytest
import torch

from turbodiffusion_amd import ops

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.float32).min


def make(lens, lens_k, H, Hkv, D, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return (torch.randn(*s, generator=g, device="cuda") * std).to(dtype)

    return r(sum(lens), H, D), r(sum(lens_k), Hkv, D), (r(sum(lens_k), Hkv, D) / std).to(dtype)


def formula(q, k, v, lens, lens_k, causal, scale, bias=None, exact_scores=False):
    T, H, D = q.shape
    G = H // k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    for m, n in zip(lens, lens_k):
        dist = torch.arange(n, device=q.device)[None, :] - (torch.arange(m, device=q.device) + n - m)[:, None]
        for h in range(H if n else 0):
            Q, K_, V = q[q0:q0 + m, h].double(), k[k0:k0 + n, h // G].double(), v[k0:k0 + n, h // G].double()
            s = (Q @ K_.t().contiguous()) * scale
            e = torch.zeros_like(s) if exact_scores else (D + 4) * 2.0 ** -24 * scale * (Q.abs() @ K_.abs().t().contiguous())
            if bias is not None:
                R = bias.shape[1] // 2
                b = bias[h].double()[dist.clamp(-R, R) + R]
                e = e + 2.0 ** -23 * (s.abs() + b.abs().nan_to_num(0.0, 0.0, 0.0))
                s = s + b
            hide = dist > 0 if causal else torch.zeros_like(dist, dtype=torch.bool)
            s = s.masked_fill(hide, -math.inf)
            mx = s.amax(1, keepdim=True)
            w = torch.exp(s - mx.masked_fill(mx == -math.inf, 0.0)).masked_fill(hide, 0.0)
            l = w.sum(1, keepdim=True)
            p = w / l.clamp_min(1e-300)
            o, A = p @ V, p @ V.abs()
            pe = torch.where(p > 0, p * e, torch.zeros_like(p))
            t = (u + 2.0 ** -18) * A + pe @ V.abs() + pe.sum(1, keepdim=True) * A
            if q.dtype == torch.float16:
                t = t + 2.0 ** -25 * ((~hide).double() @ V.abs()) / l.clamp_min(1e-300)
            out[q0:q0 + m, h], tol[q0:q0 + m, h] = o, t
        q0, k0 = q0 + m, k0 + n
    return out, tol


def check(o, ref, tol):
    u = torch.finfo(o.dtype).eps / 2
    err = (o.double() - ref).abs()
    bad = ~(err <= tol + u * (ref.abs() + tol) + torch.finfo(o.dtype).smallest_normal * u)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {err[bad].max():.3e} at {bad.nonzero()[0].tolist()}"


# every kernel form: whole prompts; single tokens on eight waves, not split and split; many tokens behind a past, split
PATHS = {
    "tile": ([300, 20], [300, 20]),
    "few": ([1, 3], [700, 300]),
    "few-split": ([1, 1], [6000, 40]),
    "tile-split": ([100, 2], [9000, 65]),
}


def plan_of(path, H, Hkv, D, causal):
    lens, lens_k = PATHS[path]
    plan = ops.AttentionPlan(lens, lens_k, heads=H, kv_heads=Hkv, head_dim=D, causal=causal)
    assert (plan._counts[0] == 0) == path.startswith("few") and (plan._counts[2] > 0) == path.endswith("split")
    return lens, lens_k, plan


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("low", [LOW, -1e30, -1e9, -1e5, -math.inf])
def test_windows_written_as_bias(dtype, D, path, low):
    """the ends of the table as low as they get, so that whole key tiles weigh nothing; scores of more than 20 nats"""
    for R in (3, 20):
        for causal in (False, True):
            lens, lens_k, plan = plan_of(path, 4, 2, D, causal)
            q, k, v = make(lens, lens_k, 4, 2, D, dtype, seed=R, std=2.0)
            bias = torch.randn(4, 2 * R + 1, device="cuda")
            bias[:, 0] = bias[:, -1] = low
            bias[0, -1] = 0.5                                  # one head looks ahead without a limit
            assert (q[:, 0].double() @ k[:, 0].double().t().contiguous()).abs().max() > 20
            ref, tol = formula(q, k, v, lens, lens_k, causal, 1.0, bias)
            check(ops.packed_attention(q, k, v, plan, scale=1.0, bias=bias), ref, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("path", PATHS)
def test_a_bias_that_absorbs_every_score(dtype, D, path):
    """the type's lowest value everywhere: equal scores, in 32 bits as in 64, so the mean"""
    lens, lens_k, plan = plan_of(path, 4, 2, D, False)
    q, k, v = make(lens, lens_k, 4, 2, D, dtype, seed=1, std=2.0)
    bias = torch.full((4, 41), LOW, device="cuda")
    ref, tol = formula(q, k, v, lens, lens_k, False, 1.0, bias, exact_scores=True)
    V = v.double().abs().mean()
    tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -18) * torch.ones_like(tol) * 4 * V          # u A; A, a mean of >= 20 |v|, is below 4 of their mean
    assert ref.isfinite().all()
    check(ops.packed_attention(q, k, v, plan, scale=1.0, bias=bias), ref, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_past_32_bits_of_steps(dtype, D, path, sign):
    """scores of up to 2^31, one product each and so exact: one step of fp32 there is 2^8, far more than a softmax sees, and the keys
    of the largest score share the weight evenly"""
    lens, lens_k, plan = plan_of(path, 4, 2, D, True)
    q, k, v = make(lens, lens_k, 4, 2, D, dtype, seed=2)
    q.zero_()
    k.zero_()
    i = torch.arange(q.shape[0], device="cuda", dtype=torch.float32)
    j = torch.arange(k.shape[0], device="cuda", dtype=torch.float32)
    q[:, :, 0] = (20000 + 331 * (i % 113)).to(dtype)[:, None]
    k[:, :, 0] = (sign * (4000 + 800 * (j * 37 % 61))).to(dtype)[:, None]
    ref, tol = formula(q, k, v, lens, lens_k, True, 1.0, exact_scores=True)
    check(ops.packed_attention(q, k, v, plan, scale=1.0), ref, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [(4, 4), (10, 2)])
def test_a_neighbour_with_large_scores_changes_no_bits(D, heads):
    H, Hkv = heads
    lens = [90, 7]
    q, k, v = make(lens, lens, H, Hkv, D, torch.bfloat16, seed=4, std=3.0)
    plan = ops.AttentionPlan(lens, heads=H, kv_heads=Hkv, head_dim=D, causal=False)
    first = ops.packed_attention(q, k, v, plan)
    other = q.clone()
    other[1:90:2] *= 1e8                               # every second row; rows of large and of ordinary scores share waves
    o = ops.packed_attention(other, k, v, plan)
    assert torch.equal(o[0:90:2], first[0:90:2]) and torch.equal(o[90:], first[90:]) and o.isfinite().all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("past,here", [(-0.9e37, -1.1e37), (-1.1e37, -0.9e37), (1.1e37, 0.9e37), (0.9e37, 1.1e37), (-1e38, LOW), (2e38, -LOW)])
def test_order_of_the_largest_biases(D, path, past, here):
    """the keys of the larger bias take all the weight, evenly: no score is more than a rounding of such a bias"""
    lens, lens_k, plan = plan_of(path, 4, 2, D, False)
    q, k, v = make(lens, lens_k, 4, 2, D, torch.bfloat16, seed=3)
    bias = torch.full((4, 21), here, device="cuda")
    bias[:, :8] = past
    ref, _ = formula(q, k, v, lens, lens_k, False, 1.0, bias, exact_scores=True)
    u = torch.finfo(torch.bfloat16).eps / 2
    check(ops.packed_attention(q, k, v, plan, scale=1.0, bias=bias), ref, torch.full_like(ref, (u + 2.0 ** -18) * v.double().abs().max()))       # u A


@pytest.mark.parametrize("heads", [(4, 4), (4, 2)])
def test_out_between_the_heads_of_a_fused_buffer(heads):
    """q | k | v | room for o in one buffer: out interleaves with every input and touches none"""
    H, Hkv = heads
    lens = [70, 1, 130]
    buf = torch.randn(201, 2 * H + 2 * Hkv, 128, device="cuda").to(torch.bfloat16)
    q, k, v, out = buf.split([H, Hkv, Hkv, H], 1)
    plan = ops.AttentionPlan(lens, heads=H, kv_heads=Hkv, head_dim=128, causal=True)
    want, before = ops.packed_attention(q, k, v, plan), buf.clone()
    assert ops.packed_attention(q, k, v, plan, out=out) is out
    assert torch.equal(out, want) and torch.equal(buf[:, :-H], before[:, :-H])
    for bad in (buf[:, 1:1 + H], buf[:, -H - 1:-1]):
        with pytest.raises(ValueError):
            ops.packed_attention(q, k, v, plan, out=bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 5])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("layout", ["plain", "padded", "heads"])
def test_some_tokens_behind_long_pasts(dtype, D, G, causal, layout):
    """up to 32 rows each on the kernel whose waves take different keys: several tokens an item, another end for each under a causal
    mask, no keys, fewer keys than queries, split ranges"""
    Hkv = 2
    H = G * Hkv
    lens = [min(n, 32 // G) for n in (2, 7, 31, 1, 32, 5, 6, 0, 16)]
    for lens_k in ([700, 5000, 131, 0, 32, 3, 200, 40, 257], [130, 129, 33, 1, 64, 300, 5, 0, 16]):
        g = torch.Generator(device="cuda").manual_seed(G)

        def r(t, h):
            if layout == "heads":
                return torch.randn(h, t, D, generator=g, device="cuda").to(dtype).transpose(0, 1)
            wide = torch.randn(t, h + 1, D + 8, generator=g, device="cuda").to(dtype)
            return wide[:, 1:, :D] if layout == "padded" else wide[:, 1:, :D].contiguous()

        q, k, v = r(sum(lens), H), r(sum(lens_k), Hkv), r(sum(lens_k), Hkv)
        plan = ops.AttentionPlan(lens, lens_k, heads=H, kv_heads=Hkv, head_dim=D, causal=causal)
        assert plan._counts[0] == 0 and (plan._counts[2] > 0) == (max(lens_k) > 4000)
        for R in (None, 0, 20):
            bias = None if R is None else torch.randn(H, 2 * R + 1, device="cuda")
            ref, tol = formula(q, k, v, lens, lens_k, causal, D ** -0.5, bias)
            check(ops.packed_attention(q, k, v, plan, bias=bias), ref, tol)
        big = torch.full((sum(lens) + 2, H + 1, D + 8), 7.0, dtype=dtype, device="cuda")
        ops.packed_attention(q, k, v, plan, bias=bias, out=big[1:-1, 1:, :D])
        check(big[1:-1, 1:, :D], ref, tol)
        big[1:-1, 1:, :D] = 7.0
        assert (big == 7.0).all()
