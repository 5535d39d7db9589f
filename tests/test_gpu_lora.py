"""Adapters of many requests (csrc/lora.hip) against the formula in 64 bits.

Bound on one output (u = half a step of the 16-bit type): the output is rounded once, u |o|; s S (S = A x) is rounded once before
the second product, u sum_r |s S_r B_r|; the fp32 sum of K products behind S is off by at most (K + 8) 2^-24 sum |x a|, and the
fp32 sum over the ranks, the scale and y by (rank + 4) 2^-24 of the sum of what it adds up."""
import pytest
import torch

from turbodiffusion_amd import ops, packed
from turbodiffusion_amd._lib import TurboDiffusionAMDError

pytestmark = pytest.mark.gpu


def formula(y, x, pairs, scales, lens, ids):
    out, tol = y.double(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    u, f = torch.finfo(y.dtype).eps / 2, 2.0 ** -24
    r0 = 0
    for m, i in zip(lens, ids):
        if i >= 0 and m:
            xs = x[r0:r0 + m].double()
            a, b = pairs[i][0].double(), pairs[i][1].double()
            s = scales[i] * (xs @ a.t().contiguous())
            out[r0:r0 + m] += s @ b.t().contiguous()
            e = u * s.abs() + (x.shape[1] + 8) * f * abs(scales[i]) * (xs.abs() @ a.abs().t().contiguous())
            if y.dtype == torch.float16:
                e = e + 2.0 ** -25
            bt = b.abs().t().contiguous()
            tol[r0:r0 + m] = e @ bt + (a.shape[0] + 4) * f * (s.abs() @ bt + y[r0:r0 + m].double().abs())
        r0 += m
    return out, tol


def check(o, ref, tol):
    u = torch.finfo(o.dtype).eps / 2
    err = (o.double() - ref).abs()
    bad = ~(err <= tol + u * (ref.abs() + tol) + torch.finfo(o.dtype).smallest_normal * u)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {err[bad].max():.3e} at {bad.nonzero()[0].tolist()}"


def make(rows, k, n, ranks, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    pairs = [((r(q, k) * k ** -0.5).to(dtype), r(n, q).to(dtype)) for q in ranks]
    return r(rows, n).to(dtype), r(rows, k).to(dtype), pairs, [(-1.0) ** i * (0.5 + i) for i in range(len(ranks))]


CASES = [
    # lens, ids, ranks
    ([1], [0], [16]),
    ([1], [0], [1]),
    ([1, 1, 1, 1, 1, 1], [2, 0, -1, 2, 1, 2], [8, 13, 64]),
    ([17, 0, 64, 65, 3], [1, 0, -1, 0, 1], [4, 128]),
    ([200, 130, 64, 1], [0, 0, 1, 0], [33, 256]),
    ([5, 6], [-1, -1], [16]),
    ([63, 1, 70], [0, 1, 0], [16, 32]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,n", [(64, 64), (1536, 200), (8, 8), (1000, 1544), (4096, 136)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_lora_rows_ranks_and_sizes(dtype, k, n, case):
    lens, ids, ranks = CASES[case]
    y, x, pairs, scales = make(sum(lens), k, n, ranks, dtype, seed=case)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    ref, tol = formula(y, x, pairs, scales, lens, ids)
    y0 = y.clone()
    o = ops.lora_add(y, x, bank, plan)
    check(o, ref, tol)
    assert torch.equal(y, y0)
    assert ops.lora_add(y, x, bank, plan, out=y) is y            # in place: the same bits
    assert torch.equal(y, o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n", [(1500, 1000, 1544), (1, 10240, 64), (70, 10248, 256), (300, 4104, 6152)])
def test_lora_two_launches(dtype, rows, k, n):
    """between one launch and many rows: K split over workgroups, tiles of 32 rows, small ranks"""
    lens, ids = [rows // 3, rows - rows // 3], [1, 0]
    y, x, pairs, scales = make(rows, k, n, [12, 64], dtype, seed=3)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    assert packed._lora_layout(y, x, bank, plan, None)[3] > 0
    ref, tol = formula(y, x, pairs, scales, lens, ids)
    check(ops.lora_add(y, x, bank, plan), ref, tol)


@pytest.mark.parametrize("rank", [16, 100])
def test_lora_many_rows(rank):
    """enough rows for tiles of 256"""
    lens, ids = [20000, 13001], [1, 0]
    y, x, pairs, scales = make(sum(lens), 520, 264, [rank, 24], torch.bfloat16, seed=2)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    ref, tol = formula(y, x, pairs, scales, lens, ids)
    check(ops.lora_add(y, x, bank, plan), ref, tol)


def test_lora_strides_and_guard_rows():
    lens, ids = [30, 70, 5], [0, 1, -1]
    y, x, pairs, scales = make(105, 256, 128, [16, 40], torch.bfloat16, seed=4)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    ref, tol = formula(y, x, pairs, scales, lens, ids)
    wide = torch.full((110, 640), 3.0, dtype=torch.bfloat16, device="cuda")
    wide[2:107, 256:384] = y
    xw = torch.full((105, 520), float("nan"), dtype=torch.bfloat16, device="cuda")
    xw[:, 8:264] = x
    o = wide[2:107, 256:384]
    assert ops.lora_add(o, xw[:, 8:264], bank, plan, out=o) is o
    check(o, ref, tol)
    wide[2:107, 256:384] = 3.0
    assert (wide == 3.0).all()
    out = torch.full((107, 136), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.lora_add(y, x, bank, plan, out=out[1:106, :128])
    check(out[1:106, :128], ref, tol)
    out[1:106, :128] = 5.0
    assert (out == 5.0).all()


def test_lora_rows_of_other_requests_do_not_leak():
    lens, ids = [10, 20, 10], [0, 1, 0]
    y, x, pairs, scales = make(40, 128, 64, [16, 16], torch.float16, seed=5)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    base = ops.lora_add(y, x, bank, plan)
    x[10:30] = float("nan")
    y[35] = float("inf")
    o = ops.lora_add(y, x, bank, plan)
    keep = list(range(10)) + list(range(30, 35)) + list(range(36, 40))
    assert torch.equal(o[keep], base[keep])


@pytest.mark.parametrize("rank", [5, 8, 24, 40, 100, 200])
@pytest.mark.parametrize("rows,k", [(3, 64), (40, 8192), (8200, 64)])
def test_lora_infinities_stay_what_the_formula_makes_of_them(rank, rows, k):
    """a row whose A x overflows f16 in one rank, and one with an infinite x: infinities of B's signs, no NaN from the ranks that
    the layout adds"""
    y, x, pairs, _ = make(rows, k, 64, [rank], torch.float16, seed=6)
    a, b = pairs[0]
    x[0], x[1] = 0.0, 0.0
    x[0, 3] = 60000.0
    x[1, 3] = float("inf")
    a[:, 3] = 0.5
    a[0, 3] = 4.0                                     # 60000 * 4 is past f16, 60000 / 2 is not
    b.copy_(b.abs() * 2.0 ** -6)
    o = ops.lora_add(y, x, ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0]))
    assert (o[0] == float("inf")).all() and (o[1] == float("inf")).all()
    assert torch.isfinite(o[2:]).all()


def test_lora_row_offsets_past_32_bits():
    """rows 2 MB apart in x, y and out"""
    lens, ids = [1500, 700], [0, -1]
    y, x, pairs, scales = make(2200, 64, 64, [16], torch.bfloat16, seed=6)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    far = torch.empty(2200, 1 << 20, dtype=torch.bfloat16, device="cuda")
    far[:, :64], far[:, 64:128] = y, x
    ref, tol = formula(y, x, pairs, scales, lens, ids)
    check(ops.lora_add(far[:, :64], far[:, 64:128], bank, plan), ref, tol)
    check(ops.lora_add(far[:, :64], far[:, 64:128].contiguous(), bank, plan, out=far[:, :64]), ref, tol)


def test_lora_same_bits_on_any_stream_and_in_graphs():
    lens, ids = [100, 1, 64, 300], [0, 1, 2, 0]
    y, x, pairs, scales = make(465, 1024, 512, [64, 8, 16], torch.bfloat16, seed=7)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    base = ops.lora_add(y, x, bank, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = [ops.lora_add(y, x, bank, plan) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(v, base) for v in o)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.lora_add(y, x, bank, plan))
        graphs.append(gr)
    for _ in range(3):
        x.copy_(x.flip(0))
        base = ops.lora_add(y, x, bank, plan)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], base) and torch.equal(outs[1], base)


def test_lora_beside_int8_linear():
    """the shared projection in INT8, the adapters of three requests added to its output in place"""
    lens, ids = [40, 1, 90], [1, -1, 0]
    y, x, pairs, scales = make(131, 256, 384, [16, 8], torch.bfloat16, seed=8)
    lin = torch.nn.Linear(256, 384, dtype=torch.bfloat16, device="cuda")
    base = ops.Int8Linear.from_linear(lin)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    with torch.no_grad():
        y = base(x)
        ref, tol = formula(y, x, pairs, scales, lens, ids)
        check(ops.lora_add(y, x, bank, plan, out=y), ref, tol)


def test_lora_refusals():
    lens, ids = [4, 6], [0, 1]
    y, x, pairs, scales = make(10, 64, 64, [8, 16], torch.bfloat16)
    bank, plan = ops.AdapterBank(pairs, scales), ops.AdapterPlan(lens, ids)
    call = ops.lora_add
    with pytest.raises(TypeError):
        call(y.half(), x, bank, plan)
    with pytest.raises(TypeError):
        call(y.half(), x.half(), bank, plan)
    with pytest.raises(ValueError):
        call(y, x[:9], bank, plan)
    with pytest.raises(ValueError):
        call(y, x[:, :56], bank, plan)
    with pytest.raises(ValueError):
        call(y.t().contiguous().t(), x, bank, plan)
    with pytest.raises(ValueError):
        call(y, x, bank, ops.AdapterPlan(lens, [0, 2]))
    with pytest.raises(ValueError):
        call(y, x, bank, plan, out=torch.empty(1, 64, dtype=torch.bfloat16, device="cuda").expand(10, 64))
    with pytest.raises(ValueError):
        call(y, y, ops.AdapterBank([(p[0], p[1]) for p in pairs]), plan, out=y)
    big = torch.zeros(11, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        call(big[:10], x, bank, plan, out=big[1:])
    with pytest.raises(TurboDiffusionAMDError):
        call(torch.zeros(10, 68, dtype=torch.bfloat16, device="cuda")[:, :64], x, bank, plan)
    with pytest.raises(TurboDiffusionAMDError):
        call(torch.zeros(10 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(10, 64), x, bank, plan)
    with pytest.raises(TurboDiffusionAMDError):
        call(y.cpu(), x, bank, plan)
    with pytest.raises(RuntimeError):
        call(y, x.clone().requires_grad_(), bank, plan)
    with pytest.raises(ValueError):
        ops.AdapterBank([(torch.zeros(257, 64, dtype=torch.bfloat16), torch.zeros(64, 257, dtype=torch.bfloat16))])
    e = ops.AdapterPlan([], [])
    assert call(y[:0], x[:0], bank, e).shape == (0, 64)
