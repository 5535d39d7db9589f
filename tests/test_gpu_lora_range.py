"""lora_add over the range of its types' values (csrc/lora.hip), against the formula in 64 bits.

Bound on one output (u = half a step of the 16-bit type, S = A x): the output is rounded once, u |o|; S once, u |S_r|, and in f16, where
a row of S is brought to 2^14 .. 2^15 and steps stop shrinking at 2^-24, by at most 2^-25 of 2^-14 of the row's largest; the fp32 sum of K
products is off by at most (K + 8) 2^-24 sum |x a|, the one over the ranks, the scale and y by (rank + 4) 2^-24 of what it adds up."""
import pytest
import torch

from turbodiffusion_amd import ops

pytestmark = pytest.mark.gpu


def formula(y, x, a, b, scale):
    u, f = torch.finfo(y.dtype).eps / 2, 2.0 ** -24
    x, a, b, y = (t.double() for t in (x, a, b, y))
    s = x @ a.t().contiguous()
    e = u * s.abs() + (x.shape[1] + 8) * f * (x.abs() @ a.abs().t().contiguous())
    if u == 2.0 ** -11:
        e = e + 2.0 ** -39 * s.abs().amax(1, keepdim=True)
    bt = b.t().contiguous()
    out = y + scale * (s @ bt)
    return out, abs(scale) * (e @ bt.abs()) + (a.shape[0] + 4) * f * (abs(scale) * (s.abs() @ bt.abs()) + y.abs())


def check(o, ref, tol):
    """within the bound; past the type's largest value (and half a step) infinity of the right sign"""
    u, top = torch.finfo(o.dtype).eps / 2, torch.finfo(o.dtype).max * (1 + torch.finfo(o.dtype).eps / 4)
    t = tol + u * (ref.abs() + tol) + torch.finfo(o.dtype).smallest_normal * u
    d = o.double()
    near, inf = (d - ref).abs() <= t, torch.isinf(d) & (d.sign() == ref.sign()) & (ref.abs() + t >= top)
    bad = ~(near | inf)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the first {o[bad][0].item()} for {ref[bad][0].item()} at {bad.nonzero()[0].tolist()}"
    return int((~inf).sum())


# one launch; K split over workgroups; tiles of 256 rows
SIZES = [(3, 64), (40, 8192), (8200, 64)]


def make(rows, k, rank, dtype, seed=6, n=64):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    return r(rows, n).to(dtype), r(rows, k).to(dtype), (r(rank, k) * k ** -0.5).to(dtype), r(n, rank).to(dtype)


@pytest.mark.parametrize("rank", [5, 8, 24, 40, 100, 200])
@pytest.mark.parametrize("rows,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_an_inner_product_past_f16(dtype, rank, rows, k):
    """S = 240 000 in one rank and 30 000 in the others, |B| about 2^-6: finite in f16 for all but the largest ranks"""
    y, x, a, b = make(rows, k, rank, dtype)
    x[0] = 0.0
    x[0, 3] = 60000.0
    a[:, 3] = 0.5
    a[0, 3] = 4.0
    b.copy_(b.abs() * 2.0 ** -6)
    ref, tol = formula(y, x, a, b, 1.0)
    finite = check(ops.lora_add(y, x, ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0])), ref, tol)
    assert finite >= (rows if rank <= 40 else rows - 1) * 64


@pytest.mark.parametrize("rank", [5, 24, 200])
@pytest.mark.parametrize("rows,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-6, -1e-3, 64.0, 3e4])
def test_scales_and_rows_of_any_size(dtype, scale, rank, rows, k):
    """S from 2^-24 to 2^24, another size in every row, without a y that hides the update"""
    y, x, a, b = make(rows, k, rank, dtype, seed=7)
    y.zero_()
    i = torch.arange(rows, device="cuda") % 13
    x.copy_(x.float() * 2.0 ** (2 * i - 12)[:, None])
    a.copy_(a.float() * 2.0 ** (12 if scale < 1 else -12))
    ref, tol = formula(y, x, a, b, scale)
    check(ops.lora_add(y, x, ops.AdapterBank([(a, b)], [scale]), ops.AdapterPlan([rows], [0])), ref, tol)


@pytest.mark.parametrize("rank", [5, 24, 200])
@pytest.mark.parametrize("rows,k", SIZES)
def test_infinities_are_the_formulas(rank, rows, k):
    """an infinite rank beside large finite ones of the other sign, where B has a zero for it, and a NaN row"""
    y, x, a, b = make(rows, k, rank, torch.float16, seed=8)
    x[:3, 3] = torch.tensor([float("inf"), -float("inf"), float("nan")], device="cuda")
    x[0, 4] = 60000.0
    a[:, 3] = 0.0
    a[:, 4] = -16.0
    a[0, 3] = 1.0                                       # 0 * inf: NaN in every other rank ...
    o = ops.lora_add(y, x, ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0]))
    assert o[:3].isnan().all() and o[3:].isfinite().all()
    a[:, 3] = 1.0                                       # ... and here none
    b.copy_(b.abs() + 2.0 ** -6)
    b[5] = 0.0
    o = ops.lora_add(y, x, ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0]))
    col = [c for c in range(64) if c != 5]
    assert (o[0, col] == float("inf")).all() and (o[1, col] == -float("inf")).all()
    assert o[:2, 5].isnan().all() and o[2].isnan().all() and o[3:].isfinite().all()
    x[0, 3], x[1, 3] = 60000.0, -60000.0                # the infinities next to finite values of the other sign, rank by rank
    a[1:, 3] = 0.0
    a[0, 4] = 0.0
    ref, tol = formula(y, x, a, b, 1.0)
    o = ops.lora_add(y, x, ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0]))
    check(o[[0, 1] + list(range(3, rows))], ref[[0, 1] + list(range(3, rows))], tol[[0, 1] + list(range(3, rows))])


@pytest.mark.parametrize("rows,k", SIZES)
def test_columns_of_one_buffer(rows, k):
    """x, y and out as column ranges of one buffer; in place beside x"""
    y, x, a, b = make(rows, k, 16, torch.bfloat16, seed=9)
    bank, plan = ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0])
    want = ops.lora_add(y, x, bank, plan)
    buf = torch.cat([y, x, torch.zeros_like(y)], 1)
    y_, x_, out = buf.split([64, k, 64], 1)
    assert ops.lora_add(y_, x_, bank, plan, out=out) is out
    assert torch.equal(out, want) and torch.equal(y_, y) and torch.equal(x_, x)
    assert torch.equal(ops.lora_add(y_, x_, bank, plan, out=y_), want) and torch.equal(x_, x)
    for bad in (buf[:, 64:128], buf[:, 8:72]):
        with pytest.raises(ValueError):
            ops.lora_add(y_, x_, bank, plan, out=bad)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(3, 96), (40, 8224), (8200, 96), (8200, 104)])
def test_an_infinite_weight(dtype, rows, k):
    """A infinite in its last columns, where k ends inside a step of 64: infinity as in the formula, not NaN"""
    y, x, a, b = make(rows, k, 12, dtype, seed=10)
    x.copy_(x.abs() + 0.5)
    b.copy_(b.abs() + 0.5)
    a[3, k - 1] = float("inf")
    a[3, k - 20] = float("inf")
    o = ops.lora_add(y, x, ops.AdapterBank([(a, b)]), ops.AdapterPlan([rows], [0]))
    assert (o == float("inf")).all()


@pytest.mark.parametrize("rank", [24, 200])
@pytest.mark.parametrize("rows,k", SIZES)
def test_f16_on_another_stream_and_in_two_graphs(rank, rows, k):
    """the rows' powers of two are each call's own"""
    y, x, a, b = make(rows, k, rank, torch.float16, seed=11)
    bank, plan = ops.AdapterBank([(a, b)], [3.0]), ops.AdapterPlan([rows], [0])
    base = ops.lora_add(y, x, bank, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        small = ops.lora_add(y, x * 2.0 ** -9, bank, plan)
    other = ops.lora_add(y, x, bank, plan)
    torch.cuda.synchronize()
    assert torch.equal(other, base) and torch.equal(small, ops.lora_add(y, x * 2.0 ** -9, bank, plan))
    xs, graphs, outs = [x.clone(), x * 2.0 ** 6], [], []
    for x_ in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.lora_add(y, x_, bank, plan))
    for i in range(3):
        for x_ in xs:
            x_.mul_(0.5)
        want = [ops.lora_add(y, x_, bank, plan) for x_ in xs]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
