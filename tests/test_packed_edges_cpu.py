"""Host side of the packed operators: checks of arguments that need no GPU."""
import ctypes
import random

import pytest
import torch

from turbodiffusion_amd import _lib as L
from turbodiffusion_amd import packed


def shared(a, b):
    """from the elements' addresses"""
    def where(t):
        at = torch.zeros(t.shape, dtype=torch.int64)
        for d, (n, st) in enumerate(zip(t.shape, t.stride())):
            at += (torch.arange(n) * st * t.element_size()).view([-1 if i == d else 1 for i in range(t.dim())])
        return {t.data_ptr() + x + i for x in at.flatten().tolist() for i in range(t.element_size())}
    return bool(where(a) & where(b))


def test_overlap_of_slices_of_one_buffer():
    buf = torch.zeros(12, 10, 24, dtype=torch.bfloat16)
    assert not packed._overlap(buf[:, :4], buf[:, 4:8])                   # heads of a fused projection
    assert not packed._overlap(buf[:, :4], buf[:, 4:])
    assert not packed._overlap(buf[..., :8], buf[..., 8:16])              # columns of every head
    assert not packed._overlap(buf[1:11, 2:6, :16], buf[1:11, 2:6, 16:])
    assert not packed._overlap(buf[0::2], buf[1::2])                      # every other row
    assert not packed._overlap(buf.transpose(0, 1)[:3], buf.transpose(0, 1)[3:])
    assert not packed._overlap(buf[:6], buf[6:])
    assert not packed._overlap(buf[:0], buf)
    flat = buf.view(12, 240)
    assert not packed._overlap(flat[:, :64], flat[:, 64:128])
    assert packed._overlap(flat[:, :64], flat[:, 63:128])
    assert packed._overlap(buf, buf) and packed._overlap(buf[:, :4], buf[:, 3:8]) and packed._overlap(buf[:7], buf[6:])
    assert packed._overlap(buf[..., :16], buf[..., 8:])
    assert packed._overlap(buf[3:4, 2:3, :1].expand(5, 4, 8), buf)


def test_overlap_is_never_missed():
    rng, found = random.Random(0), [0, 0]
    buf = torch.zeros(1000, dtype=torch.float16)
    for _ in range(4000):
        ts = []
        for _ in range(2):
            size = [rng.choice([1, 1, 2, 3, 4]) for _ in range(rng.choice([2, 3]))]
            stride = [rng.choice([0, 1, 2, 4, 8, 12, 24, 30, 48, 96]) for _ in size]
            ts.append(torch.as_strided(buf, size, stride, rng.randrange(24)))
        if shared(*ts):
            found[0] += 1
            assert packed._overlap(*ts)
        else:
            found[1] += not packed._overlap(*ts)
    assert min(found) > 250


def test_a_scale_past_fp32_is_refused():
    """finite as Python holds it, infinite as the kernels do: the update of zero would be NaN"""
    a, b = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(24, 4, dtype=torch.bfloat16)
    for scale in (1e39, -1e300, float("inf")):
        with pytest.raises(ValueError, match="scales must be finite"):
            packed.AdapterBank([(a, b)], [scale])


@pytest.mark.parametrize("kw", [{"heads": 2.5}, {"heads": 4, "kv_heads": 1.5}, {"heads": float("nan")}, {"heads": float("inf")}, {"heads": 1 << 31}])
def test_numbers_of_heads_are_whole(kw):
    with pytest.raises(ValueError, match="heads"):
        packed.AttentionPlan([3], **kw)


@pytest.mark.parametrize("n", [float("inf"), float("nan"), 2.5, True])
def test_lengths_are_whole(n):
    for make in (lambda: packed.AttentionPlan([3, n], heads=2), lambda: packed.AttentionPlan([3, 4], [4, n], heads=2),
                 lambda: packed.AdapterPlan([n], [0]), lambda: packed.AdapterPlan([3], [n])):
        with pytest.raises(ValueError, match="whole numbers"):
            make()


def test_rows_of_out_may_not_overlap_at_the_c_entry():
    """refused before anything is launched (the addresses are not memory)"""
    counts = (ctypes.c_int64 * 6)(1, 0, 3, 3, 1, 32)
    for ldo in (0, 56):
        with pytest.raises(L.TurboDiffusionAMDError, match="overlap"):
            L.call("td_lora_add", 4096, 64, 8192, 64, 16384, ldo, L.TD_BF16, 64, 64, 4096, 4096, 1, 8, 4096, counts, 4096, None)


def test_a_table_for_both_kernels_is_refused():
    """a batch is one kernel's; refused before anything is launched"""
    counts, strides = (ctypes.c_int64 * 6)(1, 1, 0, 0, 2, 2), (ctypes.c_int64 * 8)(*[128, 64] * 4)
    with pytest.raises(L.TurboDiffusionAMDError, match="counts"):
        L.call("td_attn_packed", 4096, 8192, 16384, 32768, strides, L.TD_BF16, 2, 2, 64, 1.0, 0, None, 0, 4096, counts, None, None)


@pytest.mark.parametrize("n,buckets,max_dist", [(5, 64, 10), (8, 32, 8), (16, 64, 16), (40, 32, 128), (300, 32, 128)])
def test_buckets_that_widen_nowhere(n, buckets, max_dist):
    """as many single distances as max_dist or more: the encoder's table for prompts shorter than that is one bucket a distance"""
    from turbodiffusion_amd.text_encoder import relative_buckets
    got, half = relative_buckets(n, buckets, max_dist, "cpu"), buckets // 2
    rel = torch.arange(n)[None, :] - torch.arange(n)[:, None]
    near = rel.abs() < half // 2
    assert torch.equal(got[near], (rel.abs() + half * (rel > 0))[near])
    if max_dist <= half // 2:
        assert near.all()
        with pytest.raises(ValueError, match="widen"):
            packed.relative_bias(torch.zeros(buckets, 2), max_dist)          # its table ends at max_dist, where buckets would differ
