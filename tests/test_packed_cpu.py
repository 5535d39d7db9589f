"""Host side of the packed operators: the work tables replayed row by row, and refusals that need no GPU."""
import ctypes
import random

import pytest
import torch

from turbodiffusion_amd import _lib as L
from turbodiffusion_amd import ops, packed


def attention_table(lq, lk, heads, kv_heads, causal):
    a, b, c = packed._i64_array(lq), packed._i64_array(lk), (ctypes.c_int64 * 6)()
    L.call("td_attn_packed_plan", a, b, len(lq), heads, kv_heads, causal, None, 0, c)
    n = sum(c[:3])
    t = torch.full((n + 1, 8), -7, dtype=torch.int32)
    L.call("td_attn_packed_plan", a, b, len(lq), heads, kv_heads, causal, ctypes.c_void_p(t.data_ptr()), n, c)
    assert (t[n] == -7).all()
    return t[:n].tolist(), list(c)


@pytest.mark.parametrize("seed", range(8))
def test_attention_plan_covers_every_visible_key_once(seed):
    rng = random.Random(seed)
    for _ in range(25):
        ns, kv = rng.randint(0, 6), rng.choice([1, 2, 3])
        G = rng.choice([1, 2, 5, 40])
        lq = [rng.choice([0, 1, 2, 31, 33, 127, 129, 300]) for _ in range(ns)]
        lk = [rng.choice([0, 1, 63, 64, 65, 128, 700, 5000]) for _ in range(ns)]
        causal = rng.randint(0, 1)
        t, (tiles, few, joins, ws_rows, tq, tk) = attention_table(lq, lk, kv * G, kv, causal)
        assert (tq, tk) == (sum(lq), sum(lk))
        starts = {sum(lq[:s]): s for s in range(ns) if lq[s]}
        seen = {}
        for i, (token, head0, rows, pos, kb, a, b, slot) in enumerate(t[:tiles + few]):
            qb = max(x for x in starts if x <= token)
            s = starts[qb]
            row0 = (token - qb) * G + head0
            assert kb == sum(lk[:s]) and 0 <= head0 < G and pos == token - qb + lk[s] - lq[s] and 0 <= a <= b <= lk[s]
            assert rows == min(128 if i < tiles else 32, lq[s] * G - row0) > 0
            for row in range(row0, row0 + rows):
                seen.setdefault((s, row), []).append((a, b, slot))
        for s in range(ns):
            for row in range(lq[s] * G):
                end = min(lk[s], max(0, row // G + lk[s] - lq[s] + 1)) if causal else lk[s]
                parts, at = sorted(seen.pop((s, row))), 0
                for a, b, slot in parts:
                    assert a == at and (slot >= 0) == (len(parts) > 1)
                    at = b
                assert end <= at <= lk[s]
        assert not seen
        slots = [j[3] + i * j[5] for j in t[tiles + few:] for i in range(j[4])]
        rows = [x + r for j in t[tiles + few:] for x in range(j[3], j[3] + j[4] * j[5], j[5]) for r in range(j[5])]
        assert sorted(slots) == sorted(x[7] for x in t[:tiles + few] if x[7] >= 0)
        assert len(set(rows)) == len(rows) and (not rows or max(rows) < ws_rows)


@pytest.mark.parametrize("kv", [1, 3, 8, 12, 40, 300])
def test_attention_plan_splits_long_pasts(kv):
    """one new token over up to 2^30 keys: ranges of at least 256 keys (but a sequence's last), no shorter part before a longer one,
    enough workgroups where there are keys for them; no split while no sequence has more than 1024 keys"""
    for lk in ([1024] * 3, [1, 1024, 129], [1025], [32760], [8000] * 8, [32760, 1, 129, 20011, 777], [8000] * 256, [1 << 30], [1 << 29, 300, 1 << 28]):
        t, (tiles, few, joins, ws_rows, tq, tk) = attention_table([1] * len(lk), lk, kv, kv, 1)
        assert tiles == 0 and few >= len(lk)
        items = sorted(t[:few])
        for s, n in enumerate(lk):
            parts = [x for x in items if x[0] == s]
            assert [x[5] for x in parts] == [0] + [x[6] for x in parts[:-1]] and parts[-1][6] == n
            assert all(x[6] - x[5] >= 256 and (x[6] - x[5]) % 128 == 0 for x in parts[:-1])
            assert len(parts) == 1 or max(lk) > 1024
        sizes = [x[6] - x[5] for x in t[:few]]
        assert sizes == sorted(sizes, reverse=True)
        if max(lk) > 1024 and sum(lk) * kv >= 256 * 1024:
            assert few * kv >= 176


def test_attention_plan_refusals():
    with pytest.raises(ValueError):
        ops.AttentionPlan([3, 4], [3], heads=2)
    with pytest.raises(ValueError):
        ops.AttentionPlan([3], heads=5, kv_heads=2)
    with pytest.raises(ValueError):
        ops.AttentionPlan([3], heads=2, head_dim=96)
    with pytest.raises(ValueError):
        ops.AttentionPlan([2.5], heads=2)
    with pytest.raises(ValueError):
        ops.AttentionPlan(torch.tensor([2.0]), heads=2)
    with pytest.raises(L.TurboDiffusionAMDError):
        ops.AttentionPlan([-1], heads=2)
    with pytest.raises(L.TurboDiffusionAMDError):
        ops.AttentionPlan([1 << 31], heads=2)
    with pytest.raises(L.TurboDiffusionAMDError):
        ops.AttentionPlan([1 << 30, 1 << 30], heads=2)
    with pytest.raises(ValueError):
        ops.AttentionPlan([3], heads=2, device="cpu")
    with pytest.raises(ValueError):
        ops.AttentionPlan([(1 << 64) + 3], heads=2)          # would be 3 in 64 bits
    with pytest.raises(ValueError):
        ops.AdapterPlan([3], [(1 << 64) - 1])                # would be -1


def test_attention_refuses_cpu_tensors():
    class Plan:
        heads, kv_heads, head_dim, device = 2, 2, 64, torch.device("cuda", 0)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(L.TurboDiffusionAMDError):
        ops.packed_attention(q, q, q, Plan())


@pytest.mark.parametrize("seed", range(4))
def test_adapter_plan_takes_every_row_once(seed):
    rng = random.Random(seed)
    for _ in range(40):
        ns = rng.randint(0, 9)
        lens = [rng.choice([0, 1, 2, 31, 32, 33, 300, 5000]) for _ in range(ns)]
        ids = [rng.randint(-1, 3) for _ in range(ns)]
        a, b, c = packed._i64_array(lens), packed._i64_array(ids), (ctypes.c_int64 * 6)()
        L.call("td_lora_plan", a, b, ns, None, 0, c)
        n = 4 * (c[0] + c[1]) + c[2]
        t = torch.full((n + 1,), -7, dtype=torch.int32)
        L.call("td_lora_plan", a, b, ns, ctypes.c_void_p(t.data_ptr()), n, c)
        assert t[n] == -7
        t = t.tolist()
        owner = [i for m, i in zip(lens, ids) for _ in range(m)]
        assert list(c)[2:5] == [len(owner), sum(i >= 0 for i in owner), max(ids, default=-1) + 1]
        perm, seen = t[4 * (c[0] + c[1]):n], []
        for j in range(c[0] + c[1]):
            p0, rows, adapter, _ = t[4 * j:4 * j + 4]
            assert 1 <= rows <= c[5] and (adapter >= 0) == (j < c[0])
            if adapter >= 0:
                assert p0 + rows <= c[3]           # rows of the fp32 workspace
            assert all(owner[r] == adapter for r in perm[p0:p0 + rows])
            seen += perm[p0:p0 + rows]
        assert sorted(seen) == list(range(len(owner)))


def test_adapter_refusals():
    a, b = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(24, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.AdapterPlan([3], [0, 1])
    with pytest.raises(L.TurboDiffusionAMDError):
        ops.AdapterPlan([3], [-2])
    with pytest.raises(L.TurboDiffusionAMDError):
        ops.AdapterPlan([-3], [0])
    with pytest.raises(ValueError):
        ops.AdapterBank([])
    with pytest.raises(ValueError):
        ops.AdapterBank([(a, b)], scales=[1.0, 2.0])
    with pytest.raises(ValueError):
        ops.AdapterBank([(a, b)], scales=[float("nan")])
    with pytest.raises(TypeError):
        ops.AdapterBank([(a.float(), b.float())])
    with pytest.raises(TypeError):
        ops.AdapterBank([(a, b), (a.half(), b.half())])
    with pytest.raises(ValueError):
        ops.AdapterBank([(a, b[:, :3])])
    with pytest.raises(ValueError):
        ops.AdapterBank([(a[:, :12], b)])
    with pytest.raises(ValueError):
        ops.AdapterBank([(a, b)], device="cpu")


def test_adapter_workspace_of_every_plan():
    """no rows with an adapter need no workspace, nor do calls small enough for one launch; otherwise at least one 16-bit part of
    every such row"""
    for tiles, rows, tile in ((0, 0, 32), (1, 1, 32), (5, 150, 32), (200, 6400, 32), (32, 8192, 256), (600, 600 * 256, 256)):
        c = (ctypes.c_int64 * 6)(tiles, 0, rows, rows, 1, tile)
        for k in (8, 64, 4096, 10240):
            for n in (8, 4096, 12288):
                for rank in (8, 16, 24, 256):
                    out = ctypes.c_int64(-1)
                    L.call("td_lora_workspace", c, k, n, rank, ctypes.byref(out))
                    few = tile == 32 and rank <= 64 and k <= 4096 and tiles * -(-n // 256) <= 256
                    assert out.value == 0 if rows == 0 or few else out.value >= rows * rank // 2
    with pytest.raises(L.TurboDiffusionAMDError):
        L.call("td_lora_workspace", c, 64, 64, 257, ctypes.byref(out))


@pytest.mark.parametrize("bidirectional", [True, False])
def test_relative_bias_is_the_table_by_bucket(bidirectional):
    from turbodiffusion_amd.text_encoder import relative_buckets
    table = torch.arange(32 * 3, dtype=torch.float32).view(32, 3)
    v = ops.relative_bias(table, max_dist=128, bidirectional=bidirectional)
    assert v.shape == (3, 257) and v.dtype == torch.float32 and v.is_contiguous()
    if bidirectional:
        b = relative_buckets(300, 32, 128, "cpu")
        rel = (torch.arange(300)[None, :] - torch.arange(300)[:, None]).clamp(-128, 128)
        for h in range(3):
            assert torch.equal(v[h][rel + 128], table[b][:, :, h])
    else:
        near = [int(v[0, 128 - d]) // 3 for d in range(16)]
        assert near == list(range(16)) and (v[:, 128:] == table[0][:, None]).all() and (v[:, 0] == table[31]).all()
        assert (v[0, :129].diff() <= 0).all()                       # further back: never a smaller bucket
    with pytest.raises(ValueError):
        ops.relative_bias(table[0])
    with pytest.raises(ValueError):
        ops.relative_bias(table, max_dist=4)
