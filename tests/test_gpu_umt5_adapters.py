"""Umt5Adapters: every projection has a bank of the pairs that name it, and those alone.

Yardstick as for the packed encoder: the formula in 64 bits with merged weights, against the default path with merged weights rounded
to 16 bits; one more rounding of an output and one of the low-rank product against one of every weight: a ratio of at most
sqrt(2), the bound 1.5."""
import pytest
import torch

from oracle.f4_ref import Umt5EncoderRef
from turbodiffusion_amd import text_encoder as TE

pytestmark = pytest.mark.gpu
LENS = [40, 3, 77, 12]


def encoder_weights(seed=3):
    sd = TE.synthetic_state_dict(layers=2, dim=256, dim_ffn=512, heads=4, vocab=97, seed=seed, dtype=torch.float32)
    return {k: v * (16 if "pos_embedding" in k else 6 if k.endswith("attn.q.weight") else 1) for k, v in sd.items()}


def pairs(targets, rank, dtype, seed, blocks=(0, 1)):
    g = torch.Generator().manual_seed(seed)
    return {f"blocks.{i}.{t}": ((torch.randn(rank, 512 if t == "ffn.fc2" else 256, generator=g) / 16).to(dtype),
                                (torch.randn(256, rank, generator=g) * 0.3 * rank ** -0.5).to(dtype)) for i in blocks for t in targets}


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ranks", [(128, 96), (256, 1)])
def test_large_ranks_on_q_k_and_v(dtype, ranks):
    sd = encoder_weights()
    enc = TE.Umt5Encoder(sd, dtype=dtype)
    g = torch.Generator().manual_seed(5)
    ps = [torch.randint(0, 97, (n,), generator=g) for n in LENS]
    ads, scales = [pairs(("attn.q", "attn.k", "attn.v"), ranks[0], dtype, 1), pairs(("attn.k", "attn.o"), ranks[1], dtype, 2)], [0.5, 2.0]
    ids = [0, 1, -1, 0]
    got = enc.encode_packed(ps, TE.Umt5Adapters(enc, ads, scales), ids)
    for j in (-1, 0, 1):
        merged = {k: v.to(dtype).double() for k, v in sd.items()}
        for name, (a, b) in (ads[j] if j >= 0 else {}).items():
            merged[name + ".weight"] = merged[name + ".weight"] + scales[j] * b.double() @ a.double()
        mine = [i for i in range(len(ps)) if ids[i] == j]
        ref, base = Umt5EncoderRef(merged, dtype=torch.float64, device="cuda"), TE.Umt5Encoder(merged, dtype=dtype)
        want = torch.cat([ref(ps[i][None].cuda())[0] for i in mine])
        e1 = rel(torch.cat([base(ps[i][None])[0] for i in mine]), want)
        assert rel(torch.cat([got[i] for i in mine]), want) <= 1.5 * e1


def test_a_projection_that_an_adapter_does_not_name_is_left_alone():
    """banks hold the adapters that name a projection; a row of another adapter keeps what the shared projection gave it, whatever
    the activations are: zero pairs would make infinite ones NaN"""
    enc = TE.Umt5Encoder(encoder_weights(), dtype=torch.float16)
    ads = [pairs(("attn.q",), 8, torch.float16, 1), pairs(("attn.v", "ffn.fc2"), 4, torch.float16, 2, blocks=(1,)), pairs(("attn.q",), 16, torch.float16, 3, blocks=(1,))]
    bank = TE.Umt5Adapters(enc, ads, [1.0, 3.0, 2.0])
    assert [{t: (b.ranks, place) for t, (b, place) in blk.items()} for blk in bank.banks] == [
        {"attn.q": ([8], [0, -1, -1])},
        {"attn.q": ([8, 16], [0, -1, 1]), "attn.v": ([4], [-1, 0, -1]), "ffn.fc2": ([4], [-1, 0, -1])}]
    seen = []

    def add(y, x, bank_, plan, out=None):
        seen.append((tuple(y.shape), plan.ids))
        return real(y, x, bank_, plan, out=out)

    real = TE.lora_add
    ps = [torch.arange(5), torch.arange(7), torch.arange(3)]
    plain = enc.encode_packed(ps)
    TE.lora_add = add
    try:
        got = enc.encode_packed(ps, bank, [1, -1, 2])
        assert [s[1] for s in seen] == [[-1, -1, 1], [0, -1, -1], [0, -1, -1]] and all(s[0] == (15, 256) for s in seen)
        for same in (torch.tensor([1, -1, 2], device="cuda"), [1.0, -1.0, 2.0]):
            assert all(torch.equal(a, b) for a, b in zip(enc.encode_packed(ps, bank, same), got))
        seen.clear()
        assert all(torch.equal(a, b) for a, b in zip(enc.encode_packed(ps, bank, [-1, -1, -1]), plain)) and not seen
    finally:
        TE.lora_add = real
    assert torch.equal(got[1], plain[1]) and not torch.equal(got[0], plain[0]) and not torch.equal(got[2], plain[2])


def test_refusals():
    enc = TE.Umt5Encoder(encoder_weights())
    ad = pairs(("attn.q",), 8, torch.bfloat16, 1)
    for scales in ([1.0], [1.0, 2.0, 3.0]):
        with pytest.raises(ValueError):
            TE.Umt5Adapters(enc, [ad, ad], scales)
    with pytest.raises(ValueError):
        TE.Umt5Adapters(enc, [pairs(("attn.k",), 257, torch.bfloat16, 1)])
    with pytest.raises(ValueError):
        enc.encode_packed([[1, 2]], TE.Umt5Adapters(enc, [ad]), [0.5])
