"""The text encoder over packed prompts: the operators of csrc/attn_packed.hip and csrc/lora.hip as they are used together.

Yardstick: the encoder's formula in 64 bits (the oracle's restatement).  The packed path makes the default path's roundings except
two per attention (scores and scores + bias stay fp32), so its error may not exceed the default path's by more than the scatter
of independent roundings: a quarter.  With adapters an output is rounded once more and the update's low-rank product once; the
alternative without the operator, weights merged and rounded to 16 bits, rounds every weight instead: the ratio of the two errors
is at most sqrt(2), the bound 1.5."""
import pytest
import torch

from oracle.f4_ref import Umt5EncoderRef
from turbodiffusion_amd import text_encoder as TE

pytestmark = pytest.mark.gpu
LENS = [1, 77, 300, 0, 33, 150, 5]


def encoder_weights(dim=256, heads=4, layers=2, seed=3):
    sd = TE.synthetic_state_dict(layers=layers, dim=dim, dim_ffn=512, heads=heads, vocab=97, seed=seed, dtype=torch.float32)
    for k in sd:      # position tables and query projections of a size that shapes the attention
        if "pos_embedding" in k:
            sd[k] = sd[k] * 16
        if k.endswith("attn.q.weight"):
            sd[k] = sd[k] * 6
    return sd


def prompts(seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 97, (n,), generator=g) for n in LENS]


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def reference(sd, dtype, ps):
    """each prompt alone, weights of the 16-bit type, arithmetic in 64 bits"""
    ref = Umt5EncoderRef({k: v.to(dtype) for k, v in sd.items()}, dtype=torch.float64, device="cuda")
    return torch.cat([ref(p[None].cuda())[0] for p in ps if p.numel()])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shared_pos", [False, True])
@pytest.mark.parametrize("dim", [256, 512])
def test_packed_prompts_against_the_formula(dtype, shared_pos, dim):
    sd = encoder_weights(dim)
    if shared_pos:
        sd["pos_embedding.embedding.weight"] = sd.pop("blocks.0.pos_embedding.embedding.weight")
        sd = {k: v for k, v in sd.items() if not (k.startswith("blocks") and "pos_embedding" in k)}
    enc, ps = TE.Umt5Encoder(sd, dtype=dtype), prompts()
    want = reference(sd, dtype, ps)
    one = torch.cat([enc(p[None])[0] for p in ps if p.numel()])
    many = enc.encode_packed(ps)
    assert [m.shape[0] for m in many] == LENS
    e1, e2 = rel(one, want), rel(torch.cat(many), want)
    assert e2 <= 1.25 * e1, (e1, e2)
    alone = enc.encode_packed([ps[2]])[0]          # (the projections split K by the number of rows: not the same bits)
    assert rel(alone, reference(sd, dtype, [ps[2]])) <= 1.25 * e1


def test_padded_call_and_the_class_of_the_reference(tmp_path):
    sd = encoder_weights()
    enc = TE.Umt5Encoder(sd, packed=True)
    ps = [p for p in prompts() if 0 < p.numel() <= 160]
    ids = torch.zeros(len(ps), 160, dtype=torch.long)
    mask = torch.zeros_like(ids)
    for i, p in enumerate(ps):
        ids[i, :p.numel()], mask[i, :p.numel()] = p, 1
    out = enc(ids, mask)
    many = enc.encode_packed(ps)
    for i, p in enumerate(ps):
        assert torch.equal(out[i, :p.numel()], many[i]) and not out[i, p.numel():].any()
    with pytest.raises(ValueError):
        enc(ids, mask.flip(1))
    from tokenizers import Tokenizer, models, pre_tokenizers
    tok = Tokenizer(models.WordLevel({"<pad>": 0, "a": 1, "cat": 2, "<unk>": 3}, unk_token="<unk>"))
    tok.pre_tokenizer = pre_tokenizers.Whitespace()
    tok.save(str(tmp_path / "tokenizer.json"))
    texts = ["a cat", "cat cat a cat", "a"]
    got = {p: TE.UMT5EncoderModel(text_len=16, checkpoint_path=sd, tokenizer_path=str(tmp_path), packed=p)(texts) for p in (False, True)}
    assert got[True].shape == (3, 16, 256) and rel(got[True], got[False].double()) < 2.0 ** -5      # a few roundings apart


def adapters_for(encoder, dtype, seed=9):
    g = torch.Generator().manual_seed(seed)
    dim, da, df = encoder.dim, encoder.dim_attn, encoder.dim_ffn
    size = {"attn.q": (da, dim), "attn.k": (da, dim), "attn.v": (da, dim), "attn.o": (dim, da), "ffn.fc2": (dim, df)}
    out = []
    for j, targets in enumerate((("attn.q", "attn.v"), ("attn.q", "attn.k", "attn.v", "attn.o", "ffn.fc2"), ("ffn.fc2",))):
        ad = {}
        for i in range(len(encoder.layers)):
            if j == 2 and i == 0:
                continue
            for t in targets:
                n, k = size[t]
                r = (4, 16, 24)[j]
                ad[f"blocks.{i}.{t}"] = ((torch.randn(r, k, generator=g) * k ** -0.5).to(dtype), (torch.randn(n, r, generator=g) * 0.3 * r ** -0.5).to(dtype))
        out.append(ad)
    return out, [1.0, 0.5, 2.0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_adapter_for_each_prompt(dtype):
    sd = encoder_weights()
    enc, ps = TE.Umt5Encoder(sd, dtype=dtype), prompts()
    ads, scales = adapters_for(enc, dtype)
    bank = TE.Umt5Adapters(enc, ads, scales)
    ids = [1, 0, -1, 2, 1, 2, 0]
    got = enc.encode_packed(ps, bank, ids)
    plain = enc.encode_packed(ps)
    for j in (-1, 0, 1, 2):
        merged = {k: v.to(dtype).double() for k, v in sd.items()}
        if j >= 0:
            for name, (a, b) in ads[j].items():
                merged[name + ".weight"] = merged[name + ".weight"] + scales[j] * b.double() @ a.double()
        mine = [i for i in range(len(ps)) if ids[i] == j and LENS[i]]
        ref = Umt5EncoderRef(merged, dtype=torch.float64, device="cuda")
        want = torch.cat([ref(ps[i][None].cuda())[0] for i in mine])
        base = TE.Umt5Encoder(merged, dtype=dtype)
        e1 = rel(torch.cat([base(ps[i][None])[0] for i in mine]), want)
        e2 = rel(torch.cat([got[i] for i in mine]), want)
        assert e2 <= 1.5 * e1, (j, e1, e2)
        if j >= 0:       # ... and the adapters matter
            assert rel(torch.cat([plain[i] for i in mine]), want) > 10 * e2


def test_encoder_refusals():
    sd = encoder_weights()
    enc = TE.Umt5Encoder(sd)
    ads, scales = adapters_for(enc, torch.bfloat16)
    bank = TE.Umt5Adapters(enc, ads, scales)
    p = [torch.tensor([1, 2, 3])]
    assert [t.shape for t in enc.encode_packed([torch.tensor([], dtype=torch.long)])] == [(0, 256)]
    assert enc.encode_packed([[5, 6]])[0].shape == (2, 256)
    with pytest.raises(ValueError):
        enc.encode_packed(p, bank)
    with pytest.raises(ValueError):
        enc.encode_packed(p, bank, [0, 1])
    for bad in (3, -2):
        with pytest.raises(ValueError):
            enc.encode_packed(p, bank, [bad])
    with pytest.raises(ValueError):
        TE.Umt5Encoder(sd).encode_packed(p, bank, [0])
    with pytest.raises(ValueError):
        TE.Umt5Adapters(enc, [{"blocks.0.ffn.gate.0": ads[0]["blocks.0.attn.q"]}])
    with pytest.raises(ValueError):
        TE.Umt5Adapters(enc, [{"blocks.2.attn.q": ads[0]["blocks.0.attn.q"]}])
    with pytest.raises(ValueError):
        TE.Umt5Adapters(enc, [{"blocks.0.ffn.fc2": ads[0]["blocks.0.attn.q"]}])
    with pytest.raises(ValueError):
        TE.Umt5Adapters(enc, [])
    for bad in (97, -1):
        with pytest.raises(ValueError):
            enc.encode_packed([[1, bad]])
    with pytest.raises(ValueError):                      # heads of 32
        TE.Umt5Encoder(encoder_weights(heads=8)).encode_packed(p)
