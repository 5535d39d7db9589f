"""Speed of the operators that serve the prompts and adapters of many requests at once.

Two operators, each as a program that serves a text encoder or a video model for many requests would call it:

``attention``  softmax attention over packed sequences of different lengths (no padding between them), grouped heads, causal
               or not, with an optional bias by distance; a new token over the keys kept so far is its one-row case.
``adapters``   ``y + scale * (x A^T) B^T`` with another low-rank pair (A, B) for the rows of every request, beside the
               projection that produced ``y`` for all of them.

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the framework's operators.
"""
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_BLOCK = 1 << 28      # scores held at once by the plain form and by ``exact`` (elements)


def _ints(text):
    return [int(w) for w in text.split(",")]


def listed():
    return [
        # a short prompt through one layer of the text encoder (64 heads of 64, bias by distance): latency
        {"name": "attn-prompt-21", "op": "attention", "dtype": "bf16", "heads": 64, "kv_heads": 64, "dim": 64, "causal": False,
         "bias": 128, "fused_qkv": True, "lens": "21", "lens_k": "21"},
        # the prompts of a full batch of requests, from a few words to the encoder's limit of 512 tokens
        {"name": "attn-prompts-24", "op": "attention", "dtype": "bf16", "heads": 64, "kv_heads": 64, "dim": 64, "causal": False,
         "bias": 128, "fused_qkv": True, "lens": "77,226,13,512,5,131,64,40,390,101,19,256,88,31,1,147,512,60,23,119,205,9,300,54",
         "lens_k": "77,226,13,512,5,131,64,40,390,101,19,256,88,31,1,147,512,60,23,119,205,9,300,54"},
        # prompts of a causal model with grouped heads, packed: one long, many short, one of a single token
        {"name": "attn-causal-grouped", "op": "attention", "dtype": "bf16", "heads": 40, "kv_heads": 8, "dim": 128, "causal": True,
         "bias": 0, "fused_qkv": True, "lens": "4099,1,777,2500,64,129,1023,300", "lens_k": "4099,1,777,2500,64,129,1023,300"},
        # one sequence as long as a whole clip's tokens, causal
        {"name": "attn-causal-32760", "op": "attention", "dtype": "bf16", "heads": 12, "kv_heads": 2, "dim": 128, "causal": True,
         "bias": 0, "fused_qkv": False, "lens": "32760", "lens_k": "32760"},
        # the tokens of two clips, each over its own prompt
        {"name": "attn-clips-to-prompts", "op": "attention", "dtype": "f16", "heads": 12, "kv_heads": 12, "dim": 128, "causal": False,
         "bias": 0, "fused_qkv": False, "lens": "32760,18200", "lens_k": "226,37"},
        # one new token of one sequence over a short past: latency
        {"name": "attn-token-777", "op": "attention", "dtype": "bf16", "heads": 12, "kv_heads": 12, "dim": 128, "causal": True,
         "bias": 0, "fused_qkv": False, "lens": "1", "lens_k": "777"},
        # one new token each of sixteen sequences over pasts of very different lengths
        {"name": "attn-tokens-16", "op": "attention", "dtype": "bf16", "heads": 40, "kv_heads": 8, "dim": 128, "causal": True,
         "bias": 0, "fused_qkv": False, "lens": "1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1",
         "lens_k": "32760,1,4096,511,18200,7777,2049,12000,333,27000,64,9001,1500,21000,5000,30011"},
        # one token of one request through one adapter: latency
        {"name": "lora-token", "op": "adapters", "dtype": "bf16", "k": 4096, "n": 4096, "lens": "1", "ids": "0", "ranks": "16"},
        # one token each of 64 requests, sixteen adapters of different ranks, some requests without one
        {"name": "lora-tokens-64", "op": "adapters", "dtype": "bf16", "k": 4096, "n": 12288,
         "lens": ",".join(["1"] * 64), "ids": ",".join(str(i * 7 % 17 - 1) for i in range(64)),
         "ranks": "8,16,64,32,16,16,8,64,24,16,32,4,16,64,48,16"},
        # the q|k|v projection of the text encoder for a batch of prompts, an adapter to each request
        {"name": "lora-prompts-24", "op": "adapters", "dtype": "bf16", "k": 4096, "n": 12288,
         "lens": "77,226,13,512,5,131,64,40,390,101,19,256,88,31,1,147,512,60,23,119,205,9,300,54",
         "ids": "0,1,2,3,4,5,6,7,0,1,2,3,-1,5,6,7,0,1,2,3,4,5,6,7", "ranks": "16,32,64,16,8,64,32,16"},
        # the tokens of a clip through the video model's square projections, the largest width
        {"name": "lora-clip-5120", "op": "adapters", "dtype": "bf16", "k": 5120, "n": 5120, "lens": "32760", "ids": "0", "ranks": "32"},
        # the tokens of two clips through its first feed-forward projection
        {"name": "lora-clips-8960", "op": "adapters", "dtype": "f16", "k": 1536, "n": 8960, "lens": "32760,18200", "ids": "1,0",
         "ranks": "128,64"},
    ]


def _spread(rng, lo, hi):
    """a whole number, spread evenly over the logarithm of [lo, hi]"""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _cut(lens, total):
    """the first of ``lens`` that together stay within ``total``"""
    while sum(lens) > total:
        lens = lens[:-1]
    return lens


def draw(rng):
    dtype = rng.choice(["bf16", "f16"])
    if rng.random() < 0.55:
        case = {"op": "attention", "dtype": dtype}
        kind = rng.choice(["prompts", "causal", "clips", "tokens", "append"])
        if kind == "prompts":
            heads = rng.choice([16, 24, 64])
            lens = [_spread(rng, 1, 512) for _ in range(_spread(rng, 1, 32))]
            case.update(heads=heads, kv_heads=heads, dim=64, causal=False, bias=rng.choice([0, 64, 128]), fused_qkv=True)
            lens_k = lens
        elif kind == "causal":
            kv = rng.choice([1, 2, 4, 8])
            lens = _cut([_spread(rng, 1, 8192) for _ in range(_spread(rng, 1, 12))], 32760)
            case.update(heads=kv * rng.choice([1, 3, 4, 5]), kv_heads=kv, dim=rng.choice([64, 128]), causal=True,
                        bias=rng.choice([0, 0, 128]), fused_qkv=rng.random() < 0.5)
            lens_k = lens
        elif kind == "clips":
            heads = rng.choice([12, 40])
            lens = [_spread(rng, 900, 32760 if heads == 12 else 18200) for _ in range(rng.randint(1, 3))]
            lens_k = [_spread(rng, 1, 512) for _ in lens]
            case.update(heads=heads, kv_heads=heads, dim=128, causal=False, bias=0, fused_qkv=False)
        elif kind == "tokens":
            kv = rng.choice([1, 2, 8])
            lens_k = _cut([_spread(rng, 1, 32760) for _ in range(_spread(rng, 1, 48))], 400000)
            lens = [1] * len(lens_k)
            case.update(heads=kv * rng.choice([1, 4, 5, 8]), kv_heads=kv, dim=rng.choice([64, 128]), causal=True,
                        bias=rng.choice([0, 0, 128]), fused_qkv=False)
        else:   # some new tokens behind a long past
            kv = rng.choice([1, 2, 8])
            lens = [_spread(rng, 2, 700) for _ in range(_spread(rng, 1, 8))]
            lens_k = [m + _spread(rng, 1, 24000) for m in lens]
            case.update(heads=kv * rng.choice([1, 4, 5]), kv_heads=kv, dim=rng.choice([64, 128]), causal=True,
                        bias=0, fused_qkv=False)
        case.update(lens=",".join(map(str, lens)), lens_k=",".join(map(str, lens_k)))
        return case
    k, n = rng.choice([(1536, 1536), (1536, 8960), (8960, 1536), (4096, 4096), (4096, 12288), (10240, 4096), (5120, 5120)])
    adapters = _spread(rng, 1, 24)
    ranks = [rng.choice([4, 8, 13, 16, 32, 64, 128]) for _ in range(adapters)]
    kind = rng.choice(["tokens", "prompts", "clips"])
    if kind == "tokens":
        lens = [1] * _spread(rng, 1, 128)
    elif kind == "prompts":
        lens = [_spread(rng, 1, 512) for _ in range(_spread(rng, 1, 32))]
    else:
        lens = [_spread(rng, 900, 16000) for _ in range(rng.randint(1, 2))]
    ids = [rng.randrange(-1, adapters) if len(lens) > 1 else rng.randrange(adapters) for _ in lens]
    if all(i < 0 for i in ids):
        ids[0] = 0
    return {"op": "adapters", "dtype": dtype, "k": k, "n": n, "lens": ",".join(map(str, lens)), "ids": ",".join(map(str, ids)),
            "ranks": ",".join(map(str, ranks))}


def _attention_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    tq, tk = sum(_ints(case["lens"])), sum(_ints(case["lens_k"]))

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["fused_qkv"]:        # q, k, v are column ranges of one projection's output
        qkv = rand(tq, H + 2 * Hkv, D).to(dt)
        q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    else:
        q, k, v = rand(tq, H, D).to(dt), rand(tk, Hkv, D).to(dt), rand(tk, Hkv, D).to(dt)
    bias = rand(H, 2 * case["bias"] + 1) if case["bias"] else None
    return q, k, v, bias


def _adapter_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    rows, K, N = sum(_ints(case["lens"])), case["k"], case["n"]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    x, y = rand(rows, K).to(dt), rand(rows, N).to(dt)
    pairs = [((rand(r, K) * K ** -0.5).to(dt), (rand(N, r) * 0.5 * r ** -0.5).to(dt)) for r in _ints(case["ranks"])]
    scales = [1.0 + 0.25 * (i % 3) for i in range(len(pairs))]
    return x, y, pairs, scales


def prepare(case, seed):
    state = {"case": case}
    if case["op"] == "attention":
        state["q"], state["k"], state["v"], state["bias"] = _attention_inputs(case, seed)
        if own:
            from turbodiffusion_amd import ops
            state["plan"] = ops.AttentionPlan(_ints(case["lens"]), _ints(case["lens_k"]), heads=case["heads"],
                                              kv_heads=case["kv_heads"], head_dim=case["dim"], causal=case["causal"])
    else:
        state["x"], state["y"], state["pairs"], state["scales"] = _adapter_inputs(case, seed)
        if own:
            from turbodiffusion_amd import ops
            state["bank"] = ops.AdapterBank(state["pairs"], state["scales"])
            state["plan"] = ops.AdapterPlan(_ints(case["lens"]), _ints(case["ids"]))
    return state


def _plain_attention(q, k, v, bias, case):
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    G, R = H // Hkv, case["bias"]
    out = torch.empty(q.shape[0], H, D, dtype=q.dtype, device=q.device)
    q0 = k0 = 0
    for m, n in zip(_ints(case["lens"]), _ints(case["lens_k"])):
        kt = k[k0:k0 + n].float().permute(1, 2, 0).contiguous()             # [Hkv, D, n]
        vs = v[k0:k0 + n].float().transpose(0, 1).contiguous()              # [Hkv, n, D]
        step = max(1, min(m, _BLOCK // (H * max(n, 1))))
        cols = torch.arange(n, device=q.device)
        for a in range(0, m, step):
            b = min(m, a + step)
            rows = torch.arange(a, b, device=q.device) + (n - m)            # the queries are the last m of the n positions
            qs = q[q0 + a:q0 + b].float().view(b - a, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * (b - a), D)
            s = torch.bmm(qs, kt).mul_(D ** -0.5).view(Hkv, G, b - a, n)
            dist = cols[None, :] - rows[:, None]
            if bias is not None:
                s = s + bias.view(Hkv, G, -1)[:, :, dist.clamp(-R, R) + R]
            if case["causal"]:
                s = s.masked_fill(dist > 0, float("-inf"))
            p = torch.exp(s - s.amax(dim=-1, keepdim=True))
            o = torch.bmm(p.view(Hkv, G * (b - a), n), vs).view(Hkv, G, b - a, D) / p.sum(dim=-1, keepdim=True)
            out[q0 + a:q0 + b] = o.permute(2, 0, 1, 3).reshape(b - a, H, D).to(q.dtype)
        q0, k0 = q0 + m, k0 + n
    return out


def _plain_adapters(x, y, pairs, scales, case):
    out = y.clone()
    r0 = 0
    for m, i in zip(_ints(case["lens"]), _ints(case["ids"])):
        if i >= 0:
            a, b = pairs[i]
            s = torch.matmul(x[r0:r0 + m].float(), a.float().t())
            out[r0:r0 + m] = (y[r0:r0 + m].float() + scales[i] * torch.matmul(s, b.float().t())).to(y.dtype)
        r0 += m
    return out


def run(state):
    case = state["case"]
    if case["op"] == "attention":
        if own:
            from turbodiffusion_amd import ops
            return ops.packed_attention(state["q"], state["k"], state["v"], state["plan"], bias=state["bias"])
        return _plain_attention(state["q"], state["k"], state["v"], state["bias"], case)
    if own:
        from turbodiffusion_amd import ops
        return ops.lora_add(state["y"], state["x"], state["bank"], state["plan"])
    return _plain_adapters(state["x"], state["y"], state["pairs"], state["scales"], case)


def exact(case, seed):
    """From the definition, head by head and request by request, in 64 bits."""
    if case["op"] == "attention":
        q, k, v, bias = _attention_inputs(case, seed)
        H, G, D = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
        out = torch.zeros(q.shape[0], H, D, dtype=torch.float64, device=q.device)
        q0 = k0 = 0
        for m, n in zip(_ints(case["lens"]), _ints(case["lens_k"])):
            step = max(1, _BLOCK // 4 // max(n, 1))
            for h in range(H):
                keys, values = k[k0:k0 + n, h // G].double(), v[k0:k0 + n, h // G].double()
                for a in range(0, m, step):
                    b = min(m, a + step)
                    score = torch.mm(q[q0 + a:q0 + b, h].double(), keys.t().contiguous()) / D ** 0.5
                    place = torch.arange(n, device=q.device) - torch.arange(n - m + a, n - m + b, device=q.device).unsqueeze(1)
                    if bias is not None:
                        score += bias[h].double()[torch.clamp(place, -case["bias"], case["bias"]) + case["bias"]]
                    if case["causal"]:
                        score[place > 0] = -float("inf")
                    weight = torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True))
                    out[q0 + a:q0 + b, h] = torch.mm(weight, values)
            q0, k0 = q0 + m, k0 + n
        return out
    x, y, pairs, scales = _adapter_inputs(case, seed)
    out = y.double()
    r0 = 0
    for m, i in zip(_ints(case["lens"]), _ints(case["ids"])):
        if i >= 0:
            low = torch.mm(x[r0:r0 + m].double(), pairs[i][0].double().t().contiguous())
            out[r0:r0 + m] += scales[i] * torch.mm(low, pairs[i][1].double().t().contiguous())
        r0 += m
    return out


def work(case):
    if case["op"] == "attention":
        H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
        lens, lens_k = _ints(case["lens"]), _ints(case["lens_k"])
        pairs = 0
        for m, n in zip(lens, lens_k):
            pairs += m * (n - m) + m * (m + 1) // 2 if case["causal"] else m * n
        return {"bytes": 2 * D * (2 * sum(lens) * H + 2 * sum(lens_k) * Hkv) + 4 * H * (2 * case["bias"] + 1 if case["bias"] else 0),
                "flops": 4 * D * H * pairs}
    K, N = case["k"], case["n"]
    lens, ids, ranks = _ints(case["lens"]), _ints(case["ids"]), _ints(case["ranks"])
    with_adapter = sum(m for m, i in zip(lens, ids) if i >= 0)
    used = sum(ranks[i] for i in set(ids) if i >= 0)
    return {"bytes": 2 * (with_adapter * K + 2 * sum(lens) * N + used * (K + N)),
            "flops": sum(2 * m * ranks[i] * (K + N) for m, i in zip(lens, ids) if i >= 0)}
