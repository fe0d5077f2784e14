"""Candidates and answers that share a prompt: the measured cases of dizo_amd.prefix_attention and dizo_amd.sampling.

A case is a dict of plain values. `op` names the call that one pass makes:

  attend   attention of `groups` x `sequences` sequences: each of `length` new tokens reads the `prefix` tokens that its
           group shares, and its own keys up to itself, `slots` of them at most (shared_prefix_attention)
  write    new keys and values put into an 8-bit cache in place (cache_write)
  read     the first `length` tokens of an 8-bit cache as keys and values of a type (cache_read)
  sample   one token a row, by temperature, top-k, top-p and min-p, from given uniform numbers (sample_tokens)

Queries, keys and values come as a model's projections leave them: (batch, token, head, width) in memory. A prompt shorter
than its group's room (`ragged`) has fewer valid keys; what lies behind them is never looked at. `bits` = 8: both key and
value stores are e4m3 codes with a power of two for each token and head.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # candidate answers of 6 tokens, 16 examples x 2 at an OPT-13B layer, prompts of up to 122 tokens: short work, launches count
        _attend("candidates opt-13b fp16", 16, 2, 40, 40, 6, 122, 6, 128, "fp16", ragged=True),
        # the same at an OPT-125m layer in fp32
        _attend("candidates opt-125m fp32", 16, 2, 12, 12, 8, 56, 8, 64, "fp32", ragged=True),
        # the prompts themselves, whole causal sequences of an OPT-2.7B batch: heads of 80
        _attend("prompts opt-2.7b fp16", 16, 1, 32, 32, 256, 0, 256, 80, "fp16"),
        # 32 questions after one prompt of demonstrations: bound by the products
        _attend("questions opt-13b bf16", 1, 32, 40, 40, 61, 2048, 61, 128, "bf16"),
        # 64 answers drawn from one prompt, one token each: single rows against their own keys
        _attend("answers opt-13b fp16", 1, 64, 40, 40, 1, 2048, 256, 128, "fp16"),
        # the same from an 8-bit cache, four query heads to a key head, a long prompt
        _attend("answers 8-bit bf16", 2, 32, 32, 8, 1, 6000, 500, 128, "bf16", bits=8),
        # a prompt of demonstrations goes into the cache
        _cache("write prompt bf16", "write", 1, 40, 2048, 2048, 128, "bf16"),
        # one token of 64 answers
        _cache("write tokens fp16", "write", 64, 40, 1, 160, 128, "fp16"),
        # a kept prompt read back, heads of 80
        _cache("read prompt fp16", "read", 1, 32, 1021, 2048, 80, "fp16"),
        # a batch of answers read back
        _cache("read answers bf16", "read", 64, 40, 300, 320, 128, "bf16"),
        # the next token of one served sequence: latency
        _sample("sample one bf16", 1, 50272, "bf16", 0.7, 50, 0.95, 0.0),
        # nucleus sampling of a large batch, an odd vocabulary
        _sample("sample nucleus fp32", 512, 32003, "fp32", 1.0, 0, 0.9, 0.02),
    ]


def _attend(name, groups, sequences, heads, kv_heads, length, prefix, slots, width, dtype, ragged=False, bits=16):
    return dict(name=name, op="attend", groups=groups, sequences=sequences, heads=heads, kv_heads=kv_heads, length=length, prefix=prefix,
                slots=slots, width=width, dtype=dtype, ragged=ragged, bits=bits)


def _cache(name, op, batch, kv_heads, length, slots, width, dtype):
    return dict(name=name, op=op, batch=batch, kv_heads=kv_heads, length=length, slots=slots, width=width, dtype=dtype)


def _sample(name, rows, vocab, dtype, temperature, top_k, top_p, min_p):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: 1 to 64 sequences, one new token to 2,048, prompts of up to 8,192, heads of 8 to 128
    columns, one to eight query heads to a key head; vocabularies from a character model's to 131,072."""
    op = rng.choice(["attend", "attend", "attend", "write", "read", "sample", "sample"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    width = rng.choice([64, 80, 128, 128, 8 * rng.randrange(1, 17)])
    if op == "attend":
        shared, kv = rng.choice([1, 1, 1, 2, 4, 8]), _log(rng, 1, 40)
        groups, sequences = rng.choice([(1, _log(rng, 1, 64)), (_log(rng, 1, 16), rng.choice([1, 2, 2, 3, 4])), (_log(rng, 1, 4), _log(rng, 1, 16))])
        length = rng.choice([1, 1, rng.randrange(2, 17), _log(rng, 16, 2048)])
        prefix = rng.choice([0, _log(rng, 1, 512), _log(rng, 256, 8192)])
        slots = length + rng.choice([0, 0, _log(rng, 1, 1024)])
        heads = max(1, min(shared * kv, 64) // kv) * kv
        # no more products and no more memory than the largest listed case has
        while groups * sequences * heads * length * (prefix + slots) * width > 2.2e10 * (0.25 if dtype == "fp32" else 1.0) or \
                groups * sequences * heads * length * (prefix + slots) > 1.7e8 or groups * kv * (prefix + sequences * slots) * width > 1.0e8:
            sequences, groups, length, prefix = max(1, sequences // 2), max(1, groups - 1), max(1, length // 2), prefix * 3 // 4
            slots = max(length, slots // 2)
        c = _attend("", groups, sequences, heads, kv, length, prefix, slots, width, dtype, rng.random() < 0.5, rng.choice([16, 16, 8]))
    elif op == "sample":
        vocab = _log(rng, 300, 131072)
        rows = _log(rng, 1, max(1, int(1.6e7 / vocab)))
        c = _sample("", rows, vocab, dtype, rng.choice([1.0, 0.7, round(rng.uniform(0.3, 2.0), 2)]), rng.choice([0, 0, 1, _log(rng, 2, 300)]),
                    rng.choice([1.0, 0.9, round(rng.uniform(0.2, 0.99), 2)]), rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.001, 0.3), 3)]))
    else:
        batch, kv = _log(rng, 1, 64), _log(rng, 1, 40)
        slots = _log(rng, 8, max(9, min(4096, int(6.0e7 / (batch * kv * width)))))
        c = _cache("", op, batch, kv, rng.choice([1, max(1, slots // rng.randrange(1, 9)), rng.randrange(1, slots + 1)]), slots, width, dtype)
    return {k: v for k, v in c.items() if k != "name"}


# ----------------------------------------------------------------- inputs --
def _projected(g, dtype, *shape):
    """A projection's output, (..., token, head, width) in memory, seen as (..., head, token, width)."""
    return torch.randn(*shape[:-3], shape[-2], shape[-3], shape[-1], generator=g, device=DEV).to(DT[dtype]).transpose(-3, -2)


def _quantized(x):
    """8-bit codes with the least power of two for each token and head that leaves no value above 448."""
    m, e = torch.frexp(x.abs().amax(-1).float())
    e = torch.where(m == 0, 0, e - 9 + (m > 0.875).int())
    return torch.ldexp(x.float(), -e.unsqueeze(-1)).to(torch.float8_e4m3fn), torch.ldexp(torch.ones_like(m), e).to(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "attend":
        b, n, h, d, t = case["groups"], case["sequences"], case["kv_heads"], case["width"], case["length"]
        s["q"] = _projected(g, case["dtype"], b, n, case["heads"], t, d).mul_(1.5)
        own_kv = [_projected(g, case["dtype"], b, n, h, case["slots"], d) for _ in range(2)]
        prefix_kv = [_projected(g, case["dtype"], b, h, case["prefix"], d) for _ in range(2)] if case["prefix"] else None
        # a common component in the keys: some tokens are looked at by every query
        own_kv[0] += torch.randn(d, generator=g, device=DEV).to(own_kv[0].dtype)
        if case["bits"] == 8:
            own_kv = sum(map(list, zip(*map(_quantized, own_kv))), [])
            prefix_kv = prefix_kv and sum(map(list, zip(*map(_quantized, prefix_kv))), [])
            own_kv, prefix_kv = [x.contiguous() for x in own_kv], prefix_kv and [x.contiguous() for x in prefix_kv]
        s["own"], s["prefix"] = tuple(own_kv), prefix_kv and tuple(prefix_kv)
        most = case["slots"] - t  # the own tokens that were there before
        s["positions"] = torch.randint(most // 2, most + 1, (b, n), generator=g, device=DEV, dtype=torch.int32)
        s["prefix_lengths"] = None
        if case["ragged"] and case["prefix"]:
            s["prefix_lengths"] = torch.randint(case["prefix"] // 2, case["prefix"] + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
        s["scale"] = 1.0 / math.sqrt(d)
    elif case["op"] == "sample":
        x = torch.randn(case["rows"], case["vocab"], generator=g, device=DEV).mul_(2.0)
        x += torch.rand(case["vocab"], generator=g, device=DEV).add_(1e-4).log_().mul_(-1.0).sub_(1.0)
        x.scatter_add_(1, torch.randint(0, case["vocab"], (case["rows"], 1), generator=g, device=DEV),
                       torch.randn(case["rows"], 1, generator=g, device=DEV).mul_(3.0).add_(6.0))
        s["logits"] = x.to(DT[case["dtype"]])
        s["uniform"] = torch.rand(case["rows"], generator=g, device=DEV)
    else:
        b, h, d, n = case["batch"], case["kv_heads"], case["width"], case["slots"]
        codes = [torch.randn(b, h, n, d, generator=g, device=DEV).mul_(64.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.randint(-9, -5, (b, h, n), generator=g, device=DEV).float().exp2_().to(torch.float8_e8m0fnu) for _ in range(2)]
        s["cache"] = (codes[0], codes[1], scales[0], scales[1])
        if case["op"] == "write":
            s["k"], s["v"] = (_projected(g, case["dtype"], b, h, case["length"], d) for _ in range(2))
            s["positions"] = torch.randint(0, n - case["length"] + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    return s


# ------------------------------------------------------------- plain forms --
def _values(codes, scales):
    return codes.float() * scales.float().unsqueeze(-1)


def _keys_values(kv):
    """Keys and values in 32 bits, of either store."""
    if len(kv) == 4:
        return _values(kv[0], kv[2]), _values(kv[1], kv[3])
    return kv[0].float(), kv[1].float()


def _plain_attend(q, own_kv, prefix_kv, positions, prefix_lengths, scale):
    b, n, heads, t, d = q.shape
    k, v = _keys_values(own_kv)
    h = k.shape[2]
    # (b, n, h, shared heads x t, d): the query heads of one key head side by side
    x = q.float().reshape(b, n, h, heads // h * t, d) * scale
    at = torch.arange(k.shape[3], device=q.device)
    limit = positions.view(b, n, 1, 1, 1) + torch.arange(t, device=q.device).repeat(heads // h).view(1, 1, 1, -1, 1)
    s = torch.where(at <= limit, torch.matmul(x, k.transpose(-1, -2).contiguous()), -math.inf)
    if prefix_kv is not None:
        pk, pv = _keys_values(prefix_kv)
        p = pk.shape[2]
        y = x.transpose(1, 2).reshape(b, h, -1, d)  # the rows of all sequences of a group
        ps = torch.matmul(y, pk.transpose(-1, -2).contiguous())
        if prefix_lengths is not None:
            ps = torch.where(torch.arange(p, device=q.device) < prefix_lengths.view(b, 1, 1, 1), ps, -math.inf)
        s = torch.cat([ps.view(b, h, n, -1, p).transpose(1, 2), s], -1)
    else:
        p = 0
    e = (s - s.amax(-1, keepdim=True)).exp()
    e = e / e.sum(-1, keepdim=True)
    out = torch.matmul(e[..., p:], v)
    if p:
        out = out + torch.matmul(e[..., :p].transpose(1, 2).reshape(b, h, -1, p), pv).view(b, h, n, -1, d).transpose(1, 2)
    return out.reshape(b, n, heads, t, d).to(q.dtype)


def _plain_write(cache, k, v, positions):
    b, h, t, d = k.shape
    seq = torch.arange(b, device=k.device).view(b, 1)
    rows = positions.long().view(b, 1) + torch.arange(t, device=k.device)
    for x, codes, scales in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        c, e = _quantized(x)
        codes.view(torch.uint8).transpose(1, 2)[seq, rows] = c.view(torch.uint8).transpose(1, 2)
        scales.view(torch.uint8).transpose(1, 2)[seq, rows] = e.view(torch.uint8).transpose(1, 2)
    return list(cache)


def _plain_read(cache, length, dtype):
    return [_values(c[:, :, :length], e[:, :, :length]).to(dtype) for c, e in ((cache[0], cache[2]), (cache[1], cache[3]))]


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    x = logits.double()
    w = ((x - x.amax(-1, keepdim=True)) / temperature).exp()
    order = x.sort(dim=-1, descending=True, stable=True).indices
    best = w.gather(-1, order)
    if top_k:
        best = torch.where(torch.arange(x.shape[-1], device=x.device) < top_k, best, 0.0)
    if top_p < 1.0:
        c = best.cumsum(-1)
        best = torch.where(c - best < top_p * c[:, -1:], best, 0.0)
    best = torch.where(best >= min_p, best, 0.0)
    c = torch.zeros_like(w).scatter_(-1, order, best).cumsum(-1)
    return (c <= uniform.double().unsqueeze(-1) * c[:, -1:]).sum(-1)


# -------------------------------------------------------------------- run --
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from dizo_amd import prefix_attention as P
        from dizo_amd import sampling as S

        if op == "attend":
            store = P.QuantizedKV if case["bits"] == 8 else P.KV
            prefix = None if s["prefix"] is None else store(*s["prefix"])
            return [P.shared_prefix_attention(s["q"], store(*s["own"]), prefix, positions=s["positions"], prefix_lengths=s["prefix_lengths"],
                                              scale=s["scale"])]
        if op == "write":
            cache = P.QuantizedKV(*s["cache"])
            P.cache_write(cache, s["k"], s["v"], s["positions"])
            return list(cache)
        if op == "read":
            return list(P.cache_read(P.QuantizedKV(*s["cache"]), case["length"], DT[case["dtype"]]))
        return [S.sample_tokens(s["logits"], s["uniform"], temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"],
                                min_p=case["min_p"])]
    with torch.no_grad():
        if op == "attend":
            return [_plain_attend(s["q"], s["own"], s["prefix"], s["positions"], s["prefix_lengths"], s["scale"])]
        if op == "write":
            return _plain_write(s["cache"], s["k"], s["v"], s["positions"])
        if op == "read":
            return _plain_read(s["cache"], case["length"], DT[case["dtype"]])
        return [_plain_sample(s["logits"], s["uniform"], case["temperature"], case["top_k"], case["top_p"], case["min_p"])]


# ------------------------------------------------------------------- work --
def work(case):
    """Queries, the shared keys once a group, own keys and outputs each once; the products of the keys that a query sees,
    half of the own ones and of a ragged prompt's last half where these are drawn."""
    if case["op"] == "attend":
        size = SIZE[case["dtype"]]
        kv = 2 * case["kv_heads"] * (case["width"] + 1 if case["bits"] == 8 else size * case["width"])
        sequences = case["groups"] * case["sequences"]
        prefix = case["prefix"] * (0.75 if case["ragged"] else 1.0)
        before = (case["slots"] - case["length"]) * 0.75
        queries = sequences * case["heads"] * case["length"] * case["width"]
        return {"bytes": 2 * size * queries + kv * (case["groups"] * prefix + sequences * (before + case["length"])),
                "flops": 4 * queries * (prefix + before + (case["length"] + 1) / 2)}
    if case["op"] == "sample":
        return {"bytes": SIZE[case["dtype"]] * case["rows"] * case["vocab"] + 12 * case["rows"], "flops": 16 * case["rows"] * case["vocab"]}
    values = 2 * case["batch"] * case["kv_heads"] * case["length"]
    return {"bytes": values * (case["width"] * (SIZE[case["dtype"]] + 1) + 1), "flops": values * case["width"] * (3 if case["op"] == "write" else 1)}


# ------------------------------------------------------------------ exact --
def _exact_codes(x):
    """e4m3's nearest value, ties to even: three bits below the leading one, no step below 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))).clamp(min=-6.0) - 3.0)
    return torch.round(x / step) * step


def exact(case, seed):
    """The definitions in 64 bits: softmax over the visible keys by a mask over prefix and own keys laid side by side."""
    if case["op"] == "sample":
        return None  # a token is no computed number
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attend":
            b, n, heads, t, d = s["q"].shape
            wide = [[x.double() for x in kv[:2]] if len(kv) == 2 else [x.double() * e.double().unsqueeze(-1) for x, e in zip(kv[:2], kv[2:])]
                    for kv in (s["own"], s["prefix"]) if kv is not None]
            h = wide[0][0].shape[2]
            out = torch.empty(b, n, heads, t, d, dtype=torch.float64, device=DEV)
            for i in range(b):
                for j in range(n):
                    p = wide[1][0].shape[2] if len(wide) > 1 else 0
                    seen_p = p if s["prefix_lengths"] is None else int(s["prefix_lengths"][i])
                    k, v = (torch.cat([wide[1][x][i, :, :seen_p], wide[0][x][i, j]], 1) if p else wide[0][x][i, j] for x in range(2))
                    k, v = k.repeat_interleave(heads // h, 0), v.repeat_interleave(heads // h, 0)
                    place = torch.arange(k.shape[1], device=DEV)
                    last = (seen_p if p else 0) + int(s["positions"][i, j]) + torch.arange(t, device=DEV)
                    logits = torch.bmm(s["q"][i, j].double(), k.mT.contiguous()) * s["scale"]
                    out[i, j] = torch.bmm(logits.masked_fill(place > last.unsqueeze(-1), -math.inf).softmax(-1), v)
            return [out]
        if case["op"] == "read":
            return [x[:, :, :case["length"]].double().mul_(e[:, :, :case["length"]].double().unsqueeze(-1)) for x, e in zip(s["cache"][:2], s["cache"][2:])]
        codes, scales = [x.double() for x in s["cache"][:2]], [x.double() for x in s["cache"][2:]]
        for i, x in enumerate((s["k"].double(), s["v"].double())):
            e = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 448.0)))
            for j, at in enumerate(s["positions"].tolist()):
                codes[i][j, :, at:at + case["length"]] = _exact_codes(x[j] / e[j].unsqueeze(-1))
                scales[i][j, :, at:at + case["length"]] = e[j]
        return codes + scales
