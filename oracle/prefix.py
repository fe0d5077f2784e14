"""64-bit definitions of dizo_amd.prefix_attention and dizo_amd.sampling, one row at a time, on the CPU."""
from __future__ import annotations

import math

import torch


def attend(q, own, prefix, positions, prefix_lengths, scale):
    """Attention of (groups, sequences, heads, length, width) queries. own, prefix: (k, v) of values, or None.

    Returns (out, spread, reach) in float64: the result, sum_j w_j |v_j| / sum_j w_j (what roundings of weights and products are
    taken of), and per query the largest scale sum_d |q_d k_d| (what roundings of scores are taken of)."""
    q = q.detach().cpu().double()
    groups, sequences, heads, length, width = q.shape
    stores = [None if s is None else [x.detach().cpu().double() for x in s] for s in (own, prefix)]
    own, prefix = stores
    kv_heads = (own or prefix)[0].shape[-3]
    slots = own[0].shape[-2] if own else 0
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(q.shape[:-1], dtype=torch.float64)
    for g in range(groups):
        seen_prefix = 0
        if prefix:
            p = prefix[0].shape[-2]
            seen_prefix = p if prefix_lengths is None else min(max(int(prefix_lengths[g]), 0), p)
        for n in range(sequences):
            at = slots - length if positions is None else int(positions[g, n])
            for h in range(heads):
                kh = h * kv_heads // heads
                for t in range(length):
                    seen = min(max(at + t + 1, 0), slots)
                    k = [prefix[0][g, kh, :seen_prefix]] if seen_prefix else []
                    v = [prefix[1][g, kh, :seen_prefix]] if seen_prefix else []
                    if seen:
                        k.append(own[0][g, n, kh, :seen])
                        v.append(own[1][g, n, kh, :seen])
                    if not k:
                        continue
                    k, v = torch.cat(k), torch.cat(v)
                    w = torch.softmax(scale * (k @ q[g, n, h, t]), 0)
                    out[g, n, h, t] = w @ v
                    spread[g, n, h, t] = w @ v.abs()
                    reach[g, n, h, t] = scale * (k.abs() @ q[g, n, h, t].abs()).max()
    return out, spread, reach


def code_value(code: int) -> float:
    """e4m3: a sign, four bits of exponent (bias 7), three of fraction; no infinities, NaN where all seven are set."""
    e, f = code >> 3 & 15, code & 7
    if code & 127 == 127:
        return math.nan
    x = math.ldexp(8 + f, e - 10) if e else math.ldexp(f, -9)
    return -x if code & 128 else x


CODE_VALUES = torch.tensor([code_value(c) for c in range(256)], dtype=torch.float64)


def quantize(x, half: bool):
    """(codes' values, powers of two) of rows (..., width): the nearest code of x / 2^e, ties to the even one."""
    x = x.detach().cpu().double()
    fine = torch.isfinite(x).all(-1)
    if half:
        x = x.clamp(-61440.0, 61440.0)
    most = torch.where(fine.unsqueeze(-1), x, 0.0).abs().amax(-1)
    e = torch.zeros(most.shape, dtype=torch.float64)
    for i, m in enumerate(most.view(-1).tolist()):
        if m > 0:
            p = -100
            while m > 448.0 * 2.0**p:
                p += 1
            e.view(-1)[i] = p
    y = x / torch.exp2(e).unsqueeze(-1)
    positive = CODE_VALUES[:127]  # ascending
    a = y.abs()
    hi = torch.searchsorted(positive, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = positive[hi] - a, a - positive[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    value = torch.where(y < 0, -positive[pick], positive[pick])
    value[~fine] = math.nan
    return value, torch.exp2(e)


def kept_weights(row, temperature, top_k, top_p, min_p):
    """[(token, weight), ...] in the order of the vocabulary, of a row of float64 logits with a distribution."""
    x = row.tolist()
    m = max(x)
    if temperature == 0:
        top_k, temperature = 1, 1.0

    def weight(v):
        if m == math.inf:
            return 1.0 if v == math.inf else 0.0
        return math.exp((v - m) / temperature) if v > -math.inf else 0.0

    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    w = [(i, weight(x[i])) for i in order if x[i] > -math.inf]
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1.0:
        total, before, n = math.fsum(v for _, v in w), 0.0, 0
        sums = []
        for _, v in w:
            if n and before >= top_p * total:
                break
            n += 1
            sums.append(v)
            before = math.fsum(sums) if n < 64 else before + v
        w = w[:n]
    w = [(i, v) for i, v in w if v >= min(min_p, 1.0)]
    return sorted(w)


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> int:
    row = row.detach().cpu().double()
    if torch.isnan(row).any() or row.max() == -math.inf or not 0 <= u <= 1:
        return -1
    w = kept_weights(row, temperature, top_k, top_p, min_p)
    target, c = u * math.fsum(v for _, v in w), 0.0
    best = -1
    for i, v in w:
        c += v
        if v > 0:
            best = i
        if c > target:
            return i
    return best
