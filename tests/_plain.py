"""Plain torch forms of dizo_amd.prefix_attention and sampling for models' tests, on any device, in fp32 or the operands' type."""
import math

import torch

from oracle import prefix as O


def values(store):
    if len(store) == 2:
        return [x.float() for x in store]
    return [c.float() * s.float().unsqueeze(-1) for c, s in zip(store[:2], store[2:])]


def attention(q, own, prefix=None, *, positions=None, prefix_lengths=None, scale=None, out=None):
    groups, sequences, heads, length, width = q.shape
    scale = width ** -0.5 if scale is None else scale
    k, v = values(own)
    h, slots = k.shape[2], k.shape[3]
    x = q.float() * scale
    at = (torch.full((groups, sequences), slots - length, device=q.device) if positions is None else positions).view(groups, sequences, 1, 1, 1)
    seen = torch.arange(slots, device=q.device) <= at + torch.arange(length, device=q.device).view(-1, 1)
    s = (x @ k.repeat_interleave(heads // h, 2).transpose(-1, -2)).masked_fill(~seen, -math.inf)
    v = v.repeat_interleave(heads // h, 2)
    if prefix is not None:
        pk, pv = (t.repeat_interleave(heads // h, 1).unsqueeze(1) for t in values(prefix))
        ps = x @ pk.transpose(-1, -2)
        if prefix_lengths is not None:
            ps = ps.masked_fill(torch.arange(pk.shape[-2], device=q.device) >= prefix_lengths.view(-1, 1, 1, 1, 1), -math.inf)
        s = torch.cat([ps, s], -1)
        v = torch.cat([pv.expand(groups, sequences, *pv.shape[2:]), v], -2)
    y = (torch.softmax(s, -1) @ v).to(q.dtype)
    if out is not None:
        return out.copy_(y)
    return y


def cache_write(cache, k, v, positions):
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        value, power = O.quantize(x, x.dtype == torch.float16)
        codes[..., positions:positions + x.shape[-2], :] = value.to(torch.float32).to(codes.device, codes.dtype)
        scales[..., positions:positions + x.shape[-2]] = power.to(torch.float32).to(scales.device, scales.dtype)


def sample(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows, u = logits.reshape(-1, logits.shape[-1]), uniform.reshape(-1)
    got = [O.sample(rows[i], float(u[i]), temperature, top_k, top_p, min_p) for i in range(rows.shape[0])]
    return torch.tensor(got, device=logits.device).view(logits.shape[:-1])
