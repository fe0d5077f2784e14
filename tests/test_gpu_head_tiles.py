"""linear_token_logprobs where a workgroup goes from tile to tile: shapes of more tiles than the card holds workgroups.

The kernels' grids end at the workgroups that are resident at once, 256 or 512; `per` below is how many tiles the
busiest of them then takes. The next tile's rows, head and first slabs are asked for while this one's products
and statistics run, so each shape is run at a width of less than a slab, of whole slabs, with a part of one, and of
one that does not fill 16 bytes; with every row asked for, with some ignored, and with all but a few.

Against 64 bits. Logits are products of width d summed in fp32, off by at most 16 e sqrt(d) |h * w|_2 = x each (partial sums grow as
a walk, a rounding of each step; e = 2^-24), the statistics by what sums of v terms are: log probabilities by
e (4 |lp| + 4 ln v + v / 256 + 60) + 2 x, entropies by e (v / 256 + 60) (1 + ln v) + 2 x (1 + ln v)."""
import math

import pytest
import torch

from dizo_amd import token_loss as T

pytestmark = pytest.mark.gpu

E = 2.0**-24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def operands(n, d, v, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(n, d, generator=g, device="cuda").to(dtype)
    w = torch.randn(v, d, generator=g, device="cuda").mul_(2.5 / math.sqrt(d)).to(dtype)
    return h, w, torch.randint(0, v, (n,), generator=g, device="cuda")


def check(h, w, t, what):
    n, d, v = h.shape[0], h.shape[1], w.shape[0]
    out = T.linear_token_logprobs(h, w, t)
    live = t != -100
    assert (out.logprobs[~live] == 0).all() and (out.entropy[~live] == 0).all(), what
    x = h[live].double() @ w.double().t().contiguous()
    logq = x - x.logsumexp(-1, keepdim=True)
    lp = logq.gather(-1, t[live].unsqueeze(-1)).squeeze(-1)
    entropy = -(logq.exp() * logq).sum(-1)
    off = 2 * 16 * E * math.sqrt(d) * (h[live].double().square() @ w.double().square().t().contiguous()).amax(-1).sqrt()
    lp_tol = E * (4 * lp.abs() + 4 * math.log(v) + v / 256 + 60) + off
    ent_tol = E * (v / 256 + 60) * (1 + math.log(v)) + off * (1 + math.log(v))
    for name, got, want, tol in (("logprobs", out.logprobs, lp, lp_tol), ("entropy", out.entropy, entropy, ent_tol)):
        bad = ~((got[live].double() - want).abs() <= tol)
        assert not bad.any(), (what, name, int(bad.sum()), bad.nonzero()[:4].flatten().tolist(), got[live][bad][:4].tolist(), want[bad][:4].tolist())


# rows, vocabulary: of each kind of tile one that makes two and more a workgroup (the last column: 16-bit types, fp32)
SHAPES = [
    (5, 140000),   # 32 x 256, 552 tiles: per 3
    (50, 140000),  # 64 x 256, 552: per 3
    (50, 30000),   # 64 x 64, 472: per 2
    (100, 140000),  # 128 x 256, 552: per 3; fp32 in parts, 128 x 256
    (600, 50272),  # 256 x 256, 600: per 3; fp32 in parts, 128 x 256, 1,000: per 4
    (2000, 4000),  # 64 x 128, 1,024: per 2
]


@pytest.mark.parametrize("d", [8, 64, 72, 65, 200])
@pytest.mark.parametrize("n, v", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_workgroups_that_take_several_tiles(dtype, n, v, d):
    h, w, t = operands(n, d, v, dtype, n + d + v)
    t[-1] = v - 1
    check(h, w, t, "all rows")
    some = t.clone()
    some[torch.rand(n, generator=torch.Generator().manual_seed(d)) < 0.3] = -100
    some[0] = 0
    check(h, w, some, "some rows")
    few = torch.full_like(t, -100)
    few[n // 2] = t[n // 2]
    few[-1] = v - 1
    check(h, w, few, "few rows")


@pytest.mark.parametrize("d", [64, 65])
@pytest.mark.parametrize("n, v", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_bad_row_stays_in_its_tiles(dtype, n, v, d):
    """A row of NaN or infinities in one tile leaves nothing behind for the tiles that the workgroup takes next."""
    h, w, t = operands(n, d, v, dtype, n + d)
    clean = T.linear_token_logprobs(h, w, t)
    bad = [n // 3, n - 1]
    h[bad[0], 3] = math.nan
    h[bad[1]] = math.inf
    out = T.linear_token_logprobs(h, w, t)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert out.logprobs[bad].isnan().all() and out.entropy[bad].isnan().all()
    assert torch.equal(out.logprobs[keep], clean.logprobs[keep]) and torch.equal(out.entropy[keep], clean.entropy[keep])


@pytest.mark.parametrize("n, v", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_head_rows_that_take_no_part_in_late_tiles(dtype, n, v):
    """Head rows of -inf in the first, a middle and the last tile (hidden states above 0): the rows' statistics are the
    same as of the vocabulary without them, up to the sums' order."""
    d = 64
    h, w, _ = operands(n, d, v, dtype, n + v)
    h = h.abs() + 0.5
    gone = torch.tensor([3, v // 2, v - 2], device="cuda")
    there = torch.ones(v, dtype=torch.bool, device="cuda")
    there[gone] = False
    w0 = w.clone()
    w[gone] = -math.inf
    t = torch.where(there, torch.arange(v, device="cuda"), 0)[torch.arange(n, device="cuda") * (v // n)]
    out = T.linear_token_logprobs(h, w, t)
    x = h.double() @ w0.double().t().contiguous()
    x[:, gone] = -math.inf
    logq = x - x.logsumexp(-1, keepdim=True)
    lp = logq.gather(-1, t.unsqueeze(-1)).squeeze(-1)
    entropy = -torch.where(logq > -math.inf, logq.exp() * logq, 0.0).sum(-1)
    off = 2 * 16 * E * math.sqrt(d) * (h.double().square() @ w0.double().square().t().contiguous()).amax(-1).sqrt()
    assert ((out.logprobs.double() - lp).abs() <= E * (4 * lp.abs() + 4 * math.log(v) + v / 256 + 60) + off).all()
    assert ((out.entropy.double() - entropy).abs() <= (E * (v / 256 + 60) + off) * (1 + math.log(v))).all()
    t[0] = gone[2]
    assert T.linear_token_logprobs(h, w, t).logprobs[0] == -math.inf
