"""Gradients that are stored past the caches: those of which 256 MB do not hold logits and gradient together. They
have the bits of the same rows' gradients in calls that stay below, which go the other way (the numbers that the two
compute are the same, element by element)."""
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import token_loss as T
from dizo_amd.table import dtype_code, stream_handle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
LINE = 256 << 20


@pytest.fixture(params=[1001, 50257, 270001], ids=["short", "held", "long"])
def operands(request):
    """Rows of a vocabulary, a little more than the line; of the two halves each stays below it."""
    def make(dtype):
        v = request.param
        n = LINE // (2 * v * dtype.itemsize) + 24
        g = torch.Generator(device="cuda").manual_seed(v)
        x = (torch.randn(n, v, generator=g, device="cuda") * 3).to(dtype)
        t = torch.randint(0, v, (n,), generator=g, device="cuda")
        t[::7] = -100
        val, at = torch.randn(n, 9, generator=g, device="cuda"), torch.randint(0, v, (n, 9), generator=g, device="cuda")
        at[3::11] = -1
        at[5, 1:4] = at[5, 0]  # named twice and more
        w, u = torch.rand(n, generator=g, device="cuda") + 0.5, torch.rand(n, generator=g, device="cuda") - 0.5
        assert 2 * x.nbytes > LINE and x.nbytes < LINE
        return x, t, w, u, val, at
    return make


def in_halves(f, *tensors):
    n = tensors[0].shape[0] // 2
    a, b = f(*(t[:n] for t in tensors)), f(*(t[n:] for t in tensors))
    return torch.cat([a, b])


def same(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_token_logprobs_gradients_past_the_caches(dtype, operands):
    x, t, w, u, _, _ = operands(dtype)
    want = in_halves(lambda *a: T.token_logprobs_grad(*a)[1], x, t, w, u)
    assert not want.isnan().any() and not want[::7].any() and want[1].any()
    assert same(T.token_logprobs_grad(x, t, w, u)[1], want)
    n, v = x.shape
    out, over = torch.empty(2 * n, device="cuda"), x.clone()
    L.call("dz_token_logprobs", over.data_ptr(), dtype_code(dtype), 1, n, v, 0, v, t.data_ptr(), 0, 1, -100, 0, out.data_ptr(), out[n:].data_ptr(),
           None, None, w.data_ptr(), 0, 1, u.data_ptr(), 0, 1, over.data_ptr(), 0, v, stream_handle())
    assert same(over, want)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distillation_gradients_past_the_caches(dtype, operands):
    x, _, w, _, val, at = operands(dtype)
    want = in_halves(lambda *a: T.topk_distill_grad(*a, temperature=1.7)[1], x, val, at, w)
    assert not want.isnan().any() and not want[3::11].any() and want[0].any()
    assert same(T.topk_distill_grad(x, val, at, w, temperature=1.7)[1], want)
    n, v = x.shape
    out, over = torch.empty(n, device="cuda"), x.clone()
    L.call("dz_topk_distill", over.data_ptr(), dtype_code(dtype), 1, n, v, 0, v, val.data_ptr(), at.data_ptr(), at.shape[1], 1.7, 1, out.data_ptr(),
           w.data_ptr(), 0, 1, over.data_ptr(), 0, v, stream_handle())
    assert same(over, want)
