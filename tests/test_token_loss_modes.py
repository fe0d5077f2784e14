"""dizo_amd.token_loss under forward-mode differentiation, without a GPU: the library's calls are replaced by ones
that compute nothing, and host tensors are let through."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from dizo_amd import token_loss as T
from dizo_amd._lib import DzError


class _OnTheGpu(torch.Tensor):
    is_cuda = True


@pytest.fixture
def library(monkeypatch):
    """The names of the entry points that a call reaches."""
    reached = []
    monkeypatch.setattr(T, "_check_logits", lambda what, logits: 0)
    monkeypatch.setattr(T, "_call", lambda device, name, *args: reached.append(name))
    monkeypatch.setattr(T.L, "call", lambda name, *args: reached.append(name))
    return reached


def _operands():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 8, generator=g)
    return dict(x=x, t=torch.tensor([1, -100, 7]), w=torch.ones(3), u=torch.ones(3), val=torch.randn(3, 2, generator=g), at=torch.tensor([[0, 1]] * 3),
                head=torch.randn(8, 8, generator=g))


CALLS = {
    "token_logprobs": (lambda o: T.token_logprobs(o["x"], o["t"]), "x"),
    "token_logprobs_grad": (lambda o: T.token_logprobs_grad(o["x"], o["t"], o["w"], o["u"]), "x", "w", "u"),
    "topk_distill": (lambda o: T.topk_distill(o["x"], o["val"], o["at"]), "x", "val"),
    "topk_distill_grad": (lambda o: T.topk_distill_grad(o["x"], o["val"], o["at"], o["w"]), "x", "val", "w"),
    "linear_token_logprobs": (lambda o: T.linear_token_logprobs(o["x"].as_subclass(_OnTheGpu), o["head"].as_subclass(_OnTheGpu), o["t"]), "x", "head"),
}


@pytest.mark.parametrize("name, operand", [(n, o) for n, c in CALLS.items() for o in c[1:]])
def test_an_operand_with_a_tangent_is_refused(library, name, operand):
    """No result may lack the tangent that its operand has; nor is anything launched for it."""
    call, o = CALLS[name][0], _operands()
    with fwd.dual_level():
        call(o)  # inside a level, without tangents
        assert library, "the call was to reach the library"
        library.clear()
        o[operand] = fwd.make_dual(o[operand], torch.ones_like(o[operand]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(DzError, match="forward-mode"):
                call(o)
    assert not library


@pytest.mark.parametrize("value", [lambda o: T.token_logprobs(o["x"], o["t"]).logprobs, lambda o: T.token_logprobs(o["x"], o["t"]).entropy,
                                   lambda o: T.topk_distill(o["x"], o["val"], o["at"])], ids=["logprobs", "entropy", "distill"])
def test_a_tangent_of_the_upstream_gradient_is_refused(library, value):
    """Forward over reverse: the gradient's tangent would be lost in the backward pass."""
    o = _operands()
    o["x"].requires_grad_(True)
    y = value(o)
    torch.autograd.grad(y, o["x"], torch.ones(3), retain_graph=True)
    with fwd.dual_level(), pytest.raises(DzError, match="forward-mode"):
        torch.autograd.grad(y, o["x"], fwd.make_dual(torch.ones(3), torch.ones(3)))


def test_jvp_raises(library):
    o = _operands()
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: T.token_logprobs(x, o["t"]).logprobs, (o["x"],), (torch.ones_like(o["x"]),))
