"""dizo_amd.shared_prompt without a GPU: calls of one model from two places, and what a call leaves behind."""
import copy
import threading

import pytest
import torch

from dizo_amd import shared_prompt as S
from dizo_amd._lib import DzError
from test_shared_prompt import PAD, plain, tiny  # noqa: F401

IDS = torch.randint(2, 211, (2, 9), generator=torch.Generator().manual_seed(3))


def inside(model, call):
    """What `call` does while an answer of the model is being drawn."""
    got = []

    def hook(*_):
        if not got:
            try:
                got.append(call())
            except DzError as e:
                got.append(e)

    handle = model.base_model.register_forward_pre_hook(hook)
    answers = S.generate(model, IDS, 3, temperature=0.0)
    handle.remove()
    return answers, got[0]


def scores(model):
    with torch.no_grad():
        return S.shared_prompt_logprobs(model, IDS, None, [2, 2], 1, PAD)


@pytest.mark.parametrize("call", [lambda m: S.generate(m, IDS, 2), scores])
def test_a_second_call_of_a_model_is_refused(call, plain):  # noqa: F811
    model = tiny("opt")
    want, before = S.generate(model, IDS, 3, temperature=0.0), model.config._attn_implementation
    answers, second = inside(model, lambda: call(model))
    assert isinstance(second, DzError) and "not through" in str(second)
    assert torch.equal(answers, want) and model.config._attn_implementation == before
    call(model)  # and taken afterwards


def test_a_second_call_from_another_thread_is_refused(plain):  # noqa: F811
    model = tiny("opt")
    seen = []

    def other():
        try:
            S.generate(model, IDS, 2)
        except DzError as e:
            seen.append(str(e))

    def start():
        t = threading.Thread(target=other)
        t.start()
        t.join()

    inside(model, start)
    assert len(seen) == 1 and "not through" in seen[0]


def test_another_model_may_be_called_meanwhile(plain):  # noqa: F811
    model, other = tiny("opt"), tiny("llama")
    want = S.generate(other, IDS, 2, temperature=0.0)
    assert torch.equal(inside(model, lambda: S.generate(other, IDS, 2, temperature=0.0))[1], want)
    twin = copy.deepcopy(model)
    twin.config = model.config  # (its layers have a config of their own, which model's call would not reach)
    assert isinstance(inside(model, lambda: S.generate(twin, IDS, 2))[1], DzError)


def test_a_call_that_fails_leaves_the_model_free(plain, monkeypatch):  # noqa: F811
    model = tiny("opt")
    monkeypatch.setattr(S, "sample_tokens", lambda *a, **k: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        S.generate(model, IDS, 2)
    assert torch.isfinite(scores(model)).all()


def test_parts_of_a_model_in_evaluation_stay_there(plain):  # noqa: F811
    model = tiny("opt")
    model.train()
    model.config.dropout = model.config.attention_dropout = 0.0
    model.base_model.decoder.layers[1].eval()
    before = [m.training for m in model.modules()]
    S.generate(model, IDS, 2, temperature=0.0)
    assert [m.training for m in model.modules()] == before
