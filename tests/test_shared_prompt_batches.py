"""dizo_amd.shared_prompt without a GPU: batches whose candidates do not have one prompt take the loss of whole sequences."""
import pytest
import torch

from dizo_amd import shared_prompt as S
from dizo_amd._lib import DzError
from dizo_amd.trainer import ZOArguments, ZOTrainer, forward_wrap_with_option_len
from test_shared_prompt import PAD, batch, plain, tiny  # noqa: F401
from test_shared_prompt_models import model_of


def cut(seed, prompt, lens, most):
    """[prompt | candidate] of one example, cut from the left to `most` tokens and padded to the longest."""
    g = torch.Generator().manual_seed(seed)
    head = torch.randint(2, 211, (prompt,), generator=g)
    rows = [torch.cat([head, torch.randint(2, 211, (n,), generator=g)])[-most:] for n in lens]
    length = max(map(len, rows))
    ids, mask = torch.full((len(rows), length), PAD), torch.zeros(len(rows), length, dtype=torch.long)
    for i, r in enumerate(rows):
        ids[i, length - len(r):] = r
        mask[i, length - len(r):] = 1
    return {"input_ids": ids, "attention_mask": mask, "labels": torch.zeros(len(rows), dtype=torch.long), "option_len": torch.tensor(lens),
            "num_options": torch.full((len(rows),), len(rows))}


def whole_and(model, how, b):
    out = []
    for shared in (False, how):
        model.dz_shared_prompt = shared
        with torch.inference_mode():
            out.append(float(forward_wrap_with_option_len(model, **b, return_dict=True).loss))
    return out


@pytest.mark.parametrize("how", [True, "or whole"])
@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_sequences_cut_from_the_left(kind, how, plain):  # noqa: F811
    a, c = whole_and(tiny(kind), how, cut(1, 20, [2, 4], 16))
    assert a == c
    a, c = whole_and(tiny(kind), how, cut(1, 20, [3, 3], 16))  # cut alike
    assert a != c and abs(a - c) <= 1e-4 * max(1.0, abs(a))


@pytest.mark.parametrize("how", [True, "or whole"])
def test_masks_of_another_form(how, plain):  # noqa: F811
    model = tiny("opt")
    b = batch(4, 2, 2, [2], 16)
    b["attention_mask"][1, 8] = 0  # a token in the middle
    a, c = whole_and(model, how, b)
    assert a == c
    b = batch(4, 2, 2, [5], 16)
    b["attention_mask"][0, :12] = 0  # a prompt of no token
    a, c = whole_and(model, how, b)
    assert a == c or (a != a and c != c)


@pytest.mark.parametrize("how", [True, "or whole"])
@pytest.mark.parametrize("kind", sorted(S.COUNT_PADS))
def test_prompts_in_other_places_of_models_that_count_padding(kind, how, plain):  # noqa: F811
    a, c = whole_and(model_of(kind), how, batch(3, 3, 2, [2, 4], 24))
    assert a == c


def test_prompts_of_other_tokens(plain):  # noqa: F811
    b = batch(4, 2, 2, [2, 3], 16)
    b["input_ids"][1, 12] = 5 if b["input_ids"][1, 12] != 5 else 6
    a, c = whole_and(tiny("opt"), "or whole", b)
    assert a == c


@pytest.mark.parametrize("attention_mask", [True, False])
def test_shares_prompts(attention_mask):
    model = tiny("opt")
    b = batch(4, 2, 2, [2, 3], 16)
    mask = b["attention_mask"]
    if not attention_mask:
        b = cut(1, 13, [3, 3], 16)
        mask = None
    ids, lens = b["input_ids"], b["option_len"].tolist()
    assert S.shares_prompts(model, ids, mask, lens, 2)
    ids[1, 9] = 212 - ids[1, 9]
    assert not S.shares_prompts(model, ids, mask, lens, 2)
    assert S.shares_prompts(model, ids, mask, lens, 2, tokens=False)
    assert not S.shares_prompts(model, ids, torch.ones(len(lens), 1, 1, 16), lens, 2, tokens=False)
    lens[1] += 1
    assert not S.shares_prompts(model, ids, mask, lens, 2, tokens=False)


def test_the_trainers_option_takes_any_batch(plain):  # noqa: F811
    seen = {}
    for shared in (False, True):
        model = tiny("opt")
        b = batch(4, 2, 2, [2], 16)
        b["input_ids"][1, 12] = 5 + int(b["input_ids"][1, 12] == 5)  # not the other candidate's prompt
        trainer = ZOTrainer(model, ZOArguments(zo_shared_prompt=shared))
        seen[shared] = float(trainer.zo_forward(model, b))
        trainer.zo_close()
    assert seen[False] == seen[True]


@pytest.mark.parametrize("shape", [(4, 1, 16, 16), (4, 15), (16,)])
def test_a_mask_of_another_shape_is_refused(shape):
    b = batch(4, 2, 2, [2, 3], 16)
    with pytest.raises(DzError, match="attention_mask"), torch.no_grad():
        S.shared_prompt_logprobs(tiny("opt"), b["input_ids"], torch.ones(shape), b["option_len"].tolist(), 2, PAD)
