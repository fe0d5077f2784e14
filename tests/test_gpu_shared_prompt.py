"""Candidates and answers that share a prompt, on the GPU: the kernels together, as models use them."""
import numpy as np
import pytest
import torch

import _plain
from dizo_amd import shared_prompt as S
from dizo_amd.fused_layers import fuse_forward
from dizo_amd.synth import SHAPES, build_opt, make_batch
from dizo_amd.trainer import ZOArguments, ZOTrainer
from dizo_amd._lib import DzError
from test_shared_prompt import batch, greedy, losses, tiny

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["opt", "llama"])
@pytest.mark.parametrize("candidates, lens", [(2, [1]), (3, [2, 5, 1]), (4, [3])])
def test_losses_are_those_of_whole_sequences(kind, candidates, lens):
    a, b = losses(tiny(kind, device=DEV), batch(len(lens), 3, candidates, lens, 24, device=DEV))
    # fp32 sums of a few hundred terms in another order, through three layers and a mean
    assert abs(a - b) <= 1e-4 * max(1.0, abs(a))


def test_losses_in_16_bits_and_with_fused_layers():
    model = tiny("opt", torch.float16, DEV)
    fuse_forward(model)
    b = batch(9, 4, 2, [3, 2], 40, device=DEV)
    a, c = losses(model, b)
    # a log probability of up to 16 is rounded to half a step of 2^-8, the mean of a few and a difference of two of them to as much
    assert abs(a - c) <= 4 * 2.0**-7


def test_zeroth_order_steps_with_shared_prompts():
    gen = torch.Generator().manual_seed(3)
    seen = {}
    for shared in (False, True):
        np.random.seed(4)
        model = build_opt("opt-tiny", torch.float32, DEV)
        b = make_batch(4, SHAPES["opt-tiny"].vocab, gen=gen.manual_seed(3), device=DEV)
        tr = ZOTrainer(model, ZOArguments(learning_rate=1e-5, max_steps=10, zo_shared_prompt=shared))
        seen[shared] = tr.train([b], 4)
        tr.zo_close()
    assert np.allclose(seen[False], seen[True], rtol=1e-4, atol=1e-5)


def test_captured_steps_are_refused():
    model = build_opt("opt-tiny", torch.float32, DEV)
    with pytest.raises(DzError, match="zo_shared_prompt"):
        ZOTrainer(model, ZOArguments(zo_shared_prompt=True, zo_graph=True))


@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_greedy_answers_are_those_of_whole_forwards(kind):
    model = tiny(kind, device=DEV)
    ids = torch.randint(2, 211, (2, 9), generator=torch.Generator().manual_seed(1)).to(DEV)
    lengths = torch.tensor([9, 4], dtype=torch.int32, device=DEV)
    got = S.generate(model, ids, 6, answers=2, prompt_lengths=lengths, temperature=0.0)
    for i in range(2):
        want = greedy(model, ids[i, :int(lengths[i])], 6)
        assert torch.equal(got[i, 0], want) and torch.equal(got[i, 1], want)


@pytest.mark.parametrize("kv_bits", [16, 8])
@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_drawn_answers_are_those_of_plain_forms(kind, kv_bits, monkeypatch):
    # one run of all four operators: write, read by attention, attend, draw. (fp32: the numbers that the draws go by differ in
    # their last bits, which moves a token where a uniform number is within some 1e-6 of a border; these are not.)
    model = tiny(kind, device=DEV)
    ids = torch.randint(2, 211, (3, 11), generator=torch.Generator().manual_seed(6)).to(DEV)
    lengths = torch.tensor([11, 2, 7], dtype=torch.int32, device=DEV)
    u = torch.rand(3, 5, 12, generator=torch.Generator().manual_seed(8)).to(DEV)
    how = dict(answers=5, prompt_lengths=lengths, uniform=u, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, kv_bits=kv_bits)
    got = S.generate(model, ids, 12, **how)
    for name, f in (("shared_prefix_attention", _plain.attention), ("cache_write", _plain.cache_write), ("sample_tokens", _plain.sample)):
        monkeypatch.setattr(S, name, f)
    want = S.generate(model, ids, 12, **how)
    assert torch.equal(got, want)
    assert len({tuple(x.tolist()) for x in got[0]}) > 1  # the answers differ


def test_generate_is_repeatable_and_takes_a_generator():
    model = tiny("opt", torch.bfloat16, DEV)
    ids = torch.randint(2, 211, (1, 7), generator=torch.Generator().manual_seed(6)).to(DEV)
    runs = [S.generate(model, ids, 9, answers=40, generator=torch.Generator(DEV).manual_seed(3), kv_bits=8) for _ in range(2)]
    assert torch.equal(*runs) and runs[0].min() >= 0 and runs[0].max() < 211


def test_answers_between_steps_are_the_updated_weights():
    """A step that leaves its update for the next perturbation: answers and scores read the weights with it."""
    gen = torch.Generator().manual_seed(5)
    ids = torch.randint(4, 60, (2, 7), generator=gen).to(DEV)
    seen = {}
    for fuse in (False, True):
        np.random.seed(4)
        model = build_opt("opt-tiny", torch.float32, DEV)
        b = make_batch(4, SHAPES["opt-tiny"].vocab, gen=gen.manual_seed(3), device=DEV)
        tr = ZOTrainer(model, ZOArguments(learning_rate=1e-2, zo_eps=0.5, max_steps=10, zo_fuse_restore=fuse, zo_fuse_next_perturb=fuse))
        tr.training_step(b)
        assert (tr._pending_update is not None) == fuse
        answers = S.generate(model, ids, 8, temperature=0.0)
        assert tr._pending_update is None
        tr.training_step(b)
        with torch.no_grad():
            scores = S.shared_prompt_logprobs(model, ids, None, [2, 2], 1, model.config.pad_token_id)
        assert tr._pending_update is None
        tr.zo_close()
        seen[fuse] = answers, scores
    assert torch.equal(seen[False][0], seen[True][0])
    assert torch.equal(seen[False][1], seen[True][1])
