"""dizo_amd.shared_prompt without a GPU: the losses and answers of packed forwards against those of whole ones, with the
kernels' plain forms in their place."""
import pytest
import torch

import _plain
from dizo_amd import shared_prompt as S
from dizo_amd._lib import DzError
from dizo_amd.trainer import forward_wrap_with_option_len

PAD = 1


def tiny(kind, dtype=torch.float32, device="cpu"):
    from transformers import LlamaConfig, LlamaForCausalLM, OPTConfig, OPTForCausalLM

    torch.manual_seed(5)
    if kind == "opt":
        m = OPTForCausalLM(OPTConfig(vocab_size=211, hidden_size=64, num_hidden_layers=3, num_attention_heads=4, ffn_dim=96, max_position_embeddings=80,
                                     word_embed_proj_dim=64, pad_token_id=PAD, init_std=0.2))
    else:
        m = LlamaForCausalLM(LlamaConfig(vocab_size=211, hidden_size=64, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, intermediate_size=96,
                                         max_position_embeddings=80, pad_token_id=PAD, initializer_range=0.2))
    return m.eval().to(dtype).to(device)


def batch(seed, examples, candidates, lens, length, device="cpu"):
    """Left-padded sequences [prompt | candidate], with prompts of several lengths."""
    g = torch.Generator()
    g.manual_seed(seed)
    ids = torch.full((examples * candidates, length), PAD)
    mask = torch.zeros_like(ids)
    for e in range(examples):
        prompt = torch.randint(2, 211, (int(torch.randint(1, length - max(lens), (1,), generator=g)) if e else length - max(lens),), generator=g)
        for c in range(candidates):
            n = lens[(e * candidates + c) % len(lens)]
            row = torch.cat([prompt, torch.randint(2, 211, (n,), generator=g)])
            ids[e * candidates + c, length - len(row):] = row
            mask[e * candidates + c, length - len(row):] = 1
    option_len = torch.tensor([lens[i % len(lens)] for i in range(examples * candidates)])
    right = torch.randint(0, candidates, (examples,), generator=g).repeat_interleave(candidates)
    return {"input_ids": ids.to(device), "attention_mask": mask.to(device), "labels": right.to(device), "option_len": option_len,
            "num_options": torch.full((examples * candidates,), candidates)}


def losses(model, b):
    out = []
    for shared in (False, True):
        model.dz_shared_prompt = shared
        with torch.inference_mode():
            out.append(float(forward_wrap_with_option_len(model, **b, return_dict=True).loss))
    return out


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(S, "shared_prefix_attention", _plain.attention)
    monkeypatch.setattr(S, "cache_write", _plain.cache_write)
    monkeypatch.setattr(S, "sample_tokens", _plain.sample)


@pytest.mark.parametrize("kind", ["opt", "llama"])
@pytest.mark.parametrize("candidates, lens", [(2, [1]), (2, [3]), (3, [2, 5, 1]), (1, [4]), (4, [1, 2])])
def test_losses_are_those_of_whole_sequences(plain, kind, candidates, lens):
    a, b = losses(tiny(kind), batch(len(lens), 3, candidates, lens, 24))
    # fp32 sums of a few hundred terms in another order, through three layers and a mean
    assert abs(a - b) <= 1e-4 * max(1.0, abs(a))


def test_without_a_mask(plain):
    b = batch(7, 1, 2, [2], 16)
    b.pop("attention_mask")
    a, c = losses(tiny("opt"), b)
    assert abs(a - c) <= 1e-4


def test_other_batches_run_as_before(plain, monkeypatch):
    model = tiny("opt")
    b = batch(3, 2, 2, [2], 16)
    b["num_options"] = torch.tensor([3, 3, 3, 1])  # not the same number for all
    monkeypatch.setattr(S, "shared_prompt_logprobs", lambda *a: pytest.fail("taken"))
    b["num_options"] = torch.tensor([3, 1])
    a, c = losses(model, b)
    assert a == c
    b = batch(3, 2, 2, [2], 16)
    b["option_len"] = torch.tensor([0, 2, 2, 2])
    a, c = losses(model, b)
    assert a == c


def test_candidates_of_other_prompts_give_nan(plain):
    b = batch(4, 2, 2, [2, 3], 16)
    b["input_ids"][1, 12] = 5 if b["input_ids"][1, 12] != 5 else 6
    _, c = losses(tiny("opt"), b)
    assert c != c


def test_attention_of_the_model_is_put_back(plain):
    model = tiny("opt")
    before = model.config._attn_implementation
    b = batch(4, 2, 2, [2], 16)
    losses(model, b)
    assert model.config._attn_implementation == before
    model.config._attn_implementation = S.ATTN_IMPL
    with pytest.raises(DzError), torch.no_grad():
        model(input_ids=b["input_ids"])


def greedy(model, prompt, n):
    ids = prompt.view(1, -1)
    for _ in range(n):
        with torch.no_grad():
            ids = torch.cat([ids, model(input_ids=ids).logits[:, -1:].argmax(-1)], 1)
    return ids[0, prompt.numel():]


@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_greedy_answers_are_those_of_whole_forwards(plain, kind):
    model = tiny(kind)
    g = torch.Generator()
    g.manual_seed(1)
    ids = torch.randint(2, 211, (2, 9), generator=g)
    lengths = torch.tensor([9, 4], dtype=torch.int32)
    got = S.generate(model, ids, 6, answers=2, prompt_lengths=lengths, temperature=0.0, generator=g)
    for i in range(2):
        want = greedy(model, ids[i, :lengths[i]], 6)
        assert torch.equal(got[i, 0], want) and torch.equal(got[i, 1], want)


def test_an_answer_repeats_its_end(plain):
    model = tiny("opt")
    ids = torch.randint(2, 211, (1, 5), generator=torch.Generator().manual_seed(2))
    free = S.generate(model, ids, 8, temperature=0.0)
    end = int(free[0, 0, 2])
    got = S.generate(model, ids, 8, temperature=0.0, eos_token_id=end)[0, 0].tolist()
    first = got.index(end)
    assert got[first:] == [end] * (8 - first) and got[:first] == free[0, 0, :first].tolist()


@pytest.mark.parametrize("how", [dict(kv_bits=4), dict(answers=0), dict(prompt_lengths=torch.tensor([3])), dict(uniform=torch.zeros(1, 1, 3))])
def test_generate_refuses(how):
    with pytest.raises(DzError):
        S.generate(None, torch.zeros(1, 3, dtype=torch.long), 2, **how)


def test_logprobs_refuse():
    with pytest.raises(DzError, match="autograd"):
        S.shared_prompt_logprobs(None, torch.zeros(2, 4), None, [1, 1], 2, PAD)
    with torch.no_grad():
        for lens, n in (([1, 1], 3), ([4, 1], 2), ([0, 1], 2), ([1], 2)):
            with pytest.raises(DzError):
                S.shared_prompt_logprobs(None, torch.zeros(2, 4, dtype=torch.long), None, lens, n, PAD)


def test_prompts_without_a_token_of_their_own(plain):
    """An option as long as the sequence, and one that reaches into the padding: no answer, and no position outside of the model's."""
    b = batch(4, 2, 2, [5], 16)
    b["attention_mask"][:2] = 0
    b["attention_mask"][0, 11:] = 1  # five tokens, all of the option
    b["attention_mask"][1, 11:] = 1
    b["attention_mask"][2:] = 0  # none
    with torch.no_grad():
        got = S.shared_prompt_logprobs(tiny("opt"), b["input_ids"], b["attention_mask"], [5] * 4, 2, PAD)
    assert torch.isnan(got).all()


def refused(model, match, **how):
    ids = torch.randint(2, 211, (2, 12), generator=torch.Generator().manual_seed(3))
    with pytest.raises(DzError, match=match):
        S.generate(model, ids, 3, **how)
    with pytest.raises(DzError, match=match), torch.no_grad():
        S.shared_prompt_logprobs(model, ids, None, [2, 2], 2, PAD)


def other(kind, **how):
    import transformers

    small = dict(vocab_size=211, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, intermediate_size=96, head_dim=16,
                 max_position_embeddings=80, pad_token_id=PAD)
    return getattr(transformers, kind + "ForCausalLM")(getattr(transformers, kind + "Config")(**small, **how)).eval()


def test_models_of_other_attention_are_refused(plain):
    from transformers import BloomConfig, BloomForCausalLM

    refused(BloomForCausalLM(BloomConfig(vocab_size=211, hidden_size=64, n_layer=2, n_head=4)), "by name")
    refused(other("Mistral", sliding_window=4), "window")
    refused(other("Gemma2", final_logit_softcapping=None), "soft cap")
    refused(other("Gemma2", attn_logit_softcapping=None), "final_logit_softcapping")
    model = tiny("llama")
    model.config.num_hidden_layers = 4  # as if a layer mixed tokens in another way
    refused(model, "3 of 4 layers")
    model = tiny("llama")
    model.model.layers[1].self_attn.layer_idx = 0
    refused(model, "layer_idx")


def test_a_window_that_holds_all_tokens_is_none(plain):
    model = other("Mistral", sliding_window=64)
    ids = torch.randint(2, 211, (1, 7), generator=torch.Generator().manual_seed(4))
    assert torch.equal(S.generate(model, ids, 4, temperature=0.0)[0, 0], greedy(model, ids[0], 4))


def test_answers_end_with_the_models_positions(plain):
    model = tiny("opt")  # of 80 positions
    ids = torch.randint(2, 211, (1, 75), generator=torch.Generator().manual_seed(5))
    assert S.generate(model, ids, 6, temperature=0.0).shape == (1, 1, 6)
    with pytest.raises(DzError, match="positions"):
        S.generate(model, ids, 7, temperature=0.0)


def test_a_model_in_training_stays_there(plain):
    model = tiny("opt")
    model.train()
    model.config.dropout = model.config.attention_dropout = 0.0
    ids = torch.randint(2, 211, (1, 5), generator=torch.Generator().manual_seed(6))
    S.generate(model, ids, 2, temperature=0.0)
    assert model.training and all(m.training for m in model.modules())
