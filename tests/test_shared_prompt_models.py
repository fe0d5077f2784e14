"""dizo_amd.shared_prompt without a GPU, model by model: losses and answers are those of whole forwards, or the model is refused.

Every parameter is random, so that nothing a model does with a hidden state, a logit or a position is left at its first value of one
or nothing."""
import pytest
import torch
import transformers

from dizo_amd import shared_prompt as S
from dizo_amd._lib import DzError
from test_shared_prompt import PAD, batch, greedy, losses, plain  # noqa: F401

SMALL = dict(vocab_size=211, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, intermediate_size=96, head_dim=16,
             max_position_embeddings=80, pad_token_id=PAD, bos_token_id=2, eos_token_id=3, is_decoder=True)
OF_TYPE = {
    "opt": dict(ffn_dim=96, word_embed_proj_dim=64),
    "granitemoe": dict(num_local_experts=4, num_experts_per_tok=2), "granitemoeshared": dict(num_local_experts=4, num_experts_per_tok=2),
    "mixtral": dict(num_local_experts=4, num_experts_per_tok=2), "phimoe": dict(num_local_experts=4, num_experts_per_tok=2),
    "minimax_m2": dict(num_local_experts=4, num_experts_per_tok=2), "olmoe": dict(num_experts=4, num_experts_per_tok=2),
    "qwen2_moe": dict(num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32, shared_expert_intermediate_size=32),
    "qwen3_moe": dict(num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32),
    "ernie4_5_moe": dict(moe_num_experts=4, moe_k=2, moe_intermediate_size=32, moe_layer_start_index=0),
    "glm4_moe": dict(n_routed_experts=4, num_experts_per_tok=2, moe_intermediate_size=32, n_group=1, topk_group=1, first_k_dense_replace=1),
    "jetmoe": dict(num_local_experts=4, num_experts_per_tok=2, kv_channels=16), "flex_olmo": dict(num_experts=4, num_experts_per_tok=2),
    "hunyuan_v1_moe": dict(num_experts=4, moe_topk=2), "aria_text": dict(moe_num_experts=4, moe_topk=2),
    "solar_open": dict(n_routed_experts=4, num_experts_per_tok=2, moe_intermediate_size=32, n_group=1, topk_group=1),
    "exaone_moe": dict(num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32, n_group=1, topk_group=1),
    **{kind: dict(num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32) for kind in ("afmoe", "hy_v3", "laguna", "mellum")},
    "gemma2": dict(final_logit_softcapping=None, attn_logit_softcapping=None),
}


def model_of(kind, **how):
    config_class = transformers.models.auto.configuration_auto.CONFIG_MAPPING[kind]
    config = config_class(**{**SMALL, **OF_TYPE.get(kind, {}), **how})
    if getattr(config, "attn_logit_softcapping", 1) is None:
        config._attn_implementation = "eager"
    torch.manual_seed(0)
    model = transformers.AutoModelForCausalLM.from_config(config).eval().float()
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn_like(p) * 0.25 + (p if p.dim() < 2 else 0.0))
    return model


def same(model, b):
    whole, shared = losses(model, b)
    # fp32 sums of a few hundred terms in another order, through two layers of weights of size 1 / 4 and a mean
    return abs(whole - shared) <= 3e-4 * max(1.0, abs(whole))


BATCHES = [(7, 1, 2, [2], 16), (3, 3, 2, [2], 24), (3, 3, 2, [2, 4], 24)]


@pytest.mark.parametrize("kind", sorted(S.MODELS))
def test_prompts_of_one_length(kind, plain):  # noqa: F811
    model = model_of(kind)
    assert same(model, batch(*BATCHES[0]))
    ids = torch.randint(2, 211, (1, 9), generator=torch.Generator().manual_seed(1))
    assert torch.equal(S.generate(model, ids, 6, temperature=0.0)[0, 0], greedy(model, ids[0], 6))


@pytest.mark.parametrize("kind", sorted(S.MODELS))
def test_prompts_of_several_lengths(kind, plain):  # noqa: F811
    model = model_of(kind)
    assert same(model, batch(*BATCHES[1]))
    if kind not in S.COUNT_PADS:
        assert same(model, batch(*BATCHES[2]))


@pytest.mark.parametrize("kind", sorted(S.COUNT_PADS))
def test_prompts_in_other_places_of_models_that_count_padding(kind, plain):  # noqa: F811
    b = batch(*BATCHES[2])  # candidates of 2 and 4 tokens: their prompts start two places apart
    with torch.no_grad():
        got = S.shared_prompt_logprobs(model_of(kind), b["input_ids"], b["attention_mask"], b["option_len"].tolist(), 2, PAD)
    assert torch.equal(torch.isnan(got), torch.tensor([False, True] * 3))


@pytest.mark.parametrize("kind", ["bert", "roberta", "roberta-prelayernorm", "xlm-roberta", "data2vec-text", "modernbert-decoder"])
def test_models_whose_head_is_more_than_an_embedding_are_refused(kind, plain):  # noqa: F811
    model = model_of(kind)
    ids = torch.randint(4, 211, (2, 12), generator=torch.Generator().manual_seed(3))
    for call in (lambda: S.generate(model, ids, 3), lambda: S.shared_prompt_logprobs(model, ids, None, [2, 2], 2, PAD), lambda: losses(model, batch(*BATCHES[0]))):
        with pytest.raises(DzError, match="head"), torch.no_grad():
            call()


def test_a_head_of_several_parts_is_refused(plain):  # noqa: F811
    model = model_of("llama")
    model.norm = torch.nn.LayerNorm(64)
    ids = torch.randint(2, 211, (1, 9), generator=torch.Generator().manual_seed(1))
    with pytest.raises(DzError, match="output embedding"):
        S.generate(model, ids, 2)
    scores = transformers.OPTForSequenceClassification(model_of("opt").config).eval()
    with pytest.raises(DzError, match="output embedding"):
        S.generate(scores, ids, 2)


@pytest.mark.parametrize("how", [{}, dict(layer_types=["sliding_attention", "full_attention"], use_sliding_window=True), dict(layer_types=["full_attention"] * 2),
                                 dict(layer_types=["sliding_attention"] * 2, use_sliding_window=True)], ids=str)
@pytest.mark.parametrize("kind", sorted(S.MODELS))
def test_windows_are_refused_where_they_are_less_than_all_tokens(kind, how, plain):  # noqa: F811
    model = model_of(kind, sliding_window=4, **how)
    ids = torch.randint(2, 211, (1, 9), generator=torch.Generator().manual_seed(1))
    try:
        assert same(model, batch(*BATCHES[0]))
    except DzError as e:
        assert "window" in str(e)
    try:
        assert torch.equal(S.generate(model, ids, 6, temperature=0.0)[0, 0], greedy(model, ids[0], 6))
    except DzError as e:
        assert "window" in str(e)


def test_a_window_of_the_masks_alone_is_refused(plain):  # noqa: F811
    ids = torch.randint(2, 211, (1, 9), generator=torch.Generator().manual_seed(1))
    with pytest.raises(DzError, match="window of 4 of 15 tokens"):
        S.generate(model_of("phimoe", sliding_window=4), ids, 6)
    model = model_of("phimoe", sliding_window=15)
    assert torch.equal(S.generate(model, ids, 6, temperature=0.0)[0, 0], greedy(model, ids[0], 6))


@pytest.mark.parametrize("kind, rope, how", [
    ("llama", dict(rope_type="dynamic", factor=4.0), {}),
    ("llama", dict(rope_type="longrope", factor=4.0, short_factor=[1.0] * 8, long_factor=[4.0] * 8, original_max_position_embeddings=16), dict(max_position_embeddings=64)),
    ("phi3", dict(rope_type="longrope", short_factor=[1.0] * 8, long_factor=[4.0] * 8, original_max_position_embeddings=16),
     dict(max_position_embeddings=64, original_max_position_embeddings=16)),
], ids=["dynamic", "longrope", "phi3"])
def test_rotations_that_change_with_the_length_are_refused_past_it(kind, rope, how, plain):  # noqa: F811
    """Past 16 tokens a whole forward's rotations are others than those of a forward of the prompt, or of fewer tokens."""
    make = lambda: model_of(kind, **{"max_position_embeddings": 16, **how}, rope_parameters=dict(rope, rope_theta=100.0))  # noqa: E731
    assert same(make(), batch(7, 1, 2, [2], 16))
    with pytest.raises(DzError, match="rotations"):
        losses(make(), batch(7, 1, 2, [2], 17))
    ids = torch.randint(2, 211, (1, 12), generator=torch.Generator().manual_seed(1))
    assert torch.equal(S.generate(make(), ids, 4, temperature=0.0)[0, 0], greedy(make(), ids[0], 4))
    with pytest.raises(DzError, match="rotations"):
        S.generate(make(), ids, 5, temperature=0.0)


def test_rotations_of_other_scalings(plain):  # noqa: F811
    model = model_of("llama", rope_parameters=dict(rope_type="yarn", factor=4.0, rope_theta=100.0, original_max_position_embeddings=10), max_position_embeddings=40)
    assert same(model, batch(*BATCHES[2]))


@pytest.mark.parametrize("kind", ["mistral", "phimoe"])
def test_a_window_of_all_tokens_that_are_read_is_none(kind, plain):  # noqa: F811
    assert same(model_of(kind, sliding_window=15), batch(7, 1, 2, [2], 16))  # the last token's logits are not
    with pytest.raises(DzError, match="window"):
        losses(model_of(kind, sliding_window=14), batch(7, 1, 2, [2], 16))
