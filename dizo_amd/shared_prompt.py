"""Candidates and answers of a shared prompt through an HF causal language model, on the kernels of prefix_attention and
sampling.

``shared_prompt_logprobs``  what the option-masked loss reads (trainer.py:1466-1500), with each example's prompt
                            computed once instead of once for every candidate. ZOArguments.zo_shared_prompt makes the
                            zeroth-order forwards use it (model.dz_shared_prompt)
``generate``                answers drawn from prompts, several from each (trainer.py:1544-1568): a prompt is computed
                            once, its keys and values are kept once for all of its answers, in the model's dtype or in
                            8 bits, and each answer keeps its own

Both run the model's own layers, OPT's, LLaMA's or others of MODELS, which call the attention HF registers by name, with one of this
module's in its place (in the model's config, for as long as a forward takes: one call at a time for a model, a second one is refused): a forward gets
one row for each prompt, and the attention is told where things lie by the keyword argument dz_shared. Other models,
attention with a window, a soft cap or sinks, layers that mix tokens in another way, and heads that do more than multiply by the
output embedding are refused. Nothing is recorded by autograd.
"""
from __future__ import annotations

import contextlib
import threading
from typing import Optional, Union

import torch

from ._lib import DzError
from .prefix_attention import KV, QuantizedKV, cache_write, shared_prefix_attention
from .sampling import sample_tokens

ATTN_IMPL = "dizo_shared_prompt"
_registered = False
_lock = threading.Lock()
_running = set()  # the configs (by id, while a call holds them) whose attention is exchanged


@contextlib.contextmanager
def _alone(model):
    """One call at a time for a model, or for models of one config: a second one would put the first one's attention back as the
    model's own, and take it out of evaluation in the middle of an answer."""
    config = model.config
    with _lock:
        if id(config) in _running or config._attn_implementation == ATTN_IMPL:
            raise DzError(f"shared_prompt: another call of this {type(model).__name__} is not through")
        _running.add(id(config))
    try:
        yield
    finally:
        with _lock:
            _running.discard(id(config))


class _Candidates:
    """One forward over rows [prompt | candidate 0 | candidate 1 | ...]: prompts of up to `room` tokens, left-aligned,
    `each` tokens of every candidate."""

    def __init__(self, room: int, candidates: int, each: int, lengths: torch.Tensor):
        self.room, self.candidates, self.each, self.lengths = room, candidates, each, lengths
        self.keys, self.seen = room + each, set()  # keys that a query sees at most, and the layers that this forward has been through

    def attend(self, layer, q, k, v, scale):
        p, n, t = self.room, self.candidates, self.each
        out = q.new_empty(q.shape[0], q.shape[2], q.shape[1], q.shape[3])
        prompt = KV(k[:, :, :p], v[:, :, :p])
        shared_prefix_attention(q[:, :, :p].unsqueeze(1), KV(prompt.k.unsqueeze(1), prompt.v.unsqueeze(1)), scale=scale,
                                out=out[:, :p].unsqueeze(1).transpose(2, 3))
        if t:
            q, k, v = (x[:, :, p:].unflatten(2, (n, t)).transpose(1, 2) for x in (q, k, v))
            shared_prefix_attention(q, KV(k, v), prompt, prefix_lengths=self.lengths, scale=scale,
                                    out=out[:, p:].unflatten(1, (n, t)).transpose(2, 3))
        return out


class _Answers:
    """Forwards that draw `answers` answers of up to `room` tokens from each prompt: first the prompts, then one token of
    every answer at a time."""

    def __init__(self, prompts: int, answers: int, input_room: int, room: int, lengths: torch.Tensor, bits: int):
        self.prompts, self.answers, self.room, self.lengths, self.bits = prompts, answers, room, lengths, bits
        self.keys, self.seen = input_room + room, set()  # as above
        self.prefix, self.own = {}, {}  # of each layer
        self.at = None  # the answers' tokens that were there before this forward's; None: the prompts'

    def attend(self, layer, q, k, v, scale):
        out = q.new_empty(q.shape[0], q.shape[2], q.shape[1], q.shape[3])
        if self.at is None:
            shape = (self.prompts, self.answers, k.shape[1], self.room, k.shape[3])
            if self.bits == 8:
                self.prefix[layer] = QuantizedKV.empty(*k.shape, device=k.device)
                cache_write(self.prefix[layer], k, v, 0)
                self.own[layer] = QuantizedKV.empty(*shape, device=k.device)
            else:
                self.prefix[layer] = KV(k.contiguous(), v.contiguous())
                self.own[layer] = KV(k.new_empty(shape), v.new_empty(shape))
            shared_prefix_attention(q.unsqueeze(1), KV(k.unsqueeze(1), v.unsqueeze(1)), scale=scale, out=out.unsqueeze(1).transpose(2, 3))
            return out
        q, k, v = (x.unflatten(0, (self.prompts, self.answers)) for x in (q, k, v))
        own = self.own[layer]
        if self.bits == 8:
            cache_write(own, k, v, self.at)
        else:
            own.k[:, :, :, self.at:self.at + 1] = k
            own.v[:, :, :, self.at:self.at + 1] = v
        own = type(own)(*(x[:, :, :, :self.at + 1] for x in own))
        shared_prefix_attention(q, own, self.prefix[layer], prefix_lengths=self.lengths, scale=scale,
                                out=out.unflatten(0, (self.prompts, self.answers)).transpose(2, 3))
        return out


def _attention(module, query, key, value, attention_mask=None, scaling=None, dropout=0.0, dz_shared=None, sliding_window=None,
               softcap=None, s_aux=None, **kwargs):
    if dz_shared is None:
        raise DzError(f"{ATTN_IMPL} runs inside of shared_prompt's forwards only")
    if dropout or softcap is not None or s_aux is not None or not getattr(module, "is_causal", True):
        raise DzError("shared_prompt: attention with dropout, a soft cap or sinks, or that isn't causal")
    if sliding_window is not None and sliding_window < dz_shared.keys:
        raise DzError(f"shared_prompt: attention with a window of {sliding_window} of {dz_shared.keys} tokens")
    layer = getattr(module, "layer_idx", None)
    if layer is None or layer in dz_shared.seen:
        raise DzError(f"shared_prompt: {type(module).__name__} without a number of its own (layer_idx)")
    dz_shared.seen.add(layer)
    scale = query.shape[-1] ** -0.5 if scaling is None else scaling
    return dz_shared.attend(layer, query, key, value, scale), None


# Types of models (config.model_type) that are no more than layers of the attention above, one for each of config.num_hidden_layers, and
# an output embedding: nothing else mixes tokens, and nothing lies between the last hidden states and the head, or behind it.
MODELS = frozenset("""afmoe apertus arcee aria_text bitnet ctrl cwm ernie4_5 ernie4_5_moe exaone4 exaone_moe flex_olmo gemma gemma2
    gemma3_text glm glm4 glm4_moe gpt2 gpt_bigcode gpt_neox granite granitemoe granitemoeshared helium hunyuan_v1_dense hunyuan_v1_moe hy_v3
    hyperclovax jais2 jetmoe laguna llama mellum minimax_m2 ministral ministral3 mistral mixtral olmo olmo2 olmo3 olmoe opt persimmon phi
    phi3 phimoe qwen2 qwen2_moe qwen3 qwen3_moe seed_oss smollm3 solar_open starcoder2""".split())


# Of these, the ones to which more than the distance between two tokens matters (a vector for each position, or a norm of rotated keys
# by channel) and that count the padding on a sequence's left, too, where they are given no positions. (OPT takes positions from the mask.)
COUNT_PADS = frozenset(("ctrl", "gpt2", "gpt_bigcode", "hunyuan_v1_dense", "hunyuan_v1_moe"))


def _check_model(model, tokens: int, seen: int) -> None:
    """Whether the model's answers to sequences of up to `tokens`, of which one of those that are read sees `seen`, are what its layers
    and output embedding give here."""
    config = model.config
    if not getattr(model, "_supports_attention_backend", False):
        raise DzError(f"shared_prompt: {type(model).__name__} does not call an attention that HF registers by name")
    if getattr(config, "model_type", None) not in MODELS:
        raise DzError(f"shared_prompt: {type(model).__name__} is not one of the models whose head and layers are known: {', '.join(sorted(MODELS))}")
    head, base = model.get_output_embeddings(), model.base_model
    if not isinstance(head, torch.nn.Module) or base is model or any(m is not head and m is not base for m in model.children()):
        raise DzError(f"shared_prompt: {type(model).__name__} has more than its layers and an output embedding")
    for name in ("final_logit_softcapping", "logit_scale", "logits_scaling", "output_multiplier_scale"):
        if getattr(config, name, None) not in (None, 1, 1.0):
            raise DzError(f"shared_prompt: a model with {name}")
    # (some models have a window in their masks only, which the attention is not told of)
    for name in ("sliding_window", "attention_chunk_size"):
        window = getattr(config, name, None)
        if window and window < seen:  # (0: none)
            raise DzError(f"shared_prompt: attention with a window of {window} of {seen} tokens ({name})")
    # (rotations that change with the longest sequence of a forward, past a length)
    for name in ("rope_parameters", "rope_scaling"):
        rope = getattr(config, name, None)
        for r in (rope, *rope.values()) if isinstance(rope, dict) else ():  # (some have one for each type of layer)
            if isinstance(r, dict) and r.get("rope_type", r.get("type")) in ("dynamic", "longrope"):
                most = [n for n in (r.get("original_max_position_embeddings"), getattr(config, "original_max_position_embeddings", None),
                                    getattr(config, "max_position_embeddings", None)) if n]
                if not most or tokens > min(most):
                    raise DzError(f"shared_prompt: rotations that go by a sequence's length ({r.get('rope_type', r.get('type'))}), past that of {most}")


def _hidden(model, input_ids: torch.Tensor, position_ids: torch.Tensor, layout) -> torch.Tensor:
    """The last hidden states of a forward whose attention goes by `layout`."""
    global _registered
    if not _registered:
        from transformers import AttentionInterface

        AttentionInterface.register(ATTN_IMPL, _attention)
        _registered = True
    config = model.config
    before = config._attn_implementation
    config._attn_implementation = ATTN_IMPL
    layout.seen.clear()
    try:
        hidden = model.base_model(input_ids=input_ids, position_ids=position_ids, attention_mask=None, use_cache=False,
                                  dz_shared=layout).last_hidden_state
    finally:
        config._attn_implementation = before
    if len(layout.seen) != config.num_hidden_layers:
        raise DzError(f"shared_prompt: {len(layout.seen)} of {config.num_hidden_layers} layers called the attention")
    return hidden


class _Prompts:
    """Where the prompts of a batch of candidates lie: sequences of [padding | prompt | option]."""

    def __init__(self, model, input_ids: torch.Tensor, attention_mask: Optional[torch.Tensor], option_len, candidates: int):
        sequences, length = input_ids.shape
        device, examples = input_ids.device, sequences // candidates
        self.options = torch.as_tensor(option_len, device=device)
        columns = torch.arange(length, device=device)
        if attention_mask is None:
            self.pads, padded_left = torch.zeros_like(self.options), True
        else:
            there = attention_mask != 0
            self.pads = length - there.sum(1)
            padded_left = (there == (columns >= self.pads.unsqueeze(1))).all(1).view(examples, candidates)
        self.length = (length - self.pads - self.options).view(examples, candidates)
        self.first = self.length[:, 0]
        self.room = length - min(option_len)
        self.place = columns[:self.room]
        from_pads = (self.pads.unsqueeze(1) + self.place).clamp_(max=length - 1)
        self.tokens = input_ids.gather(1, from_pads).view(examples, candidates, self.room)  # prompts from their first token on
        # Of each sequence: whether its prompt lies as its example's first, and whether it has the same tokens there.
        self.placed = (self.length == self.length[:, :1]) & (self.length > 0) & padded_left
        self.before = 0  # a prompt's first position
        if model.config.model_type in COUNT_PADS:
            pads = self.pads.view(examples, candidates)
            self.placed &= pads == pads[:, :1]
            self.before = pads[:, :1]
        self.alike = ((self.tokens == self.tokens[:, :1]) | (self.place >= self.first.view(examples, 1, 1))).all(-1)


def shares_prompts(model, input_ids: torch.Tensor, attention_mask: Optional[torch.Tensor], option_len, candidates: int, *,
                   tokens: bool = True) -> bool:
    """Whether the candidates of each example of a batch, as shared_prompt_logprobs takes it, have one prompt: in the same
    places and (unless tokens is False) with the same tokens. The host waits for the answer."""
    if attention_mask is not None and attention_mask.shape != input_ids.shape:
        return False
    p = _Prompts(model, input_ids, attention_mask, option_len, candidates)
    return bool((p.placed & p.alike if tokens else p.placed).all())


def shared_prompt_logprobs(model, input_ids: torch.Tensor, attention_mask: Optional[torch.Tensor], option_len, candidates: int,
                           pad_id: Optional[int]) -> torch.Tensor:
    """The mean log probability of each sequence's last option_len tokens, (sequences,) in the logits' dtype: what
    trainer.py:1466-1500 selects, for a batch whose examples have `candidates` sequences each, one after another, left-padded
    (attention_mask 0), that differ in their last option_len tokens only.

    option_len: integers on the host, at least 1. Tokens that equal pad_id are left out, as there. Examples whose
    sequences do not share their prompt give NaN, and so do those of a model that counts padding (COUNT_PADS) whose sequences
    have their prompt in other places. (A sequence's last token predicts nothing that is read and is not
    computed, so that candidates of one token cost nothing beyond the prompt.)"""
    if torch.is_grad_enabled():
        raise DzError("shared_prompt_logprobs: nothing is recorded by autograd, call it under torch.no_grad()")
    sequences, length = input_ids.shape
    if candidates < 1 or sequences % candidates or len(option_len) != sequences or not 1 <= min(option_len) <= max(option_len) < length:
        raise DzError(f"shared_prompt_logprobs: {sequences} sequences of {length} tokens, {candidates} candidates each, option_len {list(option_len)[:8]}")
    if attention_mask is not None and attention_mask.shape != input_ids.shape:
        raise DzError(f"shared_prompt_logprobs: attention_mask must be {tuple(input_ids.shape)}, got {tuple(attention_mask.shape)}")
    _check_model(model, length, length - 1)  # (the last token predicts nothing)
    device, examples, most = input_ids.device, sequences // candidates, max(option_len)
    each = most - 1
    p = _Prompts(model, input_ids, attention_mask, option_len, candidates)
    options, room, place, first, same = p.options, p.room, p.place, p.first, p.placed & p.alike

    # prompts, then what each candidate adds to them
    last = torch.arange(most, device=device)
    targets = input_ids.gather(1, (length - options.unsqueeze(1) + last).clamp_(max=length - 1))  # (sequences, most)
    ids = torch.cat([p.tokens[:, 0], targets[:, :each].reshape(examples, candidates * each)], 1)
    steps = (first.unsqueeze(1) + last[:each]).repeat(1, candidates)
    positions = torch.cat([place.expand(examples, room), steps], 1) + p.before
    # (places that hold no token of a sequence repeat one, and nothing that is read sees them)
    positions = positions.clamp_(0, length - 1)

    with _alone(model):
        hidden = _hidden(model, ids, positions, _Candidates(room, candidates, each, first.to(torch.int32)))
    width = hidden.shape[-1]
    ends = hidden.gather(1, (first - 1).clamp(min=0).view(examples, 1, 1).expand(examples, 1, width))
    rows = torch.cat([ends.unsqueeze(1).expand(examples, candidates, 1, width), hidden[:, room:].view(examples, candidates, each, width)], 2)
    log_probs = torch.log_softmax(model.get_output_embeddings()(rows), -1)
    selected = log_probs.gather(-1, targets.view(examples, candidates, most, 1)).view(sequences, most)
    mask = last < options.unsqueeze(1)
    if pad_id is not None:
        mask = mask & (targets != pad_id)
    return ((selected * mask).sum(-1) / mask.sum(-1)).masked_fill_(~same.view(-1), float("nan"))


def generate(model, input_ids: torch.Tensor, max_new_tokens: int, *, answers: int = 1, prompt_lengths: Optional[torch.Tensor] = None,
             uniform: Optional[torch.Tensor] = None, generator: Optional[torch.Generator] = None,
             temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
             min_p: Union[float, torch.Tensor] = 0.0, eos_token_id: Optional[int] = None, kv_bits: int = 16) -> torch.Tensor:
    """`answers` answers of max_new_tokens tokens, (prompts, answers, max_new_tokens), to each prompt.

    input_ids (prompts, tokens): prompts from their first token on; prompt_lengths (prompts), int32: how many of them are the
    prompt's (default: all). uniform (prompts, answers, max_new_tokens), fp32: a number from 0 to 1 for each token
    (default: drawn from `generator`). temperature, top_k, top_p and min_p as sample_tokens takes them, a tensor being
    (prompts, answers). After eos_token_id an answer repeats it. kv_bits = 8 keeps keys and values in 8 bits
    (QuantizedKV). The host waits for nothing."""
    if kv_bits not in (8, 16):
        raise DzError(f"generate: kv_bits must be 16 (the model's dtype) or 8, got {kv_bits}")
    if input_ids.dim() != 2 or input_ids.shape[1] < 1 or answers < 1 or max_new_tokens < 1:
        raise DzError(f"generate: {tuple(input_ids.shape)} prompts, {answers} answers of {max_new_tokens} tokens")
    prompts, room = input_ids.shape
    device = input_ids.device
    if prompt_lengths is None:
        prompt_lengths = torch.full((prompts,), room, dtype=torch.int32, device=device)
    elif prompt_lengths.shape != (prompts,) or prompt_lengths.dtype != torch.int32:
        raise DzError(f"generate: prompt_lengths must be torch.int32 ({prompts},), got {prompt_lengths.dtype} {tuple(prompt_lengths.shape)}")
    if uniform is not None and uniform.shape != (prompts, answers, max_new_tokens):
        raise DzError(f"generate: uniform must be {(prompts, answers, max_new_tokens)}, got {tuple(uniform.shape)}")
    _check_model(model, room + max_new_tokens, room + max_new_tokens)
    most = getattr(model.config, "max_position_embeddings", None)
    if most is not None and room + max_new_tokens - 1 > most:  # (an answer's last token is not read again)
        raise DzError(f"generate: {room} tokens of a prompt and {max_new_tokens} new ones, the model has {most} positions")
    lengths = prompt_lengths.clamp(1, room)
    if uniform is None:
        uniform = torch.rand(prompts, answers, max_new_tokens, generator=generator, device=device)
    with _alone(model):
        training = [m for m in model.modules() if m.training]
        model.eval()
        try:
            return _draw(model, input_ids, max_new_tokens, answers, lengths, uniform, eos_token_id, kv_bits,
                         dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))
        finally:
            for m in training:
                m.training = True


def _draw(model, input_ids, max_new_tokens, answers, lengths, uniform, eos_token_id, kv_bits, sampling) -> torch.Tensor:
    prompts, room = input_ids.shape
    device = input_ids.device
    with torch.no_grad():
        layout = _Answers(prompts, answers, room, max_new_tokens, lengths, kv_bits)
        hidden = _hidden(model, input_ids, torch.arange(room, device=device).expand(prompts, room), layout)
        rows = hidden.gather(1, (lengths.long() - 1).view(prompts, 1, 1).expand(prompts, 1, hidden.shape[-1]))
        rows = rows.expand(prompts, answers, rows.shape[-1])
        tokens = torch.empty(prompts, answers, max_new_tokens, dtype=torch.int64, device=device)
        ended = None
        for t in range(max_new_tokens):
            logits = model.get_output_embeddings()(rows)
            drawn = sample_tokens(logits, uniform[:, :, t], **sampling)
            if eos_token_id is not None:
                drawn = drawn if ended is None else torch.where(ended, eos_token_id, drawn)
                ended = drawn == eos_token_id
            tokens[:, :, t] = drawn
            if t + 1 < max_new_tokens:
                layout.at = t
                positions = (lengths.long().view(prompts, 1) + t).expand(prompts, answers).reshape(-1, 1)
                # (a row without a distribution gives -1, which is no token: it goes on from token 0)
                rows = _hidden(model, drawn.clamp(min=0).view(-1, 1), positions, layout).view(prompts, answers, -1)
        return tokens
