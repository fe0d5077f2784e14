"""Distillation of an OPT model from a teacher's largest logits, scored as the option loss scores.

    python examples/distill_opt.py [--shape opt-mini] [--dtype bf16] [--top 32] [--fo-steps 8] [--zo-steps 8]

1. The teacher (another random OPT of the shape) reads the batches once; its `top` largest log probabilities at
   every position that predicts a token are kept, 12 bytes each, and the teacher is not needed again.
2. First-order steps: the loss and its gradient with respect to the logits in one call, then the model's backward.
3. Zeroth-order steps: the trainer's own step with the distance as its loss, forward only.
4. The candidates of each example are scored from the last hidden states and the head, without logits.

Random weights and random prompts: the numbers show that the parts fit together, not a model's quality.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from dizo_amd import synth  # noqa: E402
from dizo_amd.token_loss import IGNORE_INDEX, linear_token_logprobs, token_logprobs, topk_distill, topk_distill_grad  # noqa: E402
from dizo_amd.trainer import ZOArguments, ZOTrainer  # noqa: E402

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def next_tokens(batch) -> torch.Tensor:
    """The token that each position but the last predicts; IGNORE_INDEX where that is padding."""
    return batch["input_ids"][:, 1:].masked_fill(batch["attention_mask"][:, 1:] == 0, IGNORE_INDEX)


@torch.no_grad()
def record(teacher, batch, top: int) -> dict:
    """The batch with the teacher's largest log probabilities (positions of padding have no entries)."""
    logits = teacher(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    kept = token_logprobs(logits[:, :-1], next_tokens(batch), top=top)
    return {**batch, "teacher_values": kept.top_logprobs, "teacher_tokens": kept.top_tokens}


def position_weights(batch) -> torch.Tensor:
    """1 / (number of positions with a teacher), and 0 for the others."""
    there = (batch["teacher_tokens"][..., 0] >= 0).float()
    return there / there.sum().clamp(min=1)


def distance(logits: torch.Tensor, batch, temperature: float) -> torch.Tensor:
    rows = topk_distill(logits[:, :-1], batch["teacher_values"], batch["teacher_tokens"], temperature=temperature)
    return (rows * position_weights(batch)).sum()


def first_order_step(model, batch, lr: float, temperature: float) -> torch.Tensor:
    """One SGD step. The gradient of the logits is known with the loss, so that autograd starts there."""
    logits = model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits[:, :-1]
    weights = position_weights(batch)
    rows, grad = topk_distill_grad(logits.detach(), batch["teacher_values"], batch["teacher_tokens"], weights, temperature=temperature)
    params = [p for p in model.parameters() if p.requires_grad]
    with torch.no_grad():
        for p, g in zip(params, torch.autograd.grad(logits, params, grad, allow_unused=True)):
            if g is not None:
                p.sub_(g, alpha=lr)
    return (rows * weights).sum()


class DistillTrainer(ZOTrainer):
    """The ZO step with the distance to the recorded teacher as its loss."""

    temperature = 1.0

    def zo_forward(self, model, inputs):
        model.eval()
        with torch.inference_mode():
            logits = model(input_ids=inputs["input_ids"], attention_mask=inputs["attention_mask"]).logits
            return distance(logits, inputs, self.temperature)


@torch.no_grad()
def score(model, batch) -> torch.Tensor:
    """The log probability of each candidate's answer (its last option_len tokens, averaged), from the hidden
    states of the positions that predict them: no logits are made."""
    hidden = model.model.decoder(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).last_hidden_state
    answers = batch["option_len"].tolist()
    n = max(answers)
    tokens = batch["input_ids"][:, -n:].clone()
    for i, k in enumerate(answers):
        tokens[i, :n - k] = IGNORE_INDEX
    lp = linear_token_logprobs(hidden[:, -n - 1:-1], model.lm_head.weight, tokens).logprobs
    return lp.sum(-1) / (tokens != IGNORE_INDEX).sum(-1)


def run(shape: str = "opt-mini", dtype: str = "bf16", top: int = 32, batch_size: int = 4, fo_steps: int = 8, zo_steps: int = 8,
        lr: float = 0.5, zo_lr: float = 1e-5, temperature: float = 2.0, seed: int = 0, log=print) -> dict:
    dt, device = DTYPES[dtype], torch.device("cuda")
    vocab = synth.SHAPES[shape].vocab
    gen = torch.Generator().manual_seed(seed)
    batches = []
    for _ in range(2):
        b = synth.make_batch(batch_size, vocab, gen=gen)
        batches.append({k: v.to(device) if torch.is_tensor(v) else v for k, v in b.items()})
    teacher = synth.build_opt(shape, dtype=dt, seed=seed + 1, init_std=0.06)
    recorded = [record(teacher, b, top) for b in batches]
    del teacher
    model = synth.build_opt(shape, dtype=dt, seed=seed + 2, init_std=0.02)
    result = {"fo": [], "zo": []}
    for i in range(fo_steps):
        result["fo"].append(float(first_order_step(model, recorded[i % 2], lr, temperature)))
        log(f"first-order step {i}: distance {result['fo'][-1]:.4f}")
    np.random.seed(seed)
    trainer = DistillTrainer(model, ZOArguments(learning_rate=zo_lr, zo_eps=1e-3, max_steps=max(1, zo_steps)), train_dataloader=None)
    trainer.temperature = temperature
    for i in range(zo_steps):
        result["zo"].append(float(trainer.training_step(recorded[i % 2])))
        log(f"zeroth-order step {i}: distance {result['zo'][-1]:.4f}")
    trainer.zo_flush()
    result["scores"] = [score(model, b) for b in batches]
    log("candidates' log probabilities: " + ", ".join(f"{x:.3f}" for x in result["scores"][0].tolist()))
    result["model"], result["batches"], result["recorded"] = model, batches, recorded
    trainer.zo_close()
    return result


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--shape", default="opt-mini", choices=sorted(synth.SHAPES))
    p.add_argument("--dtype", default="bf16", choices=sorted(DTYPES))
    p.add_argument("--top", type=int, default=32)
    p.add_argument("--batch-size", type=int, default=4)
    p.add_argument("--fo-steps", type=int, default=8)
    p.add_argument("--zo-steps", type=int, default=8)
    a = p.parse_args()
    run(a.shape, a.dtype, a.top, a.batch_size, a.fo_steps, a.zo_steps)


if __name__ == "__main__":
    main()
