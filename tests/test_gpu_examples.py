"""The distillation example end to end, on a small random OPT."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("distill_opt", os.path.join(ROOT, "examples", "distill_opt.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_distillation_example(dtype):
    ex = load()
    lines = []
    r = ex.run("opt-tiny", dtype, top=16, batch_size=3, fo_steps=12, zo_steps=4, log=lines.append)
    assert len(r["fo"]) == 12 and len(r["zo"]) == 4 and len(lines) == 17
    assert all(x == x and x > 0 for x in r["fo"] + r["zo"])
    # gradient descent on two batches in turn: each one's distance falls
    assert r["fo"][-1] < r["fo"][1] and r["fo"][-2] < r["fo"][0]
    model, batch, rec = r["model"], r["batches"][0], r["recorded"][0]
    # the recorded entries: none where nothing is predicted, decreasing elsewhere
    dead = ex.next_tokens(batch) == ex.IGNORE_INDEX
    assert (rec["teacher_tokens"][dead] == -1).all() and (rec["teacher_tokens"][~dead] >= 0).all()
    assert (rec["teacher_values"][~dead].diff(dim=-1) <= 0).all()
    # the candidates' scores against the logits'
    with torch.no_grad():
        logits = model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    lp = F.log_softmax(logits[:, -2].float(), -1).gather(-1, batch["input_ids"][:, -1:]).squeeze(-1)
    # the logits are rounded to the model's type and the kernel's are not: half a step of the largest
    tol = 2 * float(logits[:, -2].abs().max()) * torch.finfo(logits.dtype).eps / 2 + 1e-5
    assert (r["scores"][0] - lp).abs().max() <= tol
