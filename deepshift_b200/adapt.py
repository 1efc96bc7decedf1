"""Adapting a frozen shift network to several tasks at once, and serving them side by side:

    python -m deepshift_b200.adapt [--tasks 4 --rank 16 --width 256 --hidden 512 --vocabulary 4000 --rows 2048 --steps 60]

A token goes through an embedding, two shift layers with packed weights and the head; all of these stay as they are.  Beside each
shift layer are the tasks' adapters (``adapters.AdaptedLinear``), the only thing trained: every row of a batch belongs to a
task, the loss is ``losses.linear_cross_entropy`` over the whole vocabulary, and the gradients of all adapters together are
clipped by ``gradients.clip_grad_norm_`` before the step.  Then requests of one token each, of mixed tasks and some of
none, are answered in one batch.

Data are synthetic: tokens come in groups, and a task's answer to a token is the first token of a group that is so many
further on.  No counterpart in the reference, whose ``use_kernel`` layers are for inference.
"""
import argparse
import time

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import adapters, gradients, losses, modules


class AdaptedModel(nn.Module):
    """Embedding, two adapted shift layers with a residual, and a head that is kept in bfloat16."""

    def __init__(self, vocabulary, width, hidden, tasks, rank, groups=16, device="cuda"):
        super().__init__()
        self.vocabulary, self.groups = vocabulary, groups
        centres = torch.randn(groups, width, device=device)
        of = torch.arange(vocabulary, device=device) * groups // vocabulary
        self.register_buffer("embedding", F.layer_norm(centres[of] + 0.3 * torch.randn(vocabulary, width, device=device), (width,)))
        self.register_buffer("head", (torch.randn(vocabulary, width, device=device) / width ** 0.5).bfloat16())

        def shift(n, m):
            return modules.LinearShift(n, m, use_kernel=True, act_integer_bits=8, act_fraction_bits=8).to(device)
        self.into = adapters.AdaptedLinear(shift(width, hidden), tasks, rank, device=device)
        self.back = adapters.AdaptedLinear(shift(hidden, width), tasks, rank, device=device)

    def forward(self, tokens, plan):
        x = self.embedding[tokens]
        h = F.layer_norm(F.relu(self.into(x, plan)), (self.into.out_features,))
        return F.layer_norm(x + self.back(h, plan), (x.shape[-1],)).bfloat16()

    def loss(self, tokens, answers, plan, reduction="mean"):
        return losses.linear_cross_entropy(self(tokens, plan), self.head, answers, reduction=reduction)

    def answer(self, tokens, tasks):
        """The answer of ``tasks`` to ``tokens``."""
        group = (tokens * self.groups // self.vocabulary + 1 + tasks) % self.groups
        return (group * self.vocabulary + self.groups - 1) // self.groups


def train(model, tasks, rows, steps, lr=1e-2, max_norm=1.0):
    """``steps`` steps on batches of ``rows`` rows; returns the losses and the gradients' norms before clipping, on the host."""
    trained = [p for p in model.parameters() if p.requires_grad]
    optimiser = torch.optim.Adam(trained, lr=lr)
    curve, norms = [], []
    for _ in range(steps):
        tokens = torch.randint(0, model.vocabulary, (rows,), device=model.head.device)
        ids = torch.randint(0, tasks, (rows,), device=model.head.device)
        loss = model.loss(tokens, model.answer(tokens, ids), adapters.plan_rows(ids, tasks))
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        norms.append(gradients.clip_grad_norm_(trained, max_norm))
        optimiser.step()
        curve.append(loss.detach())
    return torch.stack(curve).tolist(), torch.stack(norms).tolist()


def serve(model, tokens, ids, tasks):
    """The probability that each request's row gives to its task's answer (for a row without one, task -1: to task 0's)."""
    with torch.no_grad():
        plan = adapters.plan_rows(ids, tasks)
        return torch.exp(-model.loss(tokens, model.answer(tokens, ids.clamp(min=0)), plan, reduction="none"))


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tasks", 4), ("rank", 16), ("width", 256), ("hidden", 512), ("vocabulary", 4000), ("rows", 2048), ("steps", 60), ("requests", 64),
                        ("seed", 0)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--lr", type=float, default=1e-2)
    p.add_argument("--max-norm", type=float, default=1.0)
    a = p.parse_args(argv)
    if not torch.cuda.is_available():
        p.error("this needs a GPU")
    torch.manual_seed(a.seed)
    model = AdaptedModel(a.vocabulary, a.width, a.hidden, a.tasks, a.rank)
    curve, norms = train(model, a.tasks, a.rows, a.steps, a.lr, a.max_norm)
    print("loss %.3f -> %.3f, norm of the gradients %.3f -> %.3f" % (curve[0], curve[-1], norms[0], norms[-1]))
    tokens = torch.randint(0, a.vocabulary, (a.requests,), device="cuda")
    ids = torch.arange(a.requests, device="cuda") % (a.tasks + 1) - 1   # each task in turn, and none
    for _ in range(20):
        right = serve(model, tokens, ids, a.tasks)
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(20):
        serve(model, tokens, ids, a.tasks)
    torch.cuda.synchronize()
    print("%d requests: probability of the right answer %.3f with an adapter, %.5f without; %.0f us a batch"
          % (a.requests, float(right[ids >= 0].mean()), float(right[ids < 0].mean()), (time.perf_counter() - began) / 20 * 1e6))
    return curve, right, ids


if __name__ == "__main__":
    main()
