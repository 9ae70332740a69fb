"""Training steps of a small mixture-of-experts language model on the library's operators.

  python examples/moe_step.py [--steps N] [--plain]

tokens -> embedding -> router -> tokens sorted by expert -> the experts' products -> back with
the router's weights -> logits -> loss -> gradients -> clipped by their global norm -> update.
Rows are moved and summed by torch.ops.dcopy operators and the clipping by dcopy.clip_grad_norm;
the products are torch's.  --plain runs the same model on torch's own indexing instead.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "data-copy_b200"))
import dcopy  # noqa: E402
from dcopy import torch_ops  # noqa: E402,F401  (registers torch.ops.dcopy.*)

VOCAB, WIDTH, HIDDEN, EXPERTS, SLOTS, ALIGN = 1000, 128, 256, 8, 2, 16


def parameters(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        t = torch.randn(shape, generator=g, device="cuda") * shape[-2] ** -0.5
        return t.requires_grad_()

    return {"table": normal(VOCAB, WIDTH), "router": normal(WIDTH, EXPERTS),
            "up": normal(EXPERTS, WIDTH, HIDDEN), "down": normal(EXPERTS, HIDDEN, WIDTH),
            "head": normal(WIDTH, VOCAB)}


def forward(p, ids, plain):
    """Logits of a batch of token ids."""
    scale = WIDTH ** 0.5
    if plain:
        x = p["table"][ids] * scale
    else:
        x = torch.ops.dcopy.embedding(p["table"], ids, scale)
    weights, chosen = torch.softmax(x @ p["router"], dim=1).topk(SLOTS, dim=1)
    if plain:
        mixed = torch.zeros_like(x)
        for e in range(EXPERTS):
            token, slot = torch.nonzero(chosen == e, as_tuple=True)
            y = torch.relu(x[token] @ p["up"][e]) @ p["down"][e]
            mixed = mixed.index_add(0, token, y * weights[token, slot, None])
    else:
        dest, source, offsets = torch.ops.dcopy.expert_sort(chosen, EXPERTS, ALIGN)
        rows = torch.ops.dcopy.expert_dispatch(x, dest, source)
        ends = offsets.tolist()
        y = [torch.relu(rows[a:b] @ p["up"][e]) @ p["down"][e]
             for e, (a, b) in enumerate(zip(ends, ends[1:]))]
        y = torch.cat(y + [rows[ends[-1]:]])  # the rows behind the last segment hold no token
        mixed = torch.ops.dcopy.expert_combine(y, dest, source, weights)
    return (x + mixed) @ p["head"]


def train(steps, plain, seed=0, tokens=512, rate=0.5, max_norm=1.0):
    """The loss and the gradients' norm of each step."""
    p = parameters(seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    ids = torch.randint(0, VOCAB, (tokens,), generator=g, device="cuda")
    target = torch.roll(ids, -1)
    values = list(p.values())
    for v in values:
        v.grad = torch.zeros_like(v)
    grads = None if plain else dcopy.GradList([v.grad for v in values])
    norm = torch.empty(1, device="cuda")
    seen = []
    for _ in range(steps):
        loss = torch.nn.functional.cross_entropy(forward(p, ids, plain), target)
        for v in values:
            v.grad.zero_()
        loss.backward()  # into the same buffers each step: the list stays valid
        if plain:
            norm = torch.cat([v.grad.reshape(-1) for v in values]).norm().reshape(1)
            factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
            for v in values:
                v.grad.mul_(factor)
        else:
            dcopy.clip_grad_norm(grads, max_norm, norm)
        with torch.no_grad():
            for v in values:
                v -= rate * v.grad
        seen.append((loss.item(), norm.item()))
    return seen


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--plain", action="store_true")
    a = ap.parse_args()
    for k, (loss, norm) in enumerate(train(a.steps, a.plain)):
        print(f"step {k}: loss {loss:.4f}, gradient norm {norm:.4f}")


if __name__ == "__main__":
    main()
