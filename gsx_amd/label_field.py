"""A label field over a Gaussian scene, trained against a teacher's top logits: every operator of `gsx_amd.fields` as a program
uses them, one step after another.

    python -m gsx_amd.label_field [--gaussians N] [--labels L] [--steps K]

Each Gaussian holds the code of the grid cell it lies in. A field is a table with a row for each code and a head with a row for
each label. A step looks the rows up, multiplies them with the head in 8-bit blocks, compares the logits with the teacher's and
carries the gradient back to head and table, which Adam updates in float32; the head's blocks are laid out anew from them.
`LabelField.labels` answers for any Gaussians, one among them.
"""
from __future__ import annotations

import argparse

import torch

from . import fields, scenes
from ._lib import GsxHipError
from .backend import Adam


class LabelField:
    """codes: rows of the table; features: columns of table and head; labels: rows of the head. Rows travel in `dtype`, table,
    head, their gradients and Adam's moments are float32."""

    def __init__(self, codes: int, features: int, labels: int, temperature: float = 2.0, learning_rate: float = 1e-2,
                 dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.scale = 1.0 / features ** 0.5
        self.temperature = temperature
        self.dtype = dtype
        self.table = torch.randn(codes, features, device="cuda", generator=g)
        self.head = torch.randn(labels, features, device="cuda", generator=g) * 0.1
        self.table_grad = torch.zeros_like(self.table)
        self.head_grad = torch.zeros_like(self.head)
        self.optimizer = Adam([dict(parameter=self.table, gradient=self.table_grad, learning_rate=learning_rate),
                               dict(parameter=self.head, gradient=self.head_grad, learning_rate=learning_rate)])
        self._lay_out()

    def _lay_out(self):
        """The head's blocks, along features for the product and along labels for its gradient."""
        self.blocks = fields.quantize(self.head)
        self.blocks_t = fields.quantize(self.head, transpose=True)

    def logits(self, codes: torch.Tensor) -> torch.Tensor:
        """Logits [count, labels] of int32 codes; a Gaussian without a code (-1) has equal ones."""
        return fields.linear(fields.lookup(self.table, codes, self.scale, out_dtype=self.dtype), self.blocks)

    def labels(self, codes: torch.Tensor) -> torch.Tensor:
        return self.logits(codes).argmax(1)

    def step(self, codes: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
             row_weight: torch.Tensor | None = None) -> torch.Tensor:
        """One training step; the rows' losses. The gradient is that of their mean."""
        if codes.numel() == 0:
            raise GsxHipError("a step needs at least one row")
        rows = fields.lookup(self.table, codes, self.scale, out_dtype=self.dtype)
        logits = fields.linear(rows, self.blocks)
        loss, _, grad = fields.distill(logits, teacher_ids, teacher_logits, self.temperature, row_weight,
                                       grad_scale=1.0 / codes.numel())
        grad_rows, _ = fields.linear_backward(rows, grad, self.blocks_t, grad_weight=self.head_grad)
        fields.lookup_backward(grad_rows, codes, self.table.shape[0], self.scale, grad_table=self.table_grad)
        self.optimizer.step()
        self._lay_out()
        return loss


def cell_codes(mean3d: torch.Tensor, cells: int) -> torch.Tensor:
    """The code of each Gaussian: its cell in a grid of cells^3 over the scene's inner box; -1 outside of it."""
    lo, hi = torch.quantile(mean3d[:: max(1, mean3d.shape[0] // 100_000)], torch.tensor([0.02, 0.98], device="cuda"), dim=0)
    at = ((mean3d - lo) / (hi - lo) * cells).floor().int()
    inside = ((at >= 0) & (at < cells)).all(1)
    code = (at[:, 0] * cells + at[:, 1]) * cells + at[:, 2]
    return torch.where(inside, code, -1).int()


def teacher_of(mean3d: torch.Tensor, labels: int, top: int, seed: int = 1):
    """A teacher whose labels each have a place in the scene and a logit that falls with the square of the distance from it: its
    `top` largest logits and their ids for each Gaussian."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    places = mean3d[torch.randint(mean3d.shape[0], (labels,), device="cuda", generator=g)]
    apart = mean3d.std() * 3.5 / labels ** (1 / 3)
    values, ids = (-8 * (torch.cdist(mean3d, places) / apart) ** 2).topk(top, dim=1)
    return ids.int(), values


def main(argv=None) -> float:
    p = argparse.ArgumentParser(description="train a label field on a generated scene")
    p.add_argument("--gaussians", type=int, default=100_000)
    p.add_argument("--labels", type=int, default=150)
    p.add_argument("--features", type=int, default=64)
    p.add_argument("--cells", type=int, default=20)
    p.add_argument("--top", type=int, default=8)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--rate", type=float, default=0.05)
    a = p.parse_args(argv)
    mean3d = torch.from_numpy(scenes.config0(n=a.gaussians).scene.mean3d).cuda()
    codes = cell_codes(mean3d, a.cells)
    ids, logits = teacher_of(mean3d, a.labels, a.top)
    weight = (codes >= 0).float()
    field = LabelField(a.cells ** 3, a.features, a.labels, learning_rate=a.rate)
    for k in range(a.steps):
        loss = field.step(codes, ids, logits, weight)
        if k % 20 == 0 or k == a.steps - 1:
            print(f"step {k}: loss {loss.sum().item() / weight.sum().item():.4f}", flush=True)
    inside = codes >= 0
    agree = (field.labels(codes) == ids[:, 0])[inside].float().mean().item()
    print(f"the field's first label is the teacher's for {100 * agree:.1f}% of {int(inside.sum())} Gaussians")
    print(f"one Gaussian's label: {field.labels(codes[inside][:1]).item()}")
    return agree


if __name__ == "__main__":
    main()
