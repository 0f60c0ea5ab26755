"""A label field over a Gaussian scene, trained against a teacher's top logits or against given labels: every operator of
`gsx_amd.fields` as a program uses them, one step after another.

    python -m gsx_amd.label_field [--gaussians N] [--labels L] [--steps K] [--given] [--moments 32|8] [--answers K]

Each Gaussian holds the code of the grid cell it lies in. A field is a table with a row for each code and a head with a row for
each label. A step looks the rows up, multiplies them with the head in 8-bit blocks, compares the logits with the teacher's and
carries the gradient back to head and table, which Adam updates in float32; the head's blocks are laid out anew from them.
`LabelField.labels` answers for any Gaussians, one among them.

With given labels a step's loss is the labels' negative log probability. AdamW takes Adam's place where moments are asked for in 32
or 8 bits. `LabelField.answers` gives the likeliest labels with their log probabilities from a head in 4-bit blocks, half the bytes
of the 8-bit one; what it gives is also a teacher for another field's steps.
"""
from __future__ import annotations

import argparse

import torch

from . import fields, scenes
from ._lib import GsxHipError
from .backend import Adam, AdamW


class LabelField:
    """codes: rows of the table; features: columns of table and head; labels: rows of the head. Rows travel in `dtype`, table,
    head, their gradients and Adam's moments are float32. moments: None for Adam, 32 or 8 for AdamW with moments of as many bits and
    with weight_decay.

    A step writes table, head and the head's blocks where they are: one with AdamW may be captured into a graph, whose replays go on
    from whatever step was the last, and calls on other streams are the caller's to order against it. Logits and answers may be asked
    for on several streams at once."""

    def __init__(self, codes: int, features: int, labels: int, temperature: float = 2.0, learning_rate: float = 1e-2,
                 dtype=torch.bfloat16, seed: int = 0, moments: int | None = None, weight_decay: float = 0.0):
        if moments is None and weight_decay != 0.0:
            raise GsxHipError("weight decay needs AdamW: moments of 32 or 8 bits")
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.scale = 1.0 / features ** 0.5
        self.temperature = temperature
        self.dtype = dtype
        self.table = torch.randn(codes, features, device="cuda", generator=g)
        self.head = torch.randn(labels, features, device="cuda", generator=g) * 0.1
        self.table_grad = torch.zeros_like(self.table)
        self.head_grad = torch.zeros_like(self.head)
        if moments is None:
            self.optimizer = Adam([dict(parameter=self.table, gradient=self.table_grad, learning_rate=learning_rate),
                                   dict(parameter=self.head, gradient=self.head_grad, learning_rate=learning_rate)])
        else:
            self.optimizer = AdamW([dict(parameters=[self.table, self.head], gradients=[self.table_grad, self.head_grad],
                                         learning_rate=learning_rate, weight_decay=weight_decay)], bits=moments)
        self.blocks = self.blocks_t = None
        self._blocks4 = fields.quantize4(self.head)  # their memory: _stream4 says whether they are the head's
        self._ready4 = torch.cuda.Event()            # after they were laid out for an answer
        self._lay_out()

    def _lay_out(self):
        """The head's blocks, along features for the product and along labels for its gradient."""
        self.blocks = fields.quantize(self.head, out=self.blocks)
        self.blocks_t = fields.quantize(self.head, transpose=True, out=self.blocks_t)
        if torch.cuda.is_current_stream_capturing():
            fields.quantize4(self.head, out=self._blocks4)  # a replay runs nothing that could ask for it
        else:
            self._stream4 = None  # laid out, and on which stream, when the first answer after a step is asked for

    def head_blocks4(self) -> fields.Blocks4:
        """The head in 4-bit blocks, for calls on the current stream. A graph that is captured lays out blocks of its own at each
        replay, from the head as it is then."""
        if torch.cuda.is_current_stream_capturing():
            return fields.quantize4(self.head)
        handle = fields._current_stream(self.head.device.index)
        if self._stream4 is None:
            fields.quantize4(self.head, out=self._blocks4)
            self._ready4.record()
            self._stream4 = handle
        elif self._stream4 != handle:
            self._ready4.wait()
        return self._blocks4

    def logits(self, codes: torch.Tensor) -> torch.Tensor:
        """Logits [count, labels] of int32 codes; a Gaussian without a code (-1) has equal ones."""
        return fields.linear(fields.lookup(self.table, codes, self.scale, out_dtype=self.dtype), self.blocks)

    def labels(self, codes: torch.Tensor) -> torch.Tensor:
        return self.logits(codes).argmax(1)

    def answers(self, codes: torch.Tensor, top: int = 1, labels: torch.Tensor | None = None) -> fields.LogProbs:
        """The `top` likeliest labels of int32 codes with their log probabilities, the distribution's entropy, and the log
        probability of given labels, by the head in 4-bit blocks."""
        rows = fields.lookup(self.table, codes, self.scale, out_dtype=self.dtype)
        return fields.log_probs(fields.linear(rows, self.head_blocks4(), out_dtype=torch.float32), labels, top)

    def _check_step(self, codes):
        if codes.numel() == 0:
            raise GsxHipError("a step needs at least one row")
        if isinstance(self.optimizer, Adam) and torch.cuda.is_current_stream_capturing():
            raise GsxHipError("a step that is captured needs AdamW (moments of 32 or 8 bits): Adam counts its steps on the host, "
                              "replays would all be the same one")

    def step_labels(self, codes: torch.Tensor, labels: torch.Tensor, row_weight: torch.Tensor | None = None,
                    entropy_weight: float = 0.0) -> torch.Tensor:
        """One training step against given int32 labels (a row whose label lies outside of the field's has none); the rows'
        losses, -log p(label) times the row's weight less entropy_weight times the entropy. The gradient is that of their mean."""
        self._check_step(codes)
        rows = fields.lookup(self.table, codes, self.scale, out_dtype=self.dtype)
        logits = fields.linear(rows, self.blocks)
        mean = 1.0 / codes.numel()
        q = fields.log_probs(logits, labels, grad_scale=-mean, row_grad=row_weight, entropy_scale=-mean * entropy_weight)
        self._descend(rows, q.grad, codes)
        loss = -q.chosen if row_weight is None else torch.where(row_weight != 0, -q.chosen * row_weight, 0.0)
        return loss if entropy_weight == 0.0 else loss - entropy_weight * q.entropy

    def step(self, codes: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
             row_weight: torch.Tensor | None = None) -> torch.Tensor:
        """One training step; the rows' losses. The gradient is that of their mean."""
        self._check_step(codes)
        rows = fields.lookup(self.table, codes, self.scale, out_dtype=self.dtype)
        logits = fields.linear(rows, self.blocks)
        loss, _, grad = fields.distill(logits, teacher_ids, teacher_logits, self.temperature, row_weight,
                                       grad_scale=1.0 / codes.numel())
        self._descend(rows, grad, codes)
        return loss

    def _descend(self, rows, grad, codes):
        """The logits' gradient carried back, and the optimizer's step."""
        grad_rows, _ = fields.linear_backward(rows, grad, self.blocks_t, grad_weight=self.head_grad)
        fields.lookup_backward(grad_rows, codes, self.table.shape[0], self.scale, grad_table=self.table_grad)
        self.optimizer.step()
        self._lay_out()


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
    p.add_argument("--given", action="store_true", help="train against the teacher's first labels alone")
    p.add_argument("--moments", type=int, choices=(32, 8), help="AdamW with moments of so many bits instead of Adam")
    p.add_argument("--decay", type=float, default=0.0, help="AdamW's weight decay")
    p.add_argument("--answers", type=int, default=0, help="print so many likeliest labels of one Gaussian, by a 4-bit head")
    a = p.parse_args(argv)
    if not 0 <= a.answers <= min(64, a.labels):
        p.error("--answers takes 0 to 64 labels, no more than there are")
    mean3d = torch.from_numpy(scenes.config0(n=a.gaussians).scene.mean3d).cuda()
    codes = cell_codes(mean3d, a.cells)
    ids, logits = teacher_of(mean3d, a.labels, a.top)
    weight = (codes >= 0).float()
    field = LabelField(a.cells ** 3, a.features, a.labels, learning_rate=a.rate, moments=a.moments, weight_decay=a.decay)
    first = ids[:, 0].contiguous()
    for k in range(a.steps):
        loss = field.step_labels(codes, first, weight) if a.given else field.step(codes, ids, logits, weight)
        if k % 20 == 0 or k == a.steps - 1:
            print(f"step {k}: loss {loss.sum().item() / weight.sum().item():.4f}", flush=True)
    inside = codes >= 0
    agree = (field.labels(codes) == ids[:, 0])[inside].float().mean().item()
    print(f"the field's first label is the teacher's for {100 * agree:.1f}% of {int(inside.sum())} Gaussians")
    print(f"one Gaussian's label: {field.labels(codes[inside][:1]).item()}")
    if a.answers > 0:
        q = field.answers(codes, a.answers, first)
        agree4 = (q.top_ids[:, 0] == first)[inside].float().mean().item()
        print(f"by the 4-bit head for {100 * agree4:.1f}%, with {q.chosen[inside].mean().item():.3f} for the mean log probability "
              f"of the teacher's")
        one = field.answers(codes[inside][:1], a.answers)
        for label, log_q in zip(one.top_ids[0].tolist(), one.top_log_probs[0].tolist()):
            print(f"  label {label}: log probability {log_q:.3f}")
    return agree


if __name__ == "__main__":
    main()
