"""The label field's training step (lookup, head, distillation, their gradients, Adam) against the same step in float64."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_step_follows_the_formulas():
    """Gradients of a step against autograd in float64 on the quantised head: what remains is the rounding of rows, logits and
    gradients to E4M3 and bfloat16. An E4M3 value is within 2^-4 of itself (relative), a uniform error below that of 2^-4 /
    sqrt(3) rms; two roundings (rows and gradients) and sums that average them: within 2^-4 of the gradient's norm."""
    from gsx_amd.label_field import LabelField
    rows, codes, labels, features, top = 700, 40, 33, 70, 5
    g = torch.Generator("cuda").manual_seed(3)
    field = LabelField(codes, features, labels)
    c = torch.randint(-1, codes, (rows,), device="cuda", generator=g, dtype=torch.int32)
    ids = torch.stack([torch.randperm(labels, device="cuda", generator=g)[:top] for _ in range(rows)]).int()
    t = torch.randn(rows, top, device="cuda", generator=g) * 2
    weight = (c >= 0).float()
    table = field.table.double().requires_grad_()
    head = field.blocks.float().double().requires_grad_()
    z = torch.where((c >= 0)[:, None], table[c.clamp(min=0).long()], 0) * field.scale @ head.T
    p = torch.softmax(t.double() / field.temperature, 1)
    terms = p * (torch.log(p) - torch.log_softmax(z / field.temperature, 1).gather(1, ids.long()))
    want = weight.double() * field.temperature**2 * terms.sum(1)
    want.sum().div(rows).backward()
    before = field.table.clone()
    loss = field.step(c, ids, t, weight)
    # rows and logits are off by a few percent of themselves, the loss by their sum over the entries
    assert (loss - want.float()).abs().max() <= 0.05 * (1 + want.max())
    for got, exact in ((field.table_grad, table.grad), (field.head_grad, head.grad)):
        assert torch.linalg.norm(got.double() - exact) <= 2.0**-4 * torch.linalg.norm(exact)
    unused = torch.ones(codes, dtype=torch.bool, device="cuda")
    unused[c[c >= 0].long()] = False
    assert (field.table_grad[unused] == 0).all()
    # Adam's first step moves every weight with a gradient by the learning rate
    moved = (field.table - before).abs()
    assert torch.allclose(moved[field.table_grad.abs() > 1e-6], torch.tensor(1e-2, device="cuda"), rtol=0.05)


def test_training_learns_the_teacher():
    from gsx_amd.label_field import main
    assert main(["--gaussians", "20000", "--steps", "60", "--labels", "40", "--cells", "12"]) > 0.5


def test_single_query_and_batch_agree():
    from gsx_amd.label_field import LabelField
    field = LabelField(50, 64, 300)
    c = torch.arange(40, dtype=torch.int32, device="cuda")
    batch = field.logits(c)
    for i in (0, 17, 39):
        one = field.logits(c[i: i + 1])
        # the same values in another order of sums: one rounding to bfloat16 apart
        assert torch.allclose(one.float(), batch[i: i + 1].float(), rtol=2.0**-7, atol=1e-3)


def test_refusals():
    from gsx_amd._lib import GsxHipError
    from gsx_amd.label_field import LabelField
    field = LabelField(4, 8, 5)
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    with pytest.raises(GsxHipError):
        field.step(empty, empty[:, None], torch.empty(0, 1, device="cuda"))
