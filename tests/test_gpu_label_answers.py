"""The label field trained against given labels with AdamW, and its answers from a 4-bit head: the operators together, as a program
uses them, against the same steps in float64."""
import numpy as np
import pytest

import adamw_plain

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROWS, CODES, LABELS, FEATURES = 600, 40, 33, 70


def data(seed=5):
    g = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(-1, CODES, (ROWS,), device="cuda", generator=g, dtype=torch.int32)
    labels = torch.randint(-1, LABELS + 1, (ROWS,), device="cuda", generator=g, dtype=torch.int32)
    weight = torch.rand(ROWS, device="cuda", generator=g) * (codes >= 0)
    return codes, labels, weight


def exact(field, codes, labels, weight, entropy_weight):
    """(losses, table's gradient, head's gradient) in float64 on the head that the blocks stand for."""
    table = field.table.double().requires_grad_()
    head = field.blocks.float().double().requires_grad_()
    z = torch.where((codes >= 0)[:, None], table[codes.clamp(min=0).long()], 0) * field.scale @ head.T
    log_q = torch.log_softmax(z, 1)
    given = (labels >= 0) & (labels < LABELS)
    chosen = torch.where(given, log_q.gather(1, labels.clamp(0, LABELS - 1).long()[:, None])[:, 0], 0)
    w = torch.ones_like(chosen) if weight is None else weight.double()
    loss = -chosen * w + entropy_weight * (log_q.exp() * log_q).sum(1)
    loss.mean().backward()
    return loss.detach(), table.grad, head.grad


@pytest.mark.parametrize("bits,weighted,entropy_weight", [(None, True, 0.0), (32, True, 0.0), (32, False, 0.25), (8, True, 0.25)])
def test_step_labels_follows_the_formulas(bits, weighted, entropy_weight):
    """As a step against a teacher: an E4M3 rounding is within 2^-4 of its value, below 2^-4 / sqrt(3) rms for an even spread, and
    sums average the two of them (rows and gradients): within 2^-4 of the gradient's norm."""
    from gsx_amd.label_field import LabelField
    field = LabelField(CODES, FEATURES, LABELS, moments=bits)
    codes, labels, weight = data()
    weight = weight if weighted else None
    want, table_grad, head_grad = exact(field, codes, labels, weight, entropy_weight)
    before = torch.cat([field.table.flatten(), field.head.flatten()]).cpu().numpy()
    loss = field.step_labels(codes, labels, weight, entropy_weight)
    assert (loss - want.float()).abs().max() <= 0.05 * (1 + want.abs().max())
    none = (labels < 0) | (labels >= LABELS)
    if entropy_weight == 0.0:
        assert (loss[none] == 0).all()
    for got, grad in ((field.table_grad, table_grad), (field.head_grad, head_grad)):
        assert torch.linalg.norm(got.double() - grad) <= 2.0**-4 * torch.linalg.norm(grad)
    if bits is None:
        return
    # the optimizer did with these gradients what its definition says
    rates = field.optimizer.groups[0]
    at = 0
    first, second = field.optimizer.moments()
    for grad, start in ((field.table_grad, field.optimizer.offsets[0]), (field.head_grad, field.optimizer.offsets[1])):
        n = grad.numel()
        g = grad.flatten().cpu().numpy()
        zero = np.zeros(n, np.float32)
        m, v = adamw_plain.moments32(zero, zero, g, 1.0, rates)
        (p, _, _), (off, _, _) = adamw_plain.step(before[at: at + n], g, zero, zero, 1.0, 1, rates)
        if bits == 8:
            m = adamw_plain.first_values(*adamw_plain.hold_first(m))[:n]
            v = adamw_plain.second_values(*adamw_plain.hold_second(v))[:n]
        assert np.array_equal(first[start: start + n].cpu().numpy(), m)
        assert np.array_equal(second[start: start + n].cpu().numpy(), v)
        now = (field.table if at == 0 else field.head).flatten().cpu().numpy()
        assert (np.abs(now - p) <= off).all()
        at += n


def test_gradient_against_differences():
    """The head's gradient against differences of the exact mean loss along a direction, on the head that the blocks stand for. The
    difference's own error: with |direction| = 1 and step h its third derivative times h^2 / 6; a logit moves by at most
    |row| <= 3, so that is below 27 h^2 = 3e-5 for h = 1e-3. The gradient's: the bound above."""
    from gsx_amd.label_field import LabelField
    field = LabelField(CODES, FEATURES, LABELS)
    codes, labels, weight = data(7)
    head = field.blocks.float().double()
    table = field.table.double()
    rows = torch.where((codes >= 0)[:, None], table[codes.clamp(min=0).long()], 0) * field.scale
    assert rows.norm(dim=1).max() <= 3
    given = (labels >= 0) & (labels < LABELS)

    def mean_loss(w):
        log_q = torch.log_softmax(rows @ w.T, 1)
        chosen = log_q.gather(1, labels.clamp(0, LABELS - 1).long()[:, None])[:, 0]
        return (-torch.where(given, chosen, 0) * weight.double()).mean()

    field.step_labels(codes, labels, weight)
    grad = field.head_grad.double()
    g = torch.Generator("cuda").manual_seed(8)
    for _ in range(4):
        d = torch.randn(head.shape, device="cuda", generator=g, dtype=torch.float64)
        d /= d.norm()
        slope = (mean_loss(head + 1e-3 * d) - mean_loss(head - 1e-3 * d)) / 2e-3
        assert abs(slope - (grad * d).sum()) <= 2.0**-4 * grad.norm() / (1 - 2.0**-4) + 3e-5


@pytest.mark.parametrize("rows,top", [(1, 5), (1, LABELS), (ROWS, 3), (ROWS, LABELS)])
def test_answers(rows, top):
    """Rows and head in 4-bit blocks multiply to the last bit within a block; sums of blocks round once each, three of them for 70
    features, so a logit is off by 3 * 2^-24 of its terms' magnitudes, twice that between a logit and the row's sum; the logarithm,
    the exponents and the differences of values up to `size` add 160 + 8 size roundings."""
    from gsx_amd import fields
    from gsx_amd.label_field import LabelField
    field = LabelField(CODES, FEATURES, LABELS)
    codes, labels, _ = data(9)
    codes, labels = codes[:rows], labels[:rows]
    x = fields.lookup(field.table, codes, field.scale, out_dtype=torch.bfloat16)
    a, b = fields.quantize4(x).float().double(), fields.quantize4(field.head).float().double()
    z = a @ b.T
    log_q = torch.log_softmax(z, 1)
    size = (a.abs() @ b.abs().T).max() + log_q.abs().max()
    off = (160 + 16 * size.item()) * 2.0**-24
    q = field.answers(codes, top, labels)
    given = (labels >= 0) & (labels < LABELS)
    chosen = torch.where(given, log_q.gather(1, labels.clamp(0, LABELS - 1).long()[:, None])[:, 0], 0)
    assert (q.chosen - chosen).abs().max() <= off
    assert (q.entropy + (log_q.exp() * log_q).sum(1)).abs().max() <= off * (1 + log_q.abs().max())
    assert q.top_ids.shape == (rows, top)
    ids = q.top_ids.long()
    assert (ids.sort(1).values.diff(dim=1) > 0).all()
    assert (q.top_log_probs - log_q.gather(1, ids)).abs().max() <= off
    assert (q.top_log_probs - log_q.topk(top, 1).values).abs().max() <= off


def test_train_answer_teach():
    """Steps against labels, answers between them, and the answers as another field's teacher; the head's 4-bit blocks follow it."""
    from gsx_amd import fields
    from gsx_amd.label_field import LabelField
    codes, labels, weight = data(11)
    field = LabelField(CODES, FEATURES, LABELS, moments=8, weight_decay=0.01)
    pupil = LabelField(CODES, FEATURES, LABELS, seed=1, moments=32)
    for k in range(3):
        assert torch.isfinite(field.step_labels(codes, labels, weight)).all()
        q = field.answers(codes, LABELS)
        assert torch.equal(field.head_blocks4().float(), fields.quantize4(field.head).float())
        before = pupil.table.clone()
        loss = pupil.step(codes, q.top_ids, q.top_log_probs, weight)
        assert torch.isfinite(loss).all() and (loss >= -1e-4).all()
        assert torch.isfinite(pupil.table).all() and not torch.equal(pupil.table, before)
    assert field.optimizer.steps.item() == 3


def test_answers_replayed():
    """A captured answer follows the codes and the head, with steps and answers of the program between the replays; what a capture
    lays out is not what eager calls read."""
    from gsx_amd.label_field import LabelField
    field, other = LabelField(CODES, FEATURES, LABELS), LabelField(CODES, FEATURES, LABELS, seed=3, moments=8)
    codes, labels, weight = data(13)
    asked = codes[:7].clone()
    other.answers(asked, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = field.answers(asked, 4)
    for k in range(4):
        asked.copy_(codes[7 * k: 7 * k + 7])
        graph.replay()
        eager = field.answers(asked, 4)
        torch.cuda.synchronize()
        for a, b in zip(q[:5], eager[:5]):
            assert torch.equal(a, b)
        other.step_labels(codes, labels, weight)
        field.step_labels(codes, labels, weight)
        torch.cuda.synchronize()


def test_command_runs():
    from gsx_amd.label_field import main
    agree = main(["--gaussians", "20000", "--steps", "3", "--labels", "40", "--cells", "12", "--given", "--moments", "8",
                  "--decay", "0.01", "--answers", "3"])
    assert 0.0 <= agree <= 1.0


def test_refusals():
    from gsx_amd._lib import GsxHipError
    from gsx_amd.label_field import LabelField
    field = LabelField(4, 8, 5)
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    with pytest.raises(GsxHipError):
        field.step_labels(empty, empty)
    with pytest.raises(GsxHipError):
        LabelField(4, 8, 5, moments=16)
    with pytest.raises(GsxHipError):
        LabelField(4, 8, 5, weight_decay=0.1)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(GsxHipError):
        field.step_labels(one, one.long())
    for top in (6, 65):  # more than there are labels, more than are kept
        with pytest.raises(GsxHipError):
            field.answers(one, top)
