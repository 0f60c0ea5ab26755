"""Log probabilities, entropies, top alternatives and their gradient against the definition in 64 bits: every way by the sizes,
ties, masks, rows without labels or without anything, strides, streams, graphs, and the gradient against differences."""
import numpy as np
import pytest

import logprobs_plain as plain
from logprobs_ways import WAYS

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAMES = {"f32": "f", "bf16": "DF16b", "f16": "DF16_"}


def _put(x, kind, pad=0):
    """A matrix between columns of NaN."""
    rows, cols = x.shape
    room = torch.full((rows, cols + pad), float("nan"), dtype=DTYPES[kind], device="cuda")
    t = room[:, pad // 2: pad // 2 + cols]
    t.copy_(torch.from_numpy(x))
    return t


def _make(rows, vocab, kind, seed, pad=0, spread=2.0, shut=0.01):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)
    x[rng.random((rows, vocab)) < shut] = -np.inf
    ids = rng.integers(0, vocab, rows)
    x[np.arange(rows), ids] = rng.standard_normal(rows) + 2
    ids[rng.random(rows) < 0.2] = -1
    return _put(x, kind, pad), torch.from_numpy(ids.astype(np.int32)).cuda()


def _equal_nan(a, b):
    return (np.isnan(a) & np.isnan(b)) | (a == b)


def _close(got, want, off):
    with np.errstate(invalid="ignore"):
        return (_equal_nan(got, want) | (np.abs(got - want) <= off)).all()


def _half_step(kind, size):
    if kind == "f32":
        return 0.0
    t = torch.finfo(DTYPES[kind])
    return t.eps / 2 * np.maximum(size, t.smallest_normal)


def _in_range(kind, x):
    """x, infinite where the type holds nothing as large (float16 from 65520 on: 65504 and half a step)."""
    most = 65520.0 if kind == "f16" else 3.39e38
    with np.errstate(invalid="ignore"):
        return np.where(np.abs(x) >= most, np.sign(x) * np.inf, x)


def _check(z, ids, top, temperature=1.0, gl=None, gh=None, rows=None):
    """Scores, the gradient of the same pass and that of a later call, row by row (all, or those given)."""
    from gsx_amd import fields
    n, vocab = z.shape
    kind = {v: k for k, v in DTYPES.items()}[z.dtype]
    rng = np.random.default_rng(7)
    gl = rng.standard_normal(n).astype(np.float32) if gl is None else np.asarray(gl, np.float32)
    gh = rng.standard_normal(n).astype(np.float32) if gh is None else np.asarray(gh, np.float32)
    up, up_h = torch.from_numpy(gl).cuda(), torch.from_numpy(gh).cuda()
    grad = torch.full((n, vocab + 3), 7.0, dtype=z.dtype, device="cuda")
    r = fields.log_probs(z, ids, top, temperature, grad_scale=0.5, row_grad=up, entropy_scale=2.0, entropy_grad=up_h,
                         grad=grad[:, :vocab])
    later = fields.log_probs_backward(z, r.row_stats, ids, up, up_h, temperature, grad_scale=0.5, entropy_scale=2.0)
    alone = fields.log_probs(z, ids, top, temperature)
    assert (grad[:, vocab:] == 7).all()
    for a, b in zip(r[:5], alone[:5]):
        assert torch.equal(a.nan_to_num(nan=3e38), b.nan_to_num(nan=3e38))
    host = [t.double().cpu().numpy() for t in (z, r.chosen, r.entropy, r.top_log_probs, grad[:, :vocab], later, r.row_stats)]
    zz, chosen, entropy, logs, g, g2, stats = host
    top_ids = r.top_ids.cpu().numpy()
    known = ids.cpu().numpy() if ids is not None else np.full(n, -1)
    known = np.where((known >= 0) & (known < vocab), known, -1)
    for i in range(n) if rows is None else rows:
        up_i = 0.5 * float(gl[i]) if known[i] >= 0 else 0.0
        want, off = plain.row(zz[i], known[i], temperature, up_i, 2.0 * float(gh[i]), top)
        assert np.array_equal(top_ids[i], want[2]), (i, top_ids[i], want[2])
        assert _close(chosen[i], want[0], off[0]), (i, chosen[i], want[0], off[0])
        assert _close(entropy[i], want[1], off[1]), (i, entropy[i], want[1], off[1])
        assert _close(stats[i, 2], want[1], off[1])
        assert _close(logs[i], want[3], off[2]), (i, np.abs(logs[i] - want[3]).max())
        room = off[3] + _half_step(kind, np.abs(want[4]) + off[3])
        held = _in_range(kind, want[4])
        assert _close(g[i], held, room), (i, np.nanmax(np.abs(g[i] - held) - room))
        assert _close(g2[i], held, room), (i, np.nanmax(np.abs(g2[i] - held) - room))
    return r


CASES = [(kind, *way[:3]) for kind in DTYPES for way in WAYS[NAMES[kind]]]


@pytest.mark.parametrize("kind,rows,vocab,top", CASES)
def test_every_way_against_64_bits(kind, rows, vocab, top):
    print(f"[case] log probabilities {rows} x {vocab} {kind}, {top} alternatives", flush=True)
    z, ids = _make(rows, vocab, kind, rows + vocab, pad=5)
    some = None if rows * vocab < 500_000 else sorted({0, 1, rows // 2, rows - 1} & set(range(rows)))
    _check(z, ids, top, rows=some)


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 1, 0), (4, 2, 2), (300, 7, 7), (70, 63, 63), (2, 64, 64), (1, 65, 64)])
def test_small_rows(kind, rows, vocab, top):
    z, ids = _make(rows, vocab, kind, vocab, shut=0.1)
    _check(z, ids, top)


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("temperature", [1e-6, 0.3, 7.0, 1e6])
def test_temperatures(kind, temperature):
    for rows, vocab, top in ((20, 150, 5), (5, 3001, 20), (2, 20_000, 20)):
        z, ids = _make(rows, vocab, kind, 3)
        _check(z, ids, top, temperature)


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(9, 150, 8), (9, 150, 64), (5, 2000, 64), (5, 5000, 20), (193, 12_001, 64),
                                            (9, 40_003, 64)])
def test_ties_go_to_the_lowest_index(kind, rows, vocab, top):
    """Untrained rows: all equal; a few values only; zeros of both signs; the largest value on more places than alternatives."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(-2, 3, (rows, vocab)).astype(np.float32)
    x[0] = 0.25
    x[1] = np.where(rng.random(vocab) < 0.5, -0.0, 0.0)
    x[2] = np.where(rng.random(vocab) < 0.5, -1.0, -np.inf)
    x[3, :] = -np.arange(vocab) // 100
    z = _put(x, kind, 3)
    ids = torch.arange(rows, dtype=torch.int32, device="cuda")
    _check(z, ids, top, rows=range(min(rows, 9)))


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(12, 150, 8), (12, 150, 40), (12, 1500, 64), (12, 3500, 20), (200, 10_000, 64),
                                            (12, 30_000, 64)])
def test_rows_with_little_or_nothing_open(kind, rows, vocab, top):
    rng = np.random.default_rng(5)
    x = np.full((rows, vocab), -np.inf, np.float32)
    for i, n in enumerate((0, 1, 2, 5, top - 1, top, top + 1)):
        at = rng.choice(vocab, n, replace=False)
        x[i, at] = rng.standard_normal(n)
    x[7:] = rng.standard_normal((rows - 7, vocab))
    x[7, 3], x[8, vocab - 1], x[9, 0], x[9, 5] = np.nan, np.inf, np.nan, np.inf
    x[10, 1], x[10, 2] = -np.nan, np.inf
    x[11, 100] = 3e38 if kind != "f16" else 6e4  # so far above the others that they have no share
    ids = torch.full((rows,), 3, dtype=torch.int32, device="cuda")
    ids[5], ids[6] = vocab, -(2**31)
    z = _put(x, kind)
    _check(z, ids, top, rows=range(12))


def test_rows_without_an_upstream_gradient_have_none_whatever_they_hold():
    from gsx_amd import fields
    for vocab in (100, 1000, 5000):
        z = torch.full((4, vocab), float("nan"), device="cuda")
        z[1], z[2] = float("inf"), 0.0
        ids = torch.tensor([-1, 5, 5, 5], dtype=torch.int32, device="cuda")
        up = torch.tensor([1.0, 0.0, 0.0, 1.0], device="cuda")
        r = fields.log_probs(z, ids, 1, grad_scale=1.0, row_grad=up)
        assert (r.grad[:3] == 0).all() and r.grad[3].isnan().all()
        assert r.chosen[0] == 0 and r.chosen[1:].isnan().tolist() == [True, False, True]
        assert torch.equal(fields.log_probs_backward(z, r.row_stats, ids, up)[:3], r.grad[:3])


def test_without_labels_and_without_alternatives():
    from gsx_amd import fields
    for vocab in (50, 3000, 50_000):
        z, _ = _make(3, vocab, "bf16", 1)
        r = _check(z, None, min(20, vocab))
        assert (r.chosen == 0).all()
        r = fields.log_probs(z)
        assert r.top_ids.shape == (3, 0) and r.grad is None
        _check(z, None, 0)


@pytest.mark.parametrize("vocab", [100, 700, 3000, 40_000])
def test_gradients_against_differences(vocab):
    """Along a direction v: f(z + h v) - f(z - h v) is 2 h <grad, v> but for h^3 of the third derivative (at most 6 |v|_inf^3 for
    log q, 20 (1 + ln vocab) times that for H) and the values' roundings."""
    from gsx_amd import fields
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((4, vocab)).astype(np.float32)
    v = rng.choice([-1.0, 1.0], (4, vocab)).astype(np.float32)
    h = 2.0**-6
    ids = torch.from_numpy(rng.integers(0, vocab, 4).astype(np.int32)).cuda()
    ends = []
    for s in (1, -1):
        r = fields.log_probs(torch.from_numpy(x.astype(np.float64) + s * h * v).float().cuda(), ids)
        ends.append((r.chosen.double(), r.entropy.double()))
    direction = torch.from_numpy(v).cuda().double()
    z = torch.from_numpy(x).cuda()
    slack = 400 * 2.0**-24 * (1 + np.log(vocab))  # of either value: what its sums of up to 129 and a dozen roundings may lose
    for k, how in enumerate((dict(grad_scale=1.0), dict(entropy_scale=1.0))):
        along = (fields.log_probs(z, ids, **how).grad.double() * direction).sum(1)
        change = (ends[0][k] - ends[1][k]) / (2 * h)
        third = (6 if k == 0 else 20 * (1 + np.log(vocab))) * h * h / 6
        assert ((along - change).abs() <= third + slack / h + 1e-5 * (1 + along.abs())).all(), (along, change)


def test_top_alternatives_are_a_teacher():
    """One field's alternatives as another's teacher: the distance to itself is 0 where all its labels are alternatives."""
    from gsx_amd import fields
    z, _ = _make(50, 40, "f32", 9, shut=0.2)
    r = fields.log_probs(z, top=40, temperature=2.0)
    loss, _, grad = fields.distill(z, r.top_ids, r.top_log_probs * 2.0, temperature=2.0, grad_scale=1.0)
    # log p and log q each a few roundings of values up to 12
    assert loss.abs().max().item() <= 4 * 64 * 2.0**-24 * 12 and grad.abs().max().item() <= 2 * 64 * 2.0**-24 * 12


def test_rows_behind_2_31_logits():
    from gsx_amd import fields
    rows, vocab = 36_000, 60_001
    print(f"[case] {rows} x {vocab}", flush=True)
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    tail, ids = _make(3, vocab, "bf16", 4)
    z[-3:] = tail
    all_ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    all_ids[-3:] = ids
    r = fields.log_probs(z, all_ids, 5, grad_scale=1.0)
    want = fields.log_probs(torch.cat([tail, torch.zeros(300, vocab, dtype=z.dtype, device="cuda")]),
                            torch.cat([ids, all_ids[:300]]), 5, grad_scale=1.0)
    for a, b in zip(r[:4], want[:4]):
        assert torch.equal(a[-3:], b[:3])
    assert torch.equal(r.grad[-3:], want.grad[:3])
    later = fields.log_probs_backward(z, r.row_stats, all_ids)
    assert torch.equal(later[-3:], fields.log_probs_backward(tail, r.row_stats[-3:].clone(), ids))


@pytest.mark.parametrize("rows,vocab", [(500, 150), (3, 40_000), (200, 20_000)])
def test_replays_of_a_captured_call(rows, vocab):
    from gsx_amd import fields
    z, ids = _make(rows, vocab, "f32", 6)
    fields.log_probs(z, ids, 5, grad_scale=1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = fields.log_probs(z, ids, 5, grad_scale=1.0)
        later = fields.log_probs_backward(z, r.row_stats, ids)
    for k in range(4):
        fresh, _ = _make(rows, vocab, "f32", 60 + k)
        z.copy_(fresh)
        graph.replay()
        want = fields.log_probs(fresh, ids, 5, grad_scale=1.0)
        for a, b in zip(r, want):
            assert torch.equal(a, b)
        assert torch.equal(later, fields.log_probs_backward(fresh, want.row_stats, ids))


def test_calls_on_two_streams_at_once():
    from gsx_amd import fields
    cases = [_make(2, 100_000, "f32", 20 + k) for k in range(2)]
    want = [fields.log_probs(z, ids, 20) for z, ids in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[fields.log_probs(z, ids, 20, stream=s) for _ in range(10)] for (z, ids), s in zip(cases, streams)]
    torch.cuda.synchronize()
    for calls, w in zip(got, want):
        for r in calls:
            for a, b in zip(r[:5], w[:5]):
                assert torch.equal(a, b)


def test_refusals():
    from gsx_amd import fields
    from gsx_amd.backend import GsxHipError
    z, ids = torch.zeros(3, 10, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    up = torch.ones(3, device="cuda")
    r = fields.log_probs(z, ids, 2)
    for call in (lambda: fields.log_probs(z, ids.long()), lambda: fields.log_probs(z, ids[:2]),
                 lambda: fields.log_probs(z, ids, 11), lambda: fields.log_probs(z, ids, -1),
                 lambda: fields.log_probs(torch.zeros(3, 100, device="cuda"), ids, 65), lambda: fields.log_probs(z.double(), ids),
                 lambda: fields.log_probs(z, ids, temperature=0.0), lambda: fields.log_probs(z, ids, row_grad=up),
                 lambda: fields.log_probs(z, ids, grad_scale=1.0, entropy_grad=up), lambda: fields.log_probs(z, ids, grad=z),
                 lambda: fields.log_probs(z, ids, grad_scale=1.0, grad=z), lambda: fields.log_probs(z.T, ids),
                 lambda: fields.log_probs(z, ids, grad_scale=1.0, grad=z.half()), lambda: fields.log_probs(z.cpu(), ids),
                 lambda: fields.log_probs_backward(z, r.row_stats[:, :2], ids), lambda: fields.log_probs_backward(z, up, ids),
                 lambda: fields.log_probs_backward(z, r.row_stats, ids, up[:2])):
        with pytest.raises(GsxHipError):
            call()


@pytest.mark.parametrize("kind", list(DTYPES))
@pytest.mark.parametrize("vocab,top", [(3, 3), (150, 3), (250, 8), (300, 5), (500, 5), (150, 20), (900, 7), (1500, 64), (5000, 9)])
def test_nan_of_either_sign_comes_first(kind, vocab, top):
    """In the order of their indices, the first and the last logit among them, before +inf; equal numbers and zeros of either sign
    follow by their indices."""
    from gsx_amd import fields
    bits = {"f32": torch.int32, "bf16": torch.int16, "f16": torch.int16}[kind]
    minus = {"f32": -(2**31) + 0x7FC00000, "bf16": -(2**15) + 0x7FC0, "f16": -(2**15) + 0x7E00}[kind]
    z = torch.zeros(6, vocab, device="cuda", dtype=DTYPES[kind])
    z[:, 1::2] = -0.0
    z.view(bits)[0, 0] = minus
    z[1, vocab - 1] = float("nan")
    z.view(bits)[2, vocab - 1] = minus
    z[2, 0] = float("nan")
    z[2, 1] = float("inf")
    z.view(bits)[3, 1] = minus
    z[3, 0] = float("inf")
    z[4] = -float("inf")
    z.view(bits)[4, vocab // 2] = minus
    r = fields.log_probs(z, None, top)
    ids = r.top_ids.cpu().numpy()
    for i, row in enumerate(z.float().cpu().numpy()):
        assert np.array_equal(ids[i], plain.order(row, top)), i
    assert r.entropy[:5].isnan().all() and r.entropy[5].isfinite()


@pytest.mark.parametrize("kind", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,stretch", [(200, 3001, 3001), (200, 5003, 5003), (200, 16_001, 16_001), (200, 29_999, 29_999),
                                                (200, 61_001, 61_001), (3, 40_003, 4096), (300, 150_001, 16_384)])
@pytest.mark.parametrize("top", [5, 64])
def test_hundreds_of_logits_at_the_last_alternatives_value(kind, rows, vocab, stretch, top):
    """A workgroup thins its candidates out where there are more than 160 of them, up to 1024: `stretch` logits are what one has at
    least. A row in 8 has 150 equal ones in each such stretch, the others 170 to 1000, and three larger ones."""
    print(f"[case] {rows} x {vocab} {kind}, {top} alternatives", flush=True)
    from gsx_amd import fields
    rng = np.random.default_rng(vocab + top)
    x = (rng.standard_normal((8, vocab)) - 6).astype(np.float32).clip(-12, -1)
    for i, each in enumerate((150, 170, 250, 300, 500, 700, 900, 1000)):
        for start in range(0, vocab, stretch):
            span = min(stretch, vocab - start)
            x[i, start + rng.choice(span, min(each, span), replace=False)] = 0.75
        x[i, rng.choice(vocab, 3, replace=False)] = (1.0, 2.0, 1.5)
    want = np.stack([plain.order(x[i], top) for i in range(8)])[np.arange(rows) % 8]
    z = _put(x, kind).repeat(-(-rows // 8), 1)[:rows]
    got = fields.log_probs(z, top=top)
    assert np.array_equal(got.top_ids.cpu().numpy(), want)
    assert (got.top_log_probs.diff(dim=1) <= 0).all()


@pytest.mark.parametrize("kind", list(DTYPES))
@pytest.mark.parametrize("vocab,top", [(149, 3), (301, 1), (301, 8), (383, 3), (901, 5), (1023, 8), (1501, 20), (5001, 9), (40_001, 9)])
def test_nan_keeps_its_order_in_rows_that_begin_anywhere(kind, vocab, top):
    """Rows of an odd length begin at every place between two multiples of 16 bytes: NaN of different bits before the first whole
    vector, in vectors and behind the last one are equal, and come by their indices."""
    from gsx_amd import fields
    rows, bits = 16, {"f32": torch.int32, "bf16": torch.int16, "f16": torch.int16}[kind]
    quiet = {"f32": 0x7FC00000, "bf16": 0x7FC0, "f16": 0x7E00}[kind]
    full = {"f32": 0x7FFFFFFF, "bf16": 0x7FFF, "f16": 0x7FFF}[kind]
    minus = -(2**31) if kind == "f32" else -(2**15)
    z = torch.zeros(rows, vocab, device="cuda", dtype=DTYPES[kind])
    z[:, 2] = float("inf")
    for i, at in enumerate(((0, 100), (0, 1, 100), (3, 100), (0, vocab - 1), (100, vocab - 1), (1, vocab // 2, vocab - 2))):
        for j, k in enumerate(at):
            z.view(bits)[i::6, k] = (quiet, full, minus + quiet, minus + full)[(i + j) % 4]
    r = fields.log_probs(z, None, top)
    ids = r.top_ids.cpu().numpy()
    for i, row in enumerate(z.float().cpu().numpy()):
        assert np.array_equal(ids[i], plain.order(row, top)), (i, ids[i])
    assert r.entropy.isnan().all()
