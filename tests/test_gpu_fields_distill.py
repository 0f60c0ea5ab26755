"""Distillation from a teacher's top logits against its definition in 64 bits: types, lengths, strides, masks, rows without
entries, repeated entries, refusals, and the gradient against differences."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}


def _want(z, ids, t, temperature, weight, upstream):
    """(loss, gradient, the sum of its terms' magnitudes) in float64, row by row."""
    rows, vocab = z.shape
    loss, grad, size = np.zeros(rows), np.zeros(z.shape), np.zeros(z.shape)
    for r in range(rows):
        valid = (ids[r] >= 0) & (ids[r] < vocab) & (t[r] != -np.inf)
        if not valid.any() or weight[r] == 0:
            continue
        tt = t[r][valid] / temperature
        p = np.exp(tt - tt.max())
        p /= p.sum()
        log_p = tt - tt.max() - np.log(np.exp(tt - tt.max()).sum())
        if (z[r] == -np.inf).all():
            loss[r] = np.inf
            continue
        zz = z[r] / temperature
        with np.errstate(invalid="ignore"):
            all_q = (zz - zz.max()) - np.log(np.exp(zz - zz.max()).sum())  # so ordered for logits of 1e38
            q = np.exp(all_q)
        entry = ids[r][valid]
        log_q = all_q[entry]
        live = p > 0
        loss[r] = weight[r] * temperature**2 * (p[live] * (log_p[live] - log_q[live])).sum()
        g, s = q.copy(), q.copy()
        np.subtract.at(g, entry, p)
        np.add.at(s, entry, p)
        grad[r] = weight[r] * upstream[r] * temperature * g
        size[r] = np.abs(weight[r] * upstream[r]) * temperature * s
    return loss, grad, size


def _make(rows, vocab, top, kind, seed, pad=0, spread=3.0):
    rng = np.random.default_rng(seed)
    base = torch.full((rows, vocab + pad), float("nan"), device="cuda").to(DTYPES[kind])
    z = base[:, pad // 2: pad // 2 + vocab]
    z.copy_(torch.from_numpy((rng.standard_normal((rows, vocab)) * spread).astype(np.float32)))
    ids = np.stack([rng.permutation(vocab)[:top] if top <= vocab else rng.integers(0, vocab, top) for _ in range(rows)])
    ids = ids.reshape(rows, top)
    t = (rng.standard_normal((rows, top)) * 2).astype(np.float32)
    return z, ids.astype(np.int32), t


def _check(z, ids, t, temperature=1.0, weight=None, upstream=None, pad=0):
    from gsx_amd import fields
    rows, vocab = z.shape
    dev = dict(device="cuda")
    w = torch.from_numpy(weight).cuda() if weight is not None else None
    up = np.linspace(0.5, 1.5, rows).astype(np.float32) if upstream is None else upstream
    i, tt = torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
    base = torch.full((rows, vocab + pad), 3.0, dtype=z.dtype, **dev)
    step = base[:, pad - pad // 2: pad - pad // 2 + vocab]
    print(f"[case] distill {rows} x {vocab} {z.dtype} top {ids.shape[1]} T {temperature} pad {pad}", flush=True)
    loss, stats, got = fields.distill(z, i, tt, temperature, w, grad_scale=0.75, grad=step)
    alone, stats2, none = fields.distill(z, i, tt, temperature, w)
    assert none is None and torch.equal(alone.nan_to_num(7), loss.nan_to_num(7))
    apart = fields.distill_backward(z, stats, i, tt, torch.from_numpy(up).cuda(), temperature, w)
    ones = np.ones(rows, np.float32) if weight is None else weight
    zz = z.double().cpu().numpy()
    want, grad, grad_size = _want(zz, ids, t.astype(np.float64), temperature, ones.astype(np.float64), np.full(rows, 0.75))
    _, grad_apart, apart_size = _want(zz, ids, t.astype(np.float64), temperature, ones.astype(np.float64), up.astype(np.float64))
    kind = {v: k for k, v in DTYPES.items()}[z.dtype]
    finite = np.isfinite(want)
    have = loss.double().cpu().numpy()
    assert np.array_equal(have[~finite], want[~finite], equal_nan=True)
    # Exponents up to R = the row's range over T are rounded twice to 2^-24 of themselves, the sum of positive terms once per
    # addition of a tree of at most 64 + log2(vocab) steps per thread and join; every log p - log q is off by that and a few
    # roundings of its own size
    with np.errstate(invalid="ignore"):
        fin = np.where(np.isfinite(zz), zz, np.nan)
        span = np.nan_to_num(np.nanmax(fin, 1, initial=-1e30) - np.nanmin(fin, 1, initial=1e30)).clip(0, 104 * temperature)
        span_t = np.nan_to_num(t.max(1) - np.where(t == -np.inf, t.max(1)[:, None], t).min(1), posinf=0).clip(0)
    sums = 2.0**-24 * (64 + vocab / 256 + 16)
    off = (span + span_t) / temperature * 2.0**-22 + sums + ids.shape[1] * 2.0**-24 + 2.0**-21
    size = np.abs(ones) * temperature**2 * (1 + (span + span_t) / temperature + np.log(vocab) + np.log(ids.shape[1])) + np.abs(want)
    with np.errstate(invalid="ignore"):
        assert (np.abs(have - want)[finite] <= (off * size)[finite]).all()
    for g, wg, terms in ((got, grad, grad_size), (apart, grad_apart, apart_size)):
        g = g.double().cpu().numpy()
        err = np.abs(g - wg)
        # q and p are off by `off` of themselves, which their difference keeps; then one rounding
        lim = np.abs(wg) * UNIT[kind] + off[:, None] * terms + (2.0**-25 if kind == "f16" else 2.0**-126)
        assert (err <= lim).all(), (err - lim).max()
    keep = torch.ones_like(base, dtype=torch.bool)
    keep[:, pad - pad // 2: pad - pad // 2 + vocab] = False
    assert (base[keep] == 3).all()
    return loss, got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,top,pad,temperature", [
    (1, 1, 1, 0, 1.0), (5, 2, 1, 0, 2.0), (3, 7, 7, 1, 1.0), (300, 20, 5, 0, 1.0), (64, 150, 8, 0, 2.0), (70, 151, 8, 3, 0.5),
    (9, 255, 16, 0, 1.0), (9, 1000, 64, 8, 2.0), (5, 1025, 300, 1, 1.0), (4, 4097, 64, 0, 3.0), (3, 8192, 1024, 0, 1.0),
    (2, 50001, 64, 1, 2.0), (1, 131072, 64, 0, 2.0), (40, 9000, 33, 2, 1.0), (3, 131073, 5, 0, 1.0), (300, 2049, 8, 0, 1.0),
    (17, 70000, 16, 8, 1.0), (600, 20000, 16, 0, 1.0)])
def test_distill(rows, vocab, top, pad, temperature, kind):
    z, ids, t = _make(rows, vocab, top, kind, vocab + rows, pad)
    weight = np.random.default_rng(rows).uniform(0.2, 2, rows).astype(np.float32)
    _check(z, ids, t, temperature, weight if rows % 2 else None, pad=pad)


@pytest.mark.parametrize("rows,vocab", [(12, 40), (12, 3000), (12, 70001)])
def test_masked_entries_rows_and_logits(rows, vocab):
    z, ids, t = _make(rows, vocab, 6, "f32", vocab, pad=1)
    rng = np.random.default_rng(0)
    inf = float("inf")
    ids[0] = -1                       # no entry
    ids[1, 1:] = vocab                # one entry, the others past the vocabulary
    t[2] = -np.inf                    # entries of no mass
    t[3, :3] = -np.inf
    weight = np.ones(rows, np.float32)
    weight[4] = 0
    z[4] = float("nan")               # a padding row's logits mean nothing
    z[0, 0] = float("nan")
    blocked = torch.from_numpy(rng.random(vocab) < 0.6).cuda()
    z[5, blocked] = -inf              # a mask on most logits, the teacher's entries among them or not
    z[6] = -inf                       # nothing left
    z[7, blocked] = torch.finfo(torch.float32).min
    z[8] = torch.finfo(torch.float32).min  # all equal, at the lowest value
    z[9, : vocab // 2] = -inf
    t[10] = [1e4, -1e4, 0, 0, 5, 6]   # mass on one entry
    z[11] = 0
    z[11, ids[11, 0]] = 3e38          # the student is sure
    loss, grad = _check(z, ids, t, 1.0, weight, pad=1)
    assert loss[0] == 0 and loss[2] == 0 and loss[4] == 0 and loss[6] == inf
    assert (grad[[0, 2, 4, 6]] == 0).all()


@pytest.mark.parametrize("vocab", [30, 2000, 70000])
def test_non_finite_logits_give_nan_in_their_row_only(vocab):
    from gsx_amd import fields
    z, ids, t = _make(6, vocab, 4, "f32", 1)
    z[1, 3], z[2, vocab - 1], z[3] = float("nan"), float("inf"), float("nan")
    t[4, 2] = float("nan")
    i, tt = torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
    loss, stats, grad = fields.distill(z, i, tt, grad_scale=1.0)
    assert torch.isnan(loss).tolist() == [False, True, True, True, True, False]
    back = fields.distill_backward(z, stats, i, tt)
    for g in (grad, back):
        assert torch.isfinite(g[[0, 5]]).all() and torch.isnan(g[[1, 2, 3]]).all()
        assert torch.isnan(g[4][i[4].long()]).all()


@pytest.mark.parametrize("top", [2, 64, 65, 1000])
@pytest.mark.parametrize("vocab", [9, 5000])
def test_repeated_entries_add_up(vocab, top):
    z, ids, t = _make(5, vocab, top, "f32", 2)
    ids[0] = 3
    ids[1, ::2] = 1
    ids[2, -1] = ids[2, 0]
    _check(z, ids, t, 2.0)


def test_gradient_against_differences():
    """Central differences of the 64-bit loss, with steps of 2^-12: their own error is the third derivative's, below
    T^2 (1/T)^3 h^2 / 6, and 2^-52 / h of the loss."""
    from gsx_amd import fields
    z, ids, t = _make(3, 50, 6, "f32", 4)
    temperature, h = 1.5, 2.0**-12
    _, _, grad = fields.distill(z, torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda(), temperature, grad_scale=1.0)
    zz, ones = z.double().cpu().numpy(), np.ones(3)
    for r, j in ((0, 0), (1, ids[1, 0]), (1, ids[1, 5]), (2, 49)):
        up, down = zz.copy(), zz.copy()
        up[r, j] += h
        down[r, j] -= h
        diff = (_want(up, ids, t.astype(float), temperature, ones, ones)[0][r] -
                _want(down, ids, t.astype(float), temperature, ones, ones)[0][r]) / (2 * h)
        # the gradient's own error: some 2^-20 of terms of size T
        assert abs(diff - grad[r, j].item()) <= h * h + 2.0**-38 + temperature * 2.0**-19


def test_distill_past_32_bit_offsets():
    from gsx_amd import fields
    rows, vocab = 33000, 65537  # 2^31 logits and some
    z = torch.zeros((rows, vocab), dtype=torch.float16, device="cuda")
    z[-1, 5] = 4
    ids = torch.full((rows, 1), 5, dtype=torch.int32, device="cuda")
    t = torch.zeros((rows, 1), device="cuda")
    print("[case] distill past 2^31 logits", flush=True)
    loss, stats, grad = fields.distill(z, ids, t, grad_scale=1.0)
    lse = np.log(vocab - 1 + np.exp(4.0))
    # a sum of 65537 terms: see _check
    assert abs(loss[0].item() - np.log(vocab)) < 1e-4 and abs(loss[-1].item() - (lse - 4)) < 1e-4
    want = np.exp(4 - lse) - 1
    assert abs(grad[-1, 5].item() - want) <= abs(want) * 2.0**-11 + 1e-6
    del grad
    back = fields.distill_backward(z, stats, ids, t)
    assert abs(back[-1, 5].item() - want) <= abs(want) * 2.0**-11 + 1e-6


@pytest.mark.parametrize("rows,vocab", [(3, 200_000), (500, 300), (600, 12000)])
def test_distill_repeats_bit_for_bit_and_on_another_stream(rows, vocab):
    from gsx_amd import fields
    z, ids, t = _make(rows, vocab, 8, "bf16", 5)
    i, tt = torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
    loss, stats, grad = fields.distill(z, i, tt, grad_scale=1.0)
    back = fields.distill_backward(z, stats, i, tt)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(4):
        a = fields.distill(z, i, tt, grad_scale=1.0, stream=s)
        b = fields.distill_backward(z, a[1], i, tt, stream=s)
        s.synchronize()
        assert torch.equal(a[0], loss) and torch.equal(a[1], stats) and torch.equal(a[2], grad) and torch.equal(b, back)


def test_distill_in_a_graph():
    from gsx_amd import fields
    z, ids, t = _make(2, 100_000, 8, "f32", 6)
    i, tt = torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
    grad = torch.zeros_like(z)
    fields.distill(z, i, tt, grad_scale=1.0, grad=grad)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _, _ = fields.distill(z, i, tt, grad_scale=1.0, grad=grad)
    for k in range(4):
        z.copy_(torch.randn(2, 100_000, device="cuda", generator=torch.Generator("cuda").manual_seed(k)))
        grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = fields.distill(z, i, tt, grad_scale=1.0)
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[2]), k


def test_no_rows():
    from gsx_amd import fields
    z = torch.empty(0, 10, device="cuda")
    loss, stats, grad = fields.distill(z, torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                                       torch.empty(0, 2, device="cuda"), grad_scale=1.0)
    assert loss.shape == (0,) and grad.shape == (0, 10)


def test_distill_refusals():
    from gsx_amd import fields
    from gsx_amd._lib import GsxHipError
    z = torch.zeros(4, 50, device="cuda")
    i, t = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.zeros(4, 3, device="cuda")
    w = torch.ones(4, device="cuda")
    stats = torch.ones(4, 2, device="cuda")
    for bad in (lambda: fields.distill(z.double(), i, t), lambda: fields.distill(z.cpu(), i, t),
                lambda: fields.distill(z, i.long(), t), lambda: fields.distill(z, i, t.half()),
                lambda: fields.distill(z, i[:3], t[:3]), lambda: fields.distill(z, i, t[:, :2]),
                lambda: fields.distill(z, i[:, :0], t[:, :0]), lambda: fields.distill(z.T, i, t),
                lambda: fields.distill(z, i, t, temperature=0.0), lambda: fields.distill(z, i, t, temperature=-1.0),
                lambda: fields.distill(z, i, t, temperature=float("nan")),
                lambda: fields.distill(z, i, t, temperature=float("inf")),
                lambda: fields.distill(z, i, t, row_weight=w[:3]), lambda: fields.distill(z, i, t, row_weight=w.half()),
                lambda: fields.distill(z, i, t, grad=torch.zeros_like(z)),
                lambda: fields.distill(z, i, t, grad_scale=1.0, grad=z),
                lambda: fields.distill(z, i, t, grad_scale=1.0, grad=torch.zeros(4, 49, device="cuda")),
                lambda: fields.distill(z, i, t, grad_scale=1.0, grad=torch.zeros(4, 50, device="cuda").half()),
                lambda: fields.distill(z[:, :0], i, t),
                lambda: fields.distill(z, torch.zeros(4, 1025, dtype=torch.int32, device="cuda"),
                                       torch.zeros(4, 1025, device="cuda")),
                lambda: fields.distill_backward(z, stats[:, :1], i, t), lambda: fields.distill_backward(z, stats.T[:2].T, i, t, w[:2]),
                lambda: fields.distill_backward(z, stats, i, t, grad=z)):
        with pytest.raises(GsxHipError):
            bad()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(37, 512, 16), (37, 513, 16), (37, 400, 62), (37, 400, 63), (37, 256, 80), (37, 300, 150),
                                            (50, 3, 2), (1, 33, 1)])
def test_rows_that_share_a_wave(rows, vocab, top, kind):
    """About the sizes up to which 16 lanes hold a row, four rows a wave: masks, repeated entries and NaN stay in their row."""
    z, ids, t = _make(rows, vocab, top, kind, vocab + top, pad=1)
    weight = np.ones(rows, np.float32)
    if rows > 1:
        ids[0] = -1
        ids[1] = ids[1, 0]
        ids[2, -1] = ids[2, 0]
        weight[3] = 0
        z[3] = float("nan")
        z[5, : vocab // 2] = -float("inf")
    _check(z, ids, t, 2.0, weight, pad=1)
