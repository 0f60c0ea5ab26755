"""Row lookup and its gradient against 64-bit sums: types, odd widths, strides, ids outside the table, frequent ids, refusals."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half a step of the type, relative: one rounding of the result (and one of the product before it)
STEP = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}


def _strided(rows, cols, pad, dtype, fill=None):
    """A [rows, cols] view whose rows lie cols + pad elements apart, starting at an odd element when pad is odd."""
    base = torch.empty((rows, cols + pad), dtype=dtype, device="cuda")
    base.fill_(float("nan") if fill is None else fill)
    return base[:, pad // 2: pad // 2 + cols], base


def _ids(count, table_rows, seed, outside=True):
    ids = np.random.default_rng(seed).integers(0, table_rows, count).astype(np.int32)
    if outside and count > 2:
        ids[::7] = -1
        ids[1::11] = -2**31
    return ids


def _lookup_want(table, ids, scale):
    fits = (ids >= 0) & (ids < table.shape[0])
    want = np.zeros((len(ids), table.shape[1]))
    want[fits] = table[ids[fits]].double().cpu().numpy() * float(np.float32(scale))
    return want


@pytest.mark.parametrize("pad", [0, 3, 8])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("count,table_rows,width", [(1, 1, 1), (1, 7, 4096), (63, 5, 385), (257, 100, 24), (33, 9, 8200)])
def test_lookup(count, table_rows, width, kind, out, pad):
    from gsx_amd import fields
    table, _ = _strided(table_rows, width, pad, DTYPES[kind])
    table.copy_(torch.randn(table_rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(width)))
    to, to_base = _strided(count, width, pad, DTYPES[out], fill=7.0)
    ids = _ids(count, table_rows, count)
    print(f"[case] lookup {count} of {table_rows} x {width} {kind}->{out} pad {pad}", flush=True)
    got = fields.lookup(table, torch.from_numpy(ids).cuda(), scale=1.7, out=to)
    want = _lookup_want(table.cpu(), ids, 1.7)
    err = np.abs(got.double().cpu().numpy() - want)
    # the product is rounded to float, that to the result's type; denormal results of f16 step by 2^-24
    assert (err <= np.abs(want) * (STEP[out] + STEP["f32"]) * 1.01 + (2.0**-25 if out == "f16" else 0)).all()
    outside = torch.ones_like(to_base, dtype=torch.bool)
    outside[:, pad // 2: pad // 2 + width] = False
    assert (to_base[outside] == 7).all()


def test_lookup_flags_ids_past_the_table_only():
    from gsx_amd import fields
    table = torch.full((4, 8), float("inf"), device="cuda")
    for ids, want in (([0, -1, 3], 0), ([0, 4, 3], 1), ([-1, 2**31 - 1], 1)):
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = fields.lookup(table, torch.tensor(ids, dtype=torch.int32, device="cuda"), out_of_range=flag)
        assert flag.item() == want
        assert [bool((r == 0).all()) for r in got] == [not 0 <= i < 4 for i in ids]


def test_lookup_of_an_empty_table_and_of_nothing():
    from gsx_amd import fields
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert (fields.lookup(torch.empty(0, 5, device="cuda"), ids) == 0).all()
    assert fields.lookup(torch.ones(2, 5, device="cuda"), ids[:0]).shape == (0, 5)
    assert (fields.lookup_backward(torch.empty(0, 5, device="cuda"), ids[:0], 3) == torch.zeros(3, 5, device="cuda")).all()
    assert fields.lookup_backward(torch.ones(3, 5, device="cuda"), ids, 0).shape == (0, 5)


def test_lookup_past_32_bit_offsets():
    from gsx_amd import fields
    rows, width = 2**21 + 3, 1024  # 2^31 elements and some
    table = torch.empty((rows, width), dtype=torch.float16, device="cuda")
    ids = torch.tensor([rows - 1, 2**21, 0, rows], dtype=torch.int32, device="cuda")
    for k, i in enumerate((rows - 1, 2**21, 0)):
        table[i] = k + 1
    print("[case] lookup past 2^31 elements", flush=True)
    assert fields.lookup(table, ids)[:, -1].tolist() == [1, 2, 3, 0]


def _backward_want(grad, ids, table_rows, scale, before=None):
    """Sums in 64 bits and, per element, the sum of magnitudes."""
    g = grad.double().cpu().numpy() * float(np.float32(scale))
    want = np.zeros((table_rows, g.shape[1]))
    size = np.zeros_like(want)
    fits = (ids >= 0) & (ids < table_rows)
    np.add.at(want, ids[fits], g[fits])
    np.add.at(size, ids[fits], np.abs(g[fits]))
    if before is not None:
        want += before
        size += np.abs(before)
    return want, size


def _backward_check(grad, ids, table_rows, scale=0.37, accumulate=False, pad=0):
    from gsx_amd import fields
    width = grad.shape[1]
    to, base = _strided(table_rows, width, pad, torch.float32, fill=0.25 if accumulate else float("nan"))
    dev = torch.from_numpy(ids).cuda()
    print(f"[case] lookup backward {grad.shape[0]} x {width} {grad.dtype} on {table_rows}, pad {pad}", flush=True)
    got = fields.lookup_backward(grad, dev, table_rows, scale=scale, grad_table=to, accumulate=accumulate)
    first = got.cpu().numpy().copy()
    before = np.full((table_rows, width), 0.25) if accumulate else None
    want, size = _backward_want(grad, ids, table_rows, scale, before)
    most = max(1, np.bincount(ids[(ids >= 0) & (ids < table_rows)], minlength=1).max())
    # a float sum of n terms in any order is within (n - 1) 2^-24 of the terms' magnitudes, to first order; the scale and the
    # final addition round twice more
    assert (np.abs(first - want) <= size * (most + 2) * 2.0**-24 * 1.01).all()
    if accumulate:
        to.fill_(0.25)
    again = fields.lookup_backward(grad, dev, table_rows, scale=scale, grad_table=to, accumulate=accumulate)
    assert np.array_equal(first, again.cpu().numpy())


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("count,table_rows,width,pad", [
    (1, 1, 1, 0), (1, 100, 385, 3), (77, 1001, 385, 0), (500, 3, 130, 1), (513, 70000, 2, 0), (2500, 300, 64, 4),
    (5000, 17, 257, 0), (20000, 9000, 96, 0), (3000, 65535, 8, 0), (3000, 65536, 12, 2), (70001, 5, 20, 0)])
def test_lookup_backward(count, table_rows, width, pad, kind, accumulate):
    grad, _ = _strided(count, width, pad, DTYPES[kind])
    grad.copy_(torch.randn(count, width, device="cuda", generator=torch.Generator("cuda").manual_seed(count)))
    _backward_check(grad, _ids(count, table_rows, width), table_rows, accumulate=accumulate, pad=pad)


@pytest.mark.parametrize("count", [300, 4096, 50000])
@pytest.mark.parametrize("pattern", ["one", "last", "outside", "two", "ascending"])
def test_lookup_backward_of_uneven_ids(count, pattern):
    """All ids equal, all outside (with NaN rows, which must not count), two alternating, each its own."""
    table_rows = count + 5 if pattern == "ascending" else 6
    ids = {"one": np.full(count, 2), "last": np.full(count, 5), "two": np.arange(count) % 2 * 3,
           "outside": np.where(np.arange(count) % 2, -1, 6), "ascending": np.arange(count)}[pattern].astype(np.int32)
    grad = torch.randn(count, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(count))
    if pattern == "outside":
        grad.fill_(float("nan"))
    if pattern != "outside":
        ids[5] = -3
        grad[5] = float("inf")
    clean = grad.clone()
    clean[torch.from_numpy((ids < 0) | (ids >= table_rows)).cuda()] = 0
    from gsx_amd import fields
    got = fields.lookup_backward(grad, torch.from_numpy(ids).cuda(), table_rows)
    want, size = _backward_want(clean, ids, table_rows, 1.0)
    most = np.bincount(ids[ids >= 0], minlength=1).max()
    assert (np.abs(got.cpu().numpy() - want) <= size * (most + 2) * 2.0**-24 * 1.01).all()


def test_lookup_gradient_against_differences():
    """The lookup is linear: its differences are exact in 64 bits, and the gradient of sum(c * lookup) is the backward of c."""
    from gsx_amd import fields
    rng = np.random.default_rng(3)
    table, c, ids = rng.standard_normal((7, 12)), rng.standard_normal((40, 12)), _ids(40, 7, 1)
    scale = 1.25  # a binary fraction: the same in 32 bits

    def f(t):
        return (_lookup_want(torch.from_numpy(t), ids, scale) * c).sum()

    got = fields.lookup_backward(torch.from_numpy(c).float().cuda(), torch.from_numpy(ids).cuda(), 7, scale=scale)
    got = got.double().cpu().numpy()
    for v, j in ((0, 0), (3, 5), (6, 11)):
        step = np.zeros_like(table)
        step[v, j] = 0.5
        # 40 terms of size 1: rounding c to float and summing is within 42 * 2^-24 of their magnitudes
        assert abs((f(table + step) - f(table - step)) - got[v, j]) <= 43 * 2.0**-24 * scale * np.abs(c).sum(0)[j]


def test_rows_refusals():
    from gsx_amd import fields
    from gsx_amd._lib import GsxHipError
    table, ids = torch.ones(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: fields.lookup(table.double(), ids), lambda: fields.lookup(table, ids.long()),
                lambda: fields.lookup(table.cpu(), ids), lambda: fields.lookup(table.T, ids),
                lambda: fields.lookup(table[0], ids), lambda: fields.lookup(table, ids, out=torch.ones(3, 7, device="cuda")),
                lambda: fields.lookup(table, ids, out_dtype=torch.int32),
                lambda: fields.lookup(table[:1].expand(4, 8), ids),
                lambda: fields.lookup_backward(table, ids, 5),  # four rows, three ids
                lambda: fields.lookup_backward(table[:3], ids, 5, accumulate=True),
                lambda: fields.lookup_backward(table[:3], ids, 5, grad_table=torch.ones(4, 8, device="cuda")),
                lambda: fields.lookup_backward(table[:3], ids, 5, grad_table=torch.ones(5, 8, device="cuda").half())):
        with pytest.raises(GsxHipError):
            bad()


def test_rows_refusals_of_the_c_interface():
    from gsx_amd import _lib
    lib = _lib.load()
    x = torch.zeros(64, device="cuda")
    p = x.data_ptr()
    for args in ((p, 9, 4, 4, p, 1, 4, 1.0, p, 0, 4, None, None), (p, 0, 4, 3, p, 1, 4, 1.0, p, 0, 4, None, None),
                 (p, 0, 4, 4, p, -1, 4, 1.0, p, 0, 4, None, None), (p, 0, 4, 4, None, 1, 4, 1.0, p, 0, 4, None, None),
                 (p + 2, 0, 4, 4, p, 1, 4, 1.0, p, 0, 4, None, None), (p, 0, 4, 4, p, 1, 4, 1.0, p, 1, 4, None, None)):
        assert lib.gsx_hip_lookup_forward(*args) < 0
        assert b"lookup" in lib.gsx_hip_last_error_message()
    assert lib.gsx_hip_lookup_backward(p, 0, 4, p, 2**32, 4, 1.0, p, 4, 4, 0, None, None) < 0


def test_lookup_on_another_stream():
    from gsx_amd import fields
    table = torch.randn(1000, 64, device="cuda")
    ids = torch.from_numpy(_ids(5000, 1000, 4)).cuda()
    want, grad_want = fields.lookup(table, ids), None
    grad_want = fields.lookup_backward(want, ids, 1000)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = fields.lookup(table, ids, stream=s)
    grad = fields.lookup_backward(got, ids, 1000, stream=s)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(grad, grad_want)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("count,rows,width", [(1, 3, 5), (200, 50, 7), (200, 20000, 259), (700, 300, 6), (2048, 1, 257),
                                              (3000, 40, 9), (9000, 3, 259), (9000, 3, 2)])
def test_gradient_of_odd_widths_is_added_to_a_table(count, rows, width, kind):
    """The last vector of a row of an odd width overlaps the one before: their common columns are added once. A sum of c terms in
    float32 is within (c + 3) 2^-24 of the sum of its terms' magnitudes, the table's value among them."""
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(count + width)
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[kind]
    grad = torch.randn(count, width + 1, device="cuda", generator=g).to(dtype)[:, 1:]
    ids = torch.randint(-1, rows, (count,), device="cuda", generator=g, dtype=torch.int32)
    base = torch.randn(rows, width + 3, device="cuda", generator=g)
    before = base.clone()
    print(f"[case] gradient of {count} ids added to {rows} x {width} {kind}", flush=True)
    fields.lookup_backward(grad, ids, rows, 0.5, grad_table=base[:, 2: width + 2], accumulate=True)
    i, x = ids.cpu().numpy(), grad.double().cpu().numpy()
    want, size = (np.zeros((rows, width)) for _ in range(2))
    for v in np.unique(i[i >= 0]):
        want[v], size[v] = 0.5 * x[i == v].sum(0), 0.5 * np.abs(x[i == v]).sum(0)
    old = before[:, 2: width + 2].double().cpu().numpy()
    got = base[:, 2: width + 2].double().cpu().numpy()
    assert (np.abs(got - (old + want)) <= (count + 3) * 2.0**-24 * (size + np.abs(old))).all()
    outside = [0, 1, width + 2]
    assert torch.equal(base[:, outside], before[:, outside])
    plain = fields.lookup_backward(grad, ids, rows, 0.5)
    assert (np.abs(plain.double().cpu().numpy() - want) <= (count + 3) * 2.0**-24 * size).all()
