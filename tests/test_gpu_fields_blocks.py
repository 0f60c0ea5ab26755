"""8-bit block matrices: the quantiser bit by bit against its definition in 64 bits, products and gradients against 64-bit
sums of what the blocks stand for."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}


def _grid():
    """The 128 E4M3 magnitudes by byte (the last is NaN)."""
    b = np.arange(128)
    field, low = b >> 3, b & 7
    v = np.where(field == 0, low * 2.0**-9, (1 + low / 8) * 2.0 ** (field - 7.0))
    v[127] = np.nan
    return v


def _want_blocks(x):
    """(bytes, exponents) of the rows of x (float64 array), from the definition."""
    rows, cols = x.shape
    nb = -(-cols // 128)
    grid = _grid()[:127]
    padded = np.zeros((rows, nb * 128))
    padded[:, :cols] = x
    blocks = padded.reshape(rows, nb, 128)
    finite = np.isfinite(blocks)
    top = np.where(finite, np.abs(blocks), 0).max(2)
    e = np.zeros(top.shape, int)
    e[top > 0] = -100
    for k in range(-100, 121):  # the least exponent that fits
        e = np.where((top > 0) & (top > 448 * 2.0 ** e) & (e == k), k + 1, e)
    y = np.abs(np.where(finite, blocks, 0)) * 2.0 ** -e[..., None].astype(float)
    hi = np.clip(np.searchsorted(grid, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    below, above = y - grid[lo], grid[hi] - y
    take_hi = (above < below) | ((above == below) & (hi % 2 == 0))
    q = np.where(take_hi, hi, lo)
    q = np.where(y == grid[hi], hi, q)
    q = np.where(finite, q, 127) + np.where(np.signbit(blocks), 128, 0)
    return q.reshape(rows, nb * 128).astype(np.uint8), (e + 127).astype(np.uint8)


def _values(q, e, cols):
    grid = _grid()
    v = grid[q & 127] * np.where(q > 127, -1.0, 1.0)
    return (v * np.repeat(2.0 ** (e[:, : q.shape[1] // 128].astype(float) - 127), 128, 1))[:, :cols]


def _special(rows, cols, seed):
    """Values of all sizes: blocks of zeros, denormals, the largest floats, exact ties, infinities and NaN."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-12, 12, (rows, 1))
    flat = x.reshape(-1)
    flat[::5] = rng.integers(-448, 449, flat[::5].size) * 0.5
    flat[::97] = 0.0
    if rows > 4:
        x[1] = 0.0
        x[2] = rng.standard_normal(cols) * 1e-41
        x[3] = np.clip(rng.standard_normal(cols) * 3e38, -3e38, 3e38)
        x[4, :: max(1, cols // 3)] = np.inf
        x[4, cols // 2] = -np.inf
    if rows > 5:
        x[5, cols - 1] = np.nan
        x[0, 0] = 448.0
        x[0, 1:] = rng.uniform(-448, 448, cols - 1)
    if rows > 6:
        x[6] = 2.0**-104 * rng.integers(-9, 9, cols)
    return x.astype(np.float32)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (7, 5, 3), (9, 127, 0), (9, 128, 0), (13, 129, 1), (70, 300, 0),
                                           (65, 1000, 8), (130, 257, 0), (8, 513, 4)])
def test_quantize_bits(rows, cols, pad, kind, transpose):
    from gsx_amd import fields
    base = torch.full((rows, cols + pad), float("nan"), device="cuda").to(DTYPES[kind])
    x = base[:, pad // 2: pad // 2 + cols]
    special = _special(cols, rows, cols).T if transpose else _special(rows, cols, cols)
    x.copy_(torch.from_numpy(np.ascontiguousarray(special)))
    print(f"[case] quantize {rows} x {cols} {kind} transpose={transpose}", flush=True)
    got = fields.quantize(x, transpose)
    src = x.double().cpu().numpy()
    q, e = _want_blocks(src.T if transpose else src)
    nb = e.shape[1]
    assert np.array_equal(got.exponents[:, :nb].cpu().numpy(), e)
    have = got.values.cpu().numpy()
    n = src.shape[0] if transpose else cols
    nan = (q & 127) == 127
    assert np.array_equal(nan, (have & 127) == 127)
    assert np.array_equal(have[~nan] & 127, q[~nan] & 127)
    assert np.array_equal((have & 128)[:, :n][~nan[:, :n]], (q & 128)[:, :n][~nan[:, :n]])
    assert (have[:, n:] == 0).all()


def _blocks(rows, cols, seed, spread=3, poison=False):
    """Random block matrix with value rows 16 bytes apart from their end at least; what lies past the columns is NaN bytes."""
    from gsx_amd import fields
    rng = np.random.default_rng(seed)
    nb = -(-cols // 128)
    ld = -(-cols // 16) * 16 + (32 if poison else 0)
    q = rng.integers(0, 127, (rows, ld)).astype(np.uint8) | (rng.integers(0, 2, (rows, ld)) << 7).astype(np.uint8)
    if poison:
        q[:, cols:] = 127
    e = np.full((rows, -(-nb // 4) * 4 + (4 if poison else 0)), 255, np.uint8)
    e[:, :nb] = rng.integers(127 - spread, 128 + spread, (rows, nb))
    vals = np.zeros((rows, nb * 128), np.uint8)
    vals[:, :cols] = q[:, :cols]
    return fields.Blocks(torch.from_numpy(q).cuda(), torch.from_numpy(e).cuda(), cols), _values(vals, e, cols)


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 17, 128), (3, 1, 129), (16, 16, 16), (17, 33, 100), (1, 300, 4096), (5, 257, 1000), (129, 130, 200),
    (64, 150, 128), (300, 40, 5000), (128, 128, 8192), (256, 256, 512), (257, 513, 385), (31, 2000, 640), (1000, 24, 31),
    (20, 20, 100_001), (700, 900, 1300), (64, 64, 384), (90, 3000, 127)])
def test_matmul(m, n, k, out):
    from gsx_amd import fields
    a, av = _blocks(m, k, m + k)
    b, bv = _blocks(n, k, n + k + 1, poison=True)
    scale = 2.0**-14 / k  # keeps f16 results finite
    a.exponents.copy_((a.exponents.int() + int(np.log2(scale))).clamp(0, 255).to(torch.uint8))
    av = av * 2.0 ** int(np.log2(scale))
    base = torch.full((m, n + 3), 5.0, dtype=DTYPES[out], device="cuda")
    print(f"[case] matmul {m} x {n} x {k} {out}", flush=True)
    got = fields.matmul(a, b, out=base[:, 1: n + 1])
    want, size = av @ bv.T, np.abs(av) @ np.abs(bv).T
    # k products summed in float: each of the k additions of a sum is within 2^-23 of the magnitudes so far (the matrix
    # instructions may cut instead of round), and a join over parts adds a few; then one rounding to the result's type
    bound = size * (k + 8) * 2.0**-23 + np.abs(want) * UNIT[out] + (2.0**-25 if out == "f16" else 0)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    # rounding errors of a long sum do not all point one way: the whole product is far closer than that
    rel = np.linalg.norm(got.double().cpu().numpy() - want) / np.linalg.norm(want)
    assert rel <= max(2e-6, 1.01 * UNIT[out]), rel
    assert (base[:, 0] == 5).all() and (base[:, n + 1:] == 5).all()


@pytest.mark.parametrize("m,n,k", [(256, 384, 1024), (40, 40, 256), (1, 64, 512), (2048, 16, 128)])
def test_matmul_of_whole_numbers_is_exact(m, n, k):
    """Small whole numbers in distinct places: any misplaced row, column, block or scale shows."""
    from gsx_amd import fields
    rng = np.random.default_rng(m)
    x, w = rng.integers(-8, 9, (m, k)).astype(np.float32), rng.integers(-8, 9, (n, k)).astype(np.float32)
    x *= 2.0 ** rng.integers(0, 3, (m, k // 128)).repeat(128, 1)
    a, b = fields.quantize(torch.from_numpy(x).cuda()), fields.quantize(torch.from_numpy(w).cuda())
    print(f"[case] whole numbers {m} x {n} x {k}", flush=True)
    assert np.array_equal(fields.matmul(a, b).cpu().numpy(), x.astype(np.float64) @ w.T.astype(np.float64))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 5, 3), (1, 2000, 4096), (7, 150, 128), (16, 64, 1000), (17, 70, 129), (500, 33, 260),
                                   (3, 100, 20000), (2, 513, 100)])
def test_linear_is_quantize_then_matmul(m, n, k, kind):
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(m + n)
    base = torch.randn(m, k + 5, device="cuda", generator=g).to(DTYPES[kind])
    x = base[:, 2: k + 2]
    w, wv = _blocks(n, k, n, poison=True)
    print(f"[case] linear {m} x {n} x {k} {kind}", flush=True)
    got = fields.linear(x, w, out_dtype=torch.float32).double().cpu().numpy()
    src = x.double().cpu().numpy()
    xv = _values(*_want_blocks(src), k)
    bound = np.abs(xv) @ np.abs(wv).T * (k + 8) * 2.0**-23 + 2.0**-24 * np.abs(xv @ wv.T)
    assert (np.abs(got - xv @ wv.T) <= bound).all()
    assert np.linalg.norm(got - xv @ wv.T) <= 2e-6 * np.linalg.norm(xv @ wv.T)


@pytest.mark.parametrize("n", [3, 300])
def test_products_of_the_smallest_and_largest_blocks(n):
    """Scales from 2^-100 to 2^118 (448 * 2^118 is near the largest float) on one side, the other side brings the product back:
    every bit is kept."""
    from gsx_amd import fields
    k = 256
    w, _ = _blocks(n, k, 5, spread=1)
    w.exponents[:, 0], w.exponents[:, 1] = 127, 127
    q = w.values[:1].repeat(6, 1)
    x = fields.Blocks(q, torch.full((6, 4), 127, dtype=torch.uint8, device="cuda"), k)
    base = fields.matmul(x, w)
    for row, e in enumerate((-100, -99, -60, 60, 100, 118)):
        x.exponents[row] = 127 + e
        y = fields.Blocks(w.values, torch.full_like(w.exponents, 127 - min(100, e)), k)
        got = fields.matmul(x, y)[row]
        assert torch.equal(got * 2.0 ** (min(100, e) - e), base[row]), e


@pytest.mark.parametrize("m", [1, 40])
def test_non_finite_rows_stay_in_their_row(m):
    from gsx_amd import fields
    x = torch.randn(m + 2, 300, device="cuda")
    x[0, 7], x[1, 299] = float("inf"), float("nan")
    w = fields.quantize(torch.randn(50, 300, device="cuda"))
    for rows in (x, x[:1], x[1:2]):
        y = fields.linear(rows, w)
        bad = ~torch.isfinite(rows).all(1)
        assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (200, 150, 128), (1000, 33, 65), (5000, 20, 16), (130, 258, 300)])
def test_linear_backward(m, n, k, kind):
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(m)
    x = torch.randn(m, k, device="cuda", generator=g).to(DTYPES[kind])
    dy = (torch.randn(m, n, device="cuda", generator=g) * 1e-3).to(DTYPES[kind])
    w = torch.randn(n, k, device="cuda", generator=g)
    wt = fields.quantize(w, transpose=True)
    print(f"[case] linear backward {m} x {n} x {k} {kind}", flush=True)
    dx, dw = fields.linear_backward(x, dy, wt)
    assert dx.dtype == DTYPES[kind] and dw.dtype == torch.float32
    xs, ds = x.double().cpu().numpy(), dy.double().cpu().numpy()
    wv = _values(*_want_blocks(w.double().cpu().numpy().T), n)
    dv, dtv, xtv = (_values(*_want_blocks(s), s.shape[1]) for s in (ds, ds.T, xs.T))
    for got, p, q, unit, terms in ((dx, dv, wv.T, UNIT[kind], n), (dw, dtv, xtv.T, UNIT["f32"], m)):
        want, size = p @ q, np.abs(p) @ np.abs(q)
        bound = size * (terms + 8) * 2.0**-23 + np.abs(want) * unit
        assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(8192, 1, 1), (8193, 130, 127), (9000, 150, 128), (20001, 33, 257), (8200, 256, 120),
                                   (12345, 61, 200), (40000, 200, 60), (8191, 150, 128)])
def test_weight_gradient_of_narrow_layers(m, n, k, kind):
    """Many rows and few columns, with odd strides: sums of m terms in parts."""
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(m)
    x = torch.randn(m, k + 3, device="cuda", generator=g).to(DTYPES[kind])[:, 1: k + 1]
    dy = torch.randn(m, n + 1, device="cuda", generator=g).to(DTYPES[kind])[:, 1:]
    x[m // 2], dy[3, 0] = 0, 300.0
    wt = fields.quantize(torch.randn(n, k, device="cuda", generator=g), transpose=True)
    print(f"[case] weight gradient {m} x {n} x {k} {kind}", flush=True)
    base = torch.full((n, k + 2), 7.0, device="cuda")
    _, dw = fields.linear_backward(x, dy, wt, grad_weight=base[:, 1: k + 1])
    p, q = (_values(*_want_blocks(s.double().cpu().numpy().T), m) for s in (dy, x))
    want, size = p @ q.T, np.abs(p) @ np.abs(q).T
    # a part's sum of at most m terms and a join: see test_matmul
    assert (np.abs(dw.double().cpu().numpy() - want) <= size * (m + 8) * 2.0**-23 + np.abs(want) * 2.0**-24).all()
    assert np.linalg.norm(dw.double().cpu().numpy() - want) <= 2e-6 * np.linalg.norm(want) + 2.0**-23 * np.linalg.norm(size) / 16
    assert (base[:, 0] == 7).all() and (base[:, -1] == 7).all()
    again = fields.linear_backward(x, dy, wt)[1]
    assert torch.equal(again, dw)


def test_weight_gradient_of_narrow_layers_with_two_types():
    """Rows and gradients of different types take the way of wide layers, whose workspace is larger."""
    from gsx_amd import _lib, fields
    m, n, k = 8200, 40, 24
    lib = _lib.load()
    codes = {"f32": fields._type(torch.float32), "bf16": fields._type(torch.bfloat16)}
    mixed = lib.gsx_hip_linear_backward_weight_temp_bytes(codes["bf16"], codes["f32"], m, n, k)
    assert mixed >= (n + k) * (m + m // 128)
    x = torch.randn(m, k, device="cuda").bfloat16()
    dy = torch.randn(m, n, device="cuda")
    wt = fields.quantize(torch.randn(n, k, device="cuda"), transpose=True)
    print(f"[case] weight gradient {m} x {n} x {k} of two types", flush=True)
    _, dw = fields.linear_backward(x, dy, wt)
    p, q = (_values(*_want_blocks(s.double().cpu().numpy().T), m) for s in (dy, x))
    want, size = p @ q.T, np.abs(p) @ np.abs(q).T
    assert (np.abs(dw.double().cpu().numpy() - want) <= size * (m + 8) * 2.0**-23 + np.abs(want) * 2.0**-24).all()


@pytest.mark.parametrize("m,n,k", [(33000, 40, 768), (33000, 64, 700), (33000, 40, 769), (33000, 200, 128), (33000, 200, 256),
                                   (500, 200, 256), (500, 200, 300), (500, 60, 500)])
def test_linear_about_the_ways_sizes(m, n, k):
    """linear() is quantize() and matmul() on either side of the sizes at which the way changes: both are sums of the same k products in
    float32, each within k 2^-24 of the sum of their magnitudes, rounded once more."""
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(m + n + k)
    x = torch.randn(m, k, device="cuda", generator=g)
    w = fields.quantize(torch.randn(n, k, device="cuda", generator=g))
    print(f"[case] linear {m} x {n} x {k}", flush=True)
    got, q = fields.linear(x, w), fields.quantize(x)
    size = q.float().abs() @ w.float().abs().T
    assert ((got - fields.matmul(q, w)).abs() <= size * (2 * k + 8) * 2.0**-24).all()
    rows = torch.tensor([0, m // 2, m - 1], device="cuda")
    want = q.float()[rows].double() @ w.float().double().T
    assert ((got[rows] - want).abs() <= size[rows] * (k + 8) * 2.0**-24).all()


def test_weight_gradient_keeps_non_finite_columns_apart():
    from gsx_amd import fields
    x, dy = torch.randn(9000, 20, device="cuda"), torch.randn(9000, 30, device="cuda")
    x[17, 3], dy[8999, 7] = float("inf"), float("nan")
    _, dw = fields.linear_backward(x, dy, fields.quantize(torch.randn(30, 20, device="cuda"), transpose=True))
    bad = torch.zeros(30, 20, dtype=torch.bool, device="cuda")
    bad[:, 3], bad[7] = True, True
    assert torch.equal(torch.isnan(dw), bad)


def test_linear_gradient_against_differences():
    """With operands that 8 bits hold exactly the product is bilinear, so central differences of it are exact."""
    from gsx_amd import fields
    rng = np.random.default_rng(8)
    m, n, k = 6, 5, 140
    x, w, c = (rng.integers(-3, 4, s).astype(np.float64) for s in ((m, k), (n, k), (m, n)))

    def to(a):
        return torch.from_numpy(a.astype(np.float32)).cuda()

    def f(x, w):
        return (fields.linear(to(x), fields.quantize(to(w))).double().cpu().numpy() * c).sum()

    dx, dw = fields.linear_backward(to(x), to(c), fields.quantize(to(w), transpose=True))
    for i, j in ((0, 0), (5, 139), (2, 128)):
        step = np.zeros_like(x)
        step[i, j] = 1
        assert (f(x + step, w) - f(x - step, w)) / 2 == dx[i, j].item()
    for i, j in ((0, 0), (4, 139), (3, 127)):
        step = np.zeros_like(w)
        step[i, j] = 1
        assert (f(x, w + step) - f(x, w - step)) / 2 == dw[i, j].item()


def test_matmul_past_32_bit_offsets():
    from gsx_amd import fields
    m, n, k = 2**21 + 40, 24, 1040  # 2^31 bytes of values and some
    values = torch.zeros((m, k), dtype=torch.uint8, device="cuda")
    exponents = torch.full((m, 12), 127, dtype=torch.uint8, device="cuda")
    values[-1] = 0x38  # 1.0
    values[2**21] = 0x40  # 2.0
    w = fields.quantize(torch.ones(n, k, device="cuda"))
    print("[case] matmul past 2^31 bytes", flush=True)
    got = fields.matmul(fields.Blocks(values, exponents, k), w)
    assert (got[-1] == k).all() and (got[2**21] == 2 * k).all() and got.sum().item() == 3 * k * n
    got = fields.matmul(w, fields.Blocks(values, exponents, k))
    assert (got[:, -1] == k).all() and (got[:, 2**21] == 2 * k).all() and got.sum().item() == 3 * k * n


def test_empty_products():
    from gsx_amd import fields
    x = torch.ones(3, 0, device="cuda")
    w = fields.quantize(torch.ones(4, 0, device="cuda"))
    assert torch.equal(fields.linear(x, w), torch.zeros(3, 4, device="cuda"))
    w = fields.quantize(torch.ones(4, 9, device="cuda"))
    assert fields.linear(torch.ones(0, 9, device="cuda"), w).shape == (0, 4)


def test_products_repeat_bit_for_bit_and_on_another_stream():
    from gsx_amd import fields
    x, w = torch.randn(150, 30000, device="cuda"), fields.quantize(torch.randn(90, 30000, device="cuda"))
    want = fields.linear(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = [fields.linear(x, w, stream=s) for _ in range(5)]
    s.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_linear_in_a_graph():
    from gsx_amd import fields
    x, w = torch.randn(4, 3000, device="cuda"), fields.quantize(torch.randn(70, 3000, device="cuda"))
    out = torch.zeros(4, 70, device="cuda")
    fields.linear(x, w, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fields.linear(x, w, out=out)
    for k in range(4):
        x.copy_(torch.randn(4, 3000, device="cuda", generator=torch.Generator("cuda").manual_seed(k)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fields.linear(x, w)), k


def test_blocks_refusals():
    from gsx_amd import fields
    from gsx_amd._lib import GsxHipError
    x = torch.ones(4, 256, device="cuda")
    w = fields.quantize(x)
    u8 = torch.uint8
    for bad in (lambda: fields.quantize(x.double()), lambda: fields.quantize(x.cpu()), lambda: fields.quantize(x[0]),
                lambda: fields.quantize(x.T), lambda: fields.linear(x[:, :200], w), lambda: fields.linear(x.int(), w),
                lambda: fields.matmul(w, fields.quantize(x[:, :129])),
                lambda: fields.linear(x, w, out=torch.ones(4, 5, device="cuda")),
                lambda: fields.linear(x, w, out_dtype=torch.float64),
                lambda: fields.matmul(fields.Blocks(w.values[:, :255], w.exponents, 256), w),
                lambda: fields.matmul(fields.Blocks(w.values, w.exponents[:3], 256), w),
                lambda: fields.matmul(fields.Blocks(w.values, w.exponents[:, :1], 256), w),
                lambda: fields.matmul(fields.Blocks(torch.zeros(4, 265, dtype=u8, device="cuda")[:, 9:], w.exponents, 256), w),
                lambda: fields.matmul(fields.Blocks(torch.zeros(4, 260, dtype=u8, device="cuda"), w.exponents, 256), w),
                lambda: fields.matmul(fields.Blocks(w.values.float(), w.exponents, 256), w),
                lambda: fields.linear_backward(x, x[:3], w), lambda: fields.linear_backward(x, x, w)):
        with pytest.raises(GsxHipError):
            bad()


def test_blocks_refusals_of_the_c_interface():
    from gsx_amd import _lib
    lib = _lib.load()
    x = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    p = x.data_ptr()
    assert lib.gsx_hip_blocks_quantize(p, 1, 1, 16, 16, 0, p, 16, p, 4, None) == _lib.ERROR_NOT_SUPPORTED
    for args in ((p, 0, 1, 16, 15, 0, p, 16, p, 4), (p, 0, -1, 16, 16, 0, p, 16, p, 4), (p, 0, 1, 16, 16, 0, p, 24, p, 4),
                 (p, 0, 1, 16, 16, 0, p + 8, 16, p, 4), (p, 0, 1, 16, 16, 0, p, 16, p, 2), (p, 0, 1, 16, 16, 0, p, 16, p + 2, 4),
                 (p, 0, 1, 16, 16, 0, None, 16, p, 4), (None, 0, 1, 16, 16, 0, p, 16, p, 4), (p, 0, 1, 32, 32, 0, p, 16, p, 4)):
        assert lib.gsx_hip_blocks_quantize(*args, None) == _lib.ERROR_INVALID_ARGUMENT
    good = (p, 16, p, 4, p, 16, p, 4)
    for m, n, k, stride in ((-1, 1, 16, 1), (2**31, 1, 16, 1), (1, 1, 2**31, 1), (1, 2, 16, 1)):
        assert lib.gsx_hip_blocks_matmul(*good, m, n, k, p, 0, stride, None, None) < 0
    # a call that needs a workspace (some sizes need none), refused before anything runs
    y = torch.zeros(1024 * 1024, device="cuda").data_ptr()
    assert lib.gsx_hip_linear_temp_bytes(300, 300, 1024) > 0
    assert lib.gsx_hip_linear_forward(y, 0, 1024, y, 1024, y, 8, 300, 300, 1024, y, 0, 300, None,
                                      None) == _lib.ERROR_INVALID_ARGUMENT
    assert lib.gsx_hip_linear_forward(p, 0, 15, p, 16, p, 4, 1, 1, 16, p, 0, 1, None, None) == _lib.ERROR_INVALID_ARGUMENT
    assert lib.gsx_hip_linear_temp_bytes(-1, 4, 4) == 0
