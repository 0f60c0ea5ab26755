"""4-bit block matrices: the quantiser bit by bit against its definition, products and linear layers against 64-bit sums of what
the blocks stand for."""
import numpy as np
import pytest

import blocks4_plain as plain
from blocks4_ways import LINEARS as WAYS
from blocks4_ways import PRODUCTS

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 0.0, "bf16": 2.0**-8, "f16": 2.0**-11}
U = 2.0**-24


def _special(rows, cols, seed):
    """Values of all sizes: blocks of zeros, denormals, the largest floats, exact ties, infinities and NaN."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-12, 12, (rows, 1))
    flat = x.reshape(-1)
    flat[::5] = rng.integers(-24, 25, flat[::5].size) * 0.25
    flat[::97] = 0.0
    flat[1::97] = -0.0
    if rows > 7:
        x[1] = 0
        x[2] = 1e-42
        x[3, ::3] = 3.3e38
        x[4, cols // 2] = np.nan
        x[5, 0], x[5, cols - 1] = np.inf, -np.inf
        x[6] = rng.integers(-6, 7, cols) * 2.0**-100
        x[7] = 6.0 + rng.integers(0, 2, cols) * 2.0**-20
    return x.astype(np.float32)


def _put(x, kind, pad=0, lead=0):
    rows, cols = x.shape
    room = torch.full((rows, cols + pad), float("nan"), dtype=DTYPES[kind], device="cuda")
    t = room[:, lead: lead + cols]
    t.copy_(torch.from_numpy(x))
    return t


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("rows,cols,pad,lead", [(9, 32, 0, 0), (9, 1, 3, 1), (9, 31, 1, 1), (9, 33, 0, 0), (10, 129, 7, 3),
                                                (33, 1000, 0, 0), (8, 4101, 5, 5), (1, 7, 0, 0), (300, 64, 0, 0), (1, 70_001, 0, 0)])
def test_quantised_bit_by_bit(rows, cols, pad, lead, kind):
    from gsx_amd import fields
    with np.errstate(over="ignore"):
        x = _put(_special(rows, cols, cols), kind, pad, lead)
    got = fields.quantize4(x)
    q, e = plain.blocks(x.double().cpu().numpy())
    assert np.array_equal(got.exponents.cpu().numpy()[:, : e.shape[1]], e)
    assert np.array_equal(got.values.cpu().numpy(), plain.packed(q))
    with np.errstate(over="ignore"):
        want = plain.values(q, e, cols).astype(np.float32)  # 3.3e38 is held as 2^128
    assert np.array_equal(got.float().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("kind", DTYPES)
def test_every_code_and_exponent_expands(kind):
    from gsx_amd import fields
    values = torch.arange(256, dtype=torch.uint8, device="cuda").view(16, 16).repeat(16, 1)  # 256 rows of a block
    exponents = torch.zeros(256, 4, dtype=torch.uint8, device="cuda")
    exponents[:, 0] = torch.arange(256, device="cuda")
    for cols in (32, 29):
        got = fields.Blocks4(values, exponents, cols).float(DTYPES[kind])
        want = plain.values(plain.codes(values.cpu().numpy()), exponents[:, :1].cpu().numpy(), cols)
        want = torch.from_numpy(want).cuda()
        # exact but for float16's range and steps, and for what lies above float32's or below its least numbers
        assert torch.equal(got.double().nan_to_num(nan=7e77), want.float().to(DTYPES[kind]).double().nan_to_num(nan=7e77))


def _rows(rows, cols, seed):
    """Rows whose columns and themselves differ in size."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g, dtype=torch.float64)
    x *= torch.exp(torch.randn(cols, device="cuda", generator=g))
    return (x * 2.0 ** torch.randint(-3, 4, (rows, 1), device="cuda", generator=g)).float()


def _blocks(x):
    """x in blocks (whose making has tests of its own), and what they stand for; behind the last value there are other codes and NaN
    scales."""
    from gsx_amd import fields
    rows, cols = x.shape
    made = fields.quantize4(x)
    bytes_, blocks = -(-cols // 2), -(-cols // 32)
    values = torch.randint(0, 256, (rows, made.values.shape[1] + 32), dtype=torch.uint8, device="cuda")
    exponents = torch.full((rows, made.exponents.shape[1] + 4), 255, dtype=torch.uint8, device="cuda")
    values[:, :bytes_] = made.values[:, :bytes_]
    if cols % 2:
        values[:, bytes_ - 1] = made.values[:, bytes_ - 1] & 15 | 0xA0
    exponents[:, :blocks] = made.exponents[:, :blocks]
    return fields.Blocks4(values, exponents, cols), made.float().double()


def _room(a, b, k, kind, want):
    """How far a product may be: an instruction takes 128 k and rounds each of its four blocks' sums and what it adds them to, eight
    roundings at the most, each half a step of a number no larger than the terms' magnitudes together; then the result's type."""
    off = 8 * (-(-k // 128) + 1) * U * (a.abs() @ b.abs().T)
    least = 2.0**-25 if kind == "f16" else 0.0
    return off + UNIT[kind] * (want.abs() + off) + least


def _check_product(call, va, vb, k):
    m, n = va.shape[0], vb.shape[0]
    want = va @ vb.T
    for kind in DTYPES:
        room = torch.full((m, n + 3), 7.0, dtype=DTYPES[kind], device="cuda")
        call(room[:, :n])
        assert (room[:, n:] == 7).all()
        got = room[:, :n].double()
        # what lies beyond the type's range (float16: from 65520 on) is infinite there
        beyond = want.to(DTYPES[kind]).isinf() & (got == want.to(DTYPES[kind]).double())
        assert ((got - want).abs() <= _room(va, vb, k, kind, want)).logical_or(beyond).all(), kind


@pytest.mark.parametrize("m,n,k", [p[:3] for p in PRODUCTS])
def test_products_against_64_bits(m, n, k):
    from gsx_amd import fields
    print(f"[case] 4-bit product {m} x {n} x {k}", flush=True)
    (a, va), (b, vb) = _blocks(_rows(m, k, m + k)), _blocks(_rows(n, k, n + k) * 0.1)
    _check_product(lambda out: fields.matmul(a, b, out=out), va, vb, k)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 2), (3, 1, 33), (17, 16, 32), (16, 64, 64), (65, 65, 256), (64, 64, 257),
                                   (5, 7, 0), (2, 3, 70_001), (130, 70, 9000)])
def test_products_of_small_and_long_shapes(m, n, k):
    from gsx_amd import fields
    (a, va), (b, vb) = _blocks(_rows(m, k, k)), _blocks(_rows(n, k, k + 1))
    _check_product(lambda out: fields.matmul(a, b, out=out), va, vb, k)


@pytest.mark.parametrize("m,n", [(3, 5), (70, 80), (300, 280), (2100, 2050), (3900, 3901)])
def test_products_of_any_exponents(m, n):
    """Exponent bytes from 1 on to 254, whose products leave float32's range at either end; a NaN block spoils its row alone."""
    from gsx_amd import fields
    rng = np.random.default_rng(m)
    k = 300
    nb = 10
    made = []
    for rows in (m, n):
        q = rng.integers(0, 16, (rows, nb * 32)).astype(np.uint8)
        e = (127 + rng.integers(-6, 7, (rows, nb))).astype(np.uint8)
        e[0], e[1] = 30, 230
        e[2, 4] = 255
        made.append((q, e, np.concatenate([e, np.full((rows, 2), 255, np.uint8)], 1)))
    a, b = (fields.Blocks4(torch.from_numpy(plain.packed(q)).cuda(), torch.from_numpy(e).cuda(), k) for q, _, e in made)
    va, vb = (plain.values(q, e, k) for q, e, _ in made)
    got = fields.matmul(a, b).double().cpu().numpy()
    assert np.isnan(got[2]).all() and np.isnan(got[:, 2]).all()
    keep_a, keep_b = np.arange(m) != 2, np.arange(n) != 2
    va, vb, got = va[keep_a], vb[keep_b], got[keep_a][:, keep_b]
    with np.errstate(over="ignore"):
        want = va @ vb.T
    room = _room(*(torch.from_numpy(v) for v in (va, vb)), k, "f32", torch.from_numpy(want)).numpy() + 2.0**-126 * 128
    fits = (np.abs(va) @ np.abs(vb).T) < 3e38
    assert (np.abs(got - want) <= room)[fits].all()
    assert not fits.all()  # 2^103 times 2^103


def _cancelling(rows, k, seed, up):
    """Rows in which of every eight blocks two are +-2^up and six are 1 or 2, and the same with two of +2^up: a product of the one
    with the other is the small blocks' alone, whole numbers far below 2^24."""
    g = torch.Generator("cuda").manual_seed(seed)
    size = torch.randint(1, 3, (rows, 1), device="cuda", generator=g).float()
    x = torch.zeros(rows, k // 256, 8, 32, device="cuda")
    x[:] = size[..., None, None]
    y = x.clone()
    x[:, :, 0], x[:, :, 1] = 2.0**up, -(2.0**up)
    y[:, :, 0], y[:, :, 1] = 2.0**up, 2.0**up
    return x.view(rows, k), y.view(rows, k), size[:, 0]


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m,n,k", [(3, 40, 1024), (16, 40, 1024), (100, 90, 1024), (2900, 2900, 1024), (3901, 3300, 1280),
                                   (5000, 150, 256), (5000, 30, 1024)])
def test_small_blocks_beside_large_ones_that_cancel(m, n, k, out):
    from gsx_amd import fields
    up = 7  # 32 products of 2^14 and their sum with small whole numbers stay below 2^24
    x, _, small = _cancelling(m, k, m, up)
    _, w, weights = _cancelling(n, k, n, up)
    weight = fields.quantize4(w)
    want = (k // 256 * 6 * 32) * small[:, None] * weights[None]
    want = want.to(DTYPES[out])
    assert torch.equal(fields.matmul(fields.quantize4(x), weight, out_dtype=DTYPES[out]), want)
    assert torch.equal(fields.linear(x, weight, out_dtype=DTYPES[out]), want)


LINEARS = [(1, 1, 1), (1, 333, 130), (2, 50, 16_500), (7, 129, 257), (17, 40, 96), (500, 64, 257),
           (500, 128, 384), (500, 129, 128), (3001, 150, 257), (500, 193, 256), (300, 300, 300), (600, 257, 40),
           (5, 3, 0), (3000, 16, 1500), (999, 7, 33), (2000, 256, 777), (1, 50, 66_000)]
LINEARS += [way[:3] for way in WAYS if way[:3] not in LINEARS]


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("m,n,k", LINEARS)
def test_linear_layers_against_64_bits(m, n, k, kind):
    from gsx_amd import fields
    print(f"[case] 4-bit linear {m} x {n} x {k} {kind}", flush=True)
    room = torch.full((m, k + 5), float("nan"), dtype=DTYPES[kind], device="cuda")
    x = room[:, 1: k + 1]
    x.copy_(_rows(m, k, m + n + k))
    w, vw = _blocks(_rows(n, k, n) * 0.1)
    _check_product(lambda out: fields.linear(x, w, out=out), fields.quantize4(x).float().double(), vw, k)
    if m * n * k > 0:  # rows of the result without a gap
        whole = torch.empty(m, n, dtype=DTYPES[kind], device="cuda")
        fields.linear(x, w, out=whole)
        room = torch.empty(m, n + 1, dtype=DTYPES[kind], device="cuda")
        fields.linear(x, w, out=room[:, 1:])
        assert torch.equal(whole, room[:, 1:])


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("m,n,k", [(2, 40, 200), (16, 300, 130), (200, 150, 257), (300, 300, 500)])
def test_rows_that_are_not_finite_are_nan_alone(m, n, k, kind):
    from gsx_amd import fields
    x = _rows(m, k, 3).to(DTYPES[kind])
    w, _ = _blocks(_rows(n, k, 4))
    clean = fields.linear(x, w)
    x[0, k - 1], x[1, 0] = float("nan"), float("-inf")
    got = fields.linear(x, w)
    assert got[:2].isnan().all() and torch.equal(got[2:], clean[2:])


@pytest.mark.parametrize("n,k", [(300, 1024), (50, 4096)])
def test_a_row_alone_and_in_a_batch_agree(n, k):
    from gsx_amd import fields
    x, _, small = _cancelling(700, k, 1, 6)
    _, w, weights = _cancelling(n, k, 2, 6)
    w = fields.quantize4(w)
    for rows in (1, 2, 16, 17, 64, 700):
        assert torch.equal(fields.linear(x[:rows], w), (k // 256 * 192) * small[:rows, None] * weights[None]), rows


@pytest.mark.parametrize("m", [1, 2, 100])
def test_long_sums_start_anew(m):
    """Equal terms, one of two kinds a block, whose error points one way: a float32 sum of N of them is off by N / 2 steps of 2^-24
    of its size. Sums start anew after at most 65536 k, one such sum an instruction's 128, and their joining adds no more than the
    parts joined."""
    from gsx_amd import fields
    k, n = 2**22, 3
    x = torch.zeros(m, k, device="cuda")
    x[:, ::32], x[:, 1::32] = 6.0, 0.5
    w = fields.quantize4(torch.cat([x[:1] * (2.0**-5 if i else 1.0) for i in range(n)]))
    got = fields.linear(x, w).double()
    blocks = k // 32
    want = torch.tensor([blocks * 36.25 * (2.0**-5 if i else 1.0) for i in range(n)], dtype=torch.float64, device="cuda")
    assert ((got - want).abs() <= (4 * 512 + k / 65536 + 16) * U * want).all(), (got / want - 1).abs().max().item()


def test_results_behind_2_31_elements():
    from gsx_amd import fields
    m, n, k = 66_000, 33_000, 64
    print(f"[case] 4-bit product {m} x {n} x {k}", flush=True)
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(m, k, device="cuda", generator=g, dtype=torch.bfloat16)
    w = fields.quantize4(torch.randn(n, k, device="cuda", generator=g))
    got = fields.linear(x, w)
    want = fields.linear(x[-300:].clone(), w)
    assert torch.equal(got[-300:], want)
    wide = fields.quantize4(torch.randn(40, 2**27 // 2, device="cuda", generator=g, dtype=torch.bfloat16))
    assert wide.float(torch.bfloat16).shape == (40, 2**26)
    assert torch.equal(wide.float(torch.bfloat16)[-1], fields.Blocks4(wide.values[-1:], wide.exponents[-1:], 2**26).float(torch.bfloat16)[0])


@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (400, 150, 128), (300, 300, 3000)])
def test_replays_of_a_captured_layer(m, n, k):
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(2)
    x, weight = torch.randn(m, k, device="cuda", generator=g), torch.randn(n, k, device="cuda", generator=g)
    fields.linear(x, fields.quantize4(weight))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = fields.quantize4(weight)
        y = fields.linear(x, w)
        v = w.float()
    for _ in range(4):
        x.normal_(generator=g)
        weight.normal_(generator=g)
        graph.replay()
        want = fields.quantize4(weight)
        assert torch.equal(y, fields.linear(x, want)) and torch.equal(v, want.float())


def test_calls_on_two_streams_at_once():
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(3)
    xs = [torch.randn(300, 4000, device="cuda", generator=g) for _ in range(2)]
    w = fields.quantize4(torch.randn(300, 4000, device="cuda", generator=g))
    want = [fields.linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[fields.linear(x, w, stream=s) for _ in range(10)] for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    for calls, y in zip(got, want):
        assert all(torch.equal(z, y) for z in calls)


def test_refusals():
    from gsx_amd import fields
    from gsx_amd.backend import GsxHipError
    x = torch.zeros(4, 64, device="cuda")
    w, w8 = fields.quantize4(x), fields.quantize(x)
    for call in (lambda: fields.quantize4(x.double()), lambda: fields.quantize4(x.T), lambda: fields.quantize4(x.cpu()),
                 lambda: fields.matmul(w, w8), lambda: fields.matmul(w8, w), lambda: fields.linear(x[:, :63], w),
                 lambda: fields.matmul(w, fields.quantize4(x[:, :32])), lambda: fields.matmul(w, w, out_dtype=torch.float64),
                 lambda: fields.linear(x, fields.Blocks4(w.values[:, :16], w.exponents, 64)),
                 lambda: fields.linear(x, fields.Blocks4(w.values, w.exponents[:2], 64)),
                 lambda: fields.linear(x, fields.Blocks4(w.values.int(), w.exponents, 64)),
                 lambda: w.float(out=torch.zeros(4, 63, device="cuda")),
                 lambda: fields.linear_backward(x, torch.zeros(4, 4, device="cuda"), fields.quantize4(torch.zeros(64, 4, device="cuda")))):
        with pytest.raises(GsxHipError):
            call()
