"""Sums of block products are float32: whatever the result's type, however many rows a call has, however long the sum."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _cancelling(rows, k, seed):
    """Rows in which of every eight values two are +-256 and the others, in 1024 of the columns, 1 or 2; and the same with two
    of +256. The product of one of either kind is the sum of the small values' products alone: whole numbers, exact in float32
    in any order, which a bfloat16 or float16 holds too. The large products lie 2^16 above the small ones."""
    g = torch.Generator("cuda").manual_seed(seed)
    size = torch.randint(1, 3, (rows, 1), device="cuda", generator=g).float()
    x = torch.zeros(rows, k // 8, 8, device="cuda")
    x[:, :128] = size[..., None]
    y = x.clone()
    x[..., 0], x[..., 1] = 256, -256
    y[..., 0], y[..., 1] = 256, 256
    return x.view(rows, k), y.view(rows, k), size[:, 0]


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 1024), (100, 90, 1024), (300, 290, 4096), (2900, 2900, 1024), (3901, 3300, 1152)])
def test_small_products_beside_large_ones_that_cancel(m, n, k, out):
    from gsx_amd import fields
    x, _, small = _cancelling(m, k, m)
    _, w, weights = _cancelling(n, k, n)
    print(f"[case] cancelling sums {m} x {n} x {k} {out}", flush=True)
    got = fields.matmul(fields.quantize(x), fields.quantize(w), out_dtype=DTYPES[out])
    # 128 groups of six small products of at most 2 * 2
    assert torch.equal(got.float(), 768 * small[:, None] * weights[None])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,k", [(300, 1024), (50, 4096)])
def test_a_row_alone_and_in_a_batch_agree(n, k, kind):
    """The way that a linear layer takes depends on the number of rows; what it answers does not, as far as float32 sums are
    exact."""
    from gsx_amd import fields
    x, _, small = _cancelling(700, k, 1)
    _, w, weights = _cancelling(n, k, 2)
    x, w = x.to(DTYPES[kind]), fields.quantize(w)
    for rows in (1, 2, 16, 17, 700):
        got = fields.linear(x[:rows], w)
        assert got.dtype == DTYPES[kind]
        assert torch.equal(got.float(), 768 * small[:rows, None] * weights[None]), rows


def _steady(rows, length, along, dtype, first, second):
    """Rows of `length` values, zero but for the first two of every 128."""
    x = torch.zeros((rows, length) if along == 1 else (length, rows), dtype=dtype, device="cuda")
    t = x if along == 1 else x.T
    t[:, ::128], t[:, 1::128] = first, second
    return x


# A float32 sum of equal terms is off by half a step of its size each time: N terms by N / 2 times 2^-24 of it if they are
# rounded, N times 2^-24 if they are cut, and the error of equal terms points one way. The terms here are such that the
# sum's steps at the sizes of thousands of terms lose much of the smaller product each time. Sums that start anew after at most 512
# blocks, one term each, and the joining of the parts (16 at a time at the most, the groups' sums after it) stay within 512 + the
# parts joined.


@pytest.mark.parametrize("m", [1, 2])
def test_long_sums_of_few_rows_start_anew(m):
    from gsx_amd import fields
    k, n = 2**23, 3
    blocks = k // 128
    a, b = 1.875, 1.875 * 2.0**-6
    x, w = _steady(m, k, 1, torch.float32, a, b), fields.quantize(_steady(n, k, 1, torch.float32, a, b))
    print(f"[case] a sum of {blocks} equal terms, {m} rows", flush=True)
    got = fields.linear(x, w).double()
    want = blocks * (a * a + b * b)
    assert ((got - want).abs() <= (512 + blocks / 512 + 16) * 2.0**-24 * want).all(), (got / want - 1).abs().max().item()


def test_long_sums_of_narrow_weight_gradients_start_anew():
    from gsx_amd import fields
    m, n, k = 2**27, 4, 5
    blocks = m // 128
    a, b, c = 1.875, 1.875 * 2.0**-6, 1.875 * 2.0**-7
    x, dy = _steady(k, m, 0, torch.bfloat16, a, b), _steady(n, m, 0, torch.bfloat16, a, c)
    weight = fields.quantize(torch.ones(n, k, device="cuda"), transpose=True)
    print(f"[case] a weight gradient over {m} rows", flush=True)
    got = fields.linear_backward(x, dy, weight)[1].double()
    want = blocks * (a * a + b * c)
    assert ((got - want).abs() <= (512 + blocks / 512 / 16 + 16) * 2.0**-24 * want).all(), (got / want - 1).abs().max().item()
    assert not math.isnan(got.sum().item())
