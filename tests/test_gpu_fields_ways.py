"""Every kernel that the label fields choose by size, at sizes that take it (tests/fields_ways.py, checked against the library by
test_fields_ways_cpu.py). Operands are whole numbers, so that a sum is exact in float32 in any order: a result is the exact sum
rounded once, bit by bit."""
import os
import subprocess
import sys

import pytest

from fields_ways import DISTILLS, LINEARS, PRODUCTS

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _whole(rows, cols, seed, dtype=torch.float32, pad=0):
    """Whole numbers from -8 to 8, which every type and the blocks hold exactly (their products' sums stay below 2^24)."""
    g = torch.Generator("cuda").manual_seed(seed)
    base = torch.randint(-8, 9, (rows, cols + pad), device="cuda", generator=g, dtype=torch.int32).to(dtype)
    return base[:, pad // 2: pad // 2 + cols]


def _once(exact, dtype):
    """float64 sums that a float32 holds, rounded once."""
    assert torch.equal(exact.float().double(), exact)
    return exact.float().to(dtype)


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [s[:3] for s in PRODUCTS])
def test_products_of_whole_numbers(m, n, k, out):
    """The rows' blocks have scales that differ, so that a scale of another block or row shows."""
    from gsx_amd import fields
    x, w = _whole(m, k, m), _whole(n, k, n)
    for t, seed in ((x, 5), (w, 6)):
        scale = torch.exp2(_whole(t.shape[0], -(-k // 128), seed).remainder(3))
        t *= scale.repeat_interleave(128, 1)[:, :k]
    print(f"[case] product {m} x {n} x {k} {out}", flush=True)
    base = torch.full((m, n + 3), 7.0, dtype=DTYPES[out], device="cuda")
    got = fields.matmul(fields.quantize(x), fields.quantize(w), out=base[:, 1: n + 1])
    assert torch.equal(got, _once(x.double() @ w.double().T, DTYPES[out]))
    assert (base[:, 0] == 7).all() and (base[:, n + 1:] == 7).all()


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [s[:3] for s in LINEARS])
def test_linears_of_whole_numbers(m, n, k, kind, out):
    from gsx_amd import fields
    x, w = _whole(m, k, m + n, DTYPES[kind], pad=3), _whole(n, k, k)
    print(f"[case] linear {m} x {n} x {k} {kind} to {out}", flush=True)
    base = torch.full((m, n + 3), 7.0, dtype=DTYPES[out], device="cuda")
    got = fields.linear(x, fields.quantize(w), out=base[:, 1: n + 1])
    assert torch.equal(got, _once(x.double() @ w.double().T, DTYPES[out]))
    assert (base[:, 0] == 7).all() and (base[:, n + 1:] == 7).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(8200, 150, 128), (9001, 129, 61), (8193, 40, 200), (8500, 61, 190), (4001, 2050, 1100),
                                   (2899, 1301, 2900)])
def test_both_gradients_of_whole_numbers(m, n, k, kind):
    from gsx_amd import fields
    x, dy, w = _whole(m, k, 1, DTYPES[kind], pad=3), _whole(m, n, 2, DTYPES[kind], pad=1), _whole(n, k, 3)
    print(f"[case] gradients {m} x {n} x {k} {kind}", flush=True)
    dx, dw = fields.linear_backward(x, dy, fields.quantize(w, transpose=True))
    assert torch.equal(dx, _once(dy.double() @ w.double(), DTYPES[kind]))
    assert torch.equal(dw, _once(dy.double().T @ x.double(), torch.float32))


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(40, 50, 1100), (300, 310, 1024), (2899, 2900, 1301), (3900, 3901, 1100)])
def test_infinities_and_nan_stay_in_their_rows_of_16_bit_results(m, n, k, out):
    from gsx_amd import fields
    x, w = _whole(m, k, 1), _whole(n, k, 2)
    clean = fields.matmul(fields.quantize(x), fields.quantize(w), out_dtype=DTYPES[out])
    x[m // 2, k - 1], x[1, 7], w[n - 1, 130] = float("nan"), float("inf"), -float("inf")
    got = fields.matmul(fields.quantize(x), fields.quantize(w), out_dtype=DTYPES[out])
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[[1, m // 2]], bad[:, n - 1] = True, True
    assert torch.equal(torch.isnan(got), bad)
    # what a NaN displaces in its block leaves the block's other values as they were only if they are exact either way: they are
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("out", ["bf16", "f16"])
def test_smallest_and_largest_blocks_in_16_bit_results(out):
    """Scales from 2^-100 to 2^118 on one side; the other side's brings the products back as far as it may: no bit is lost."""
    from gsx_amd import fields
    k, n = 1152, 70
    x, w = fields.quantize(_whole(6, k, 1)), fields.quantize(_whole(n, k, 2))
    one = [fields.Blocks(t.values, torch.full_like(t.exponents, 127), k) for t in (x, w)]
    base = fields.matmul(*one).double()
    for e in (-100, -99, -60, 60, 100, 118):
        back = max(-100, -10 - e)  # 2^-10 of the sums of E4M3 values fit a float16
        a, b = (fields.Blocks(t.values, torch.full_like(t.exponents, 127 + s), k) for t, s in zip(one, (e, back)))
        got = fields.matmul(a, b, out_dtype=DTYPES[out])
        assert torch.equal(got, (base * 2.0 ** (e + back)).float().to(DTYPES[out])), e


def _distill_want(z, ids, t, temperature, weight, scale):
    """Loss and gradient in float64, a part of the rows at a time."""
    loss, grad = [], []
    for at in range(0, z.shape[0], 64):
        r = slice(at, at + 64)
        log_q = torch.log_softmax(z[r].double() / temperature, 1)
        log_p = torch.log_softmax(t[r].double() / temperature, 1)
        entry, p = ids[r].long(), log_p.exp()
        loss.append(weight[r].double() * temperature**2 * (p * (log_p - log_q.gather(1, entry))).sum(1))
        g = log_q.exp().scatter_add_(1, entry, -p)
        grad.append((weight[r].double() * scale[r].double() * temperature)[:, None] * g)
    return torch.cat(loss), torch.cat(grad)


@pytest.mark.parametrize("rows,vocab,top", [s[:3] for s in DISTILLS])
def test_distillation(rows, vocab, top):
    """Loss with its gradient, loss alone, and the gradient in a later call. Logits lie within 12 of each other: exponentials are
    off by 2^-24 of an exponent of 12 log2(e) twice, sums of positive terms by 2^-24 for each of 64 + vocab / 1024 + 16 additions in a row (a
    group of 64 threads or more, vectors of 4), and log p - log q by as much and a few roundings of a number below 32."""
    from gsx_amd import fields
    g = torch.Generator("cuda").manual_seed(rows)
    z = torch.rand(rows, vocab, device="cuda", generator=g) * 12
    ids = torch.rand(rows, vocab, device="cuda", generator=g).topk(top, 1).indices.int()
    t = torch.rand(rows, top, device="cuda", generator=g) * 6
    weight, up = (torch.rand(rows, device="cuda", generator=g) + 0.5 for _ in range(2))
    temperature = 2.0
    print(f"[case] distill {rows} x {vocab} top {top}", flush=True)
    loss, stats, grad = fields.distill(z, ids, t, temperature, weight, grad_scale=0.75)
    alone, stats2, _ = fields.distill(z, ids, t, temperature, weight)
    apart = fields.distill_backward(z, stats2, ids, t, up, temperature, weight)
    assert torch.equal(alone, loss) and torch.equal(stats, stats2)
    off = 12 / temperature * 2.0**-22 + (64 + vocab / 1024 + 16 + top / 64 + 8) * 2.0**-24 + 2.0**-21
    for got, scale in ((grad, torch.full_like(up, 0.75)), (apart, up)):
        want, wanted = _distill_want(z, ids, t, temperature, weight, scale)
        assert ((loss.double() - want).abs() <= off * 32 * temperature**2 * weight).all()
        # the two parts of a gradient are off by `off` of themselves, and p <= 1, q <= 1
        q = torch.softmax(z.double() / temperature, 1)
        size = q.scatter_add_(1, ids.long(), torch.softmax(t.double() / temperature, 1))
        size *= (weight.double() * scale.double() * temperature)[:, None]
        assert ((got.double() - wanted).abs() <= off * size + 2.0**-126).all()
        del want, wanted, q, size


FIRST_CALL = """
import sys
sys.path.insert(0, {root!r})
import torch
from gsx_amd import fields
x = torch.randint(-8, 9, (3000, 100), device="cuda").bfloat16()
values = torch.randint(0, 120, (150, 128), device="cuda").to(torch.uint8)
w = fields.Blocks(values, torch.full((150, 4), 120, dtype=torch.uint8, device="cuda"), 100)
out = torch.zeros(3000, 150, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    fields.linear(x, w, out=out)
for k in range(3):
    x.copy_(torch.randint(-8, 9, (3000, 100), device="cuda").bfloat16())
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, fields.linear(x, w, out_dtype=torch.float32)) and out.abs().sum() > 0, k
print("replayed")
"""


def test_first_call_of_a_narrow_layer_in_a_capture():
    """The library's first narrow layer is captured: what it asks HIP for once is asked during the capture."""
    res = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=ROOT)], capture_output=True, text=True, timeout=110)
    assert res.returncode == 0 and "replayed" in res.stdout, res.stdout + res.stderr
