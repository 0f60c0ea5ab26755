"""What the 4-bit blocks' C entries refuse, and which kernels their sizes lead to: nothing runs on a GPU."""
import pytest

from blocks4_ways import LINEARS, PRODUCTS
from gsx_amd import _lib
from test_fields_ways_cpu import TYPES, host  # noqa: F401  (the stand-in for the runtime)

P = 0x7000000000


def _lib_():
    return _lib.load(require_device=False)


@pytest.mark.parametrize("how,code", [
    (dict(type=2), -5), (dict(rows=-1), -1), (dict(stride=99), -1), (dict(src=None), -1), (dict(src=P + 2), -1),
    (dict(values=None), -1), (dict(values=P + 8), -1), (dict(values_stride=40), -1), (dict(values_stride=48), -1),
    (dict(exponents=P + 2), -1), (dict(exponents_stride=6), -1), (dict(exponents_stride=0), -1), (dict(rows=1 << 60), -1)])
def test_refused_quantisations(how, code):
    a = dict(src=P, type=0, rows=3, cols=100, stride=100, values=P, values_stride=64, exponents=P, exponents_stride=4, stream=None)
    assert _lib_().gsx_hip_blocks4_quantize(*dict(a, **how).values()) == code
    assert b"4-bit" in _lib_().gsx_hip_last_error_message()


@pytest.mark.parametrize("how,code", [
    (dict(type=1), -5), (dict(out=None), -1), (dict(out=P + 2), -1), (dict(stride=99), -1), (dict(values=None), -1),
    (dict(cols=-1), -1), (dict(values_stride=32), -1), (dict(exponents=None), -1)])
def test_refused_expansions(how, code):
    a = dict(values=P, values_stride=64, exponents=P, exponents_stride=4, rows=3, cols=100, out=P, type=0, stride=100, stream=None)
    assert _lib_().gsx_hip_blocks4_expand(*dict(a, **how).values()) == code


@pytest.mark.parametrize("how,code", [
    (dict(type=6), -5), (dict(m=1 << 31), -3), (dict(n=-1), -3), (dict(k=(1 << 27) + 1), -3), (dict(a_stride=1 << 28), -3),
    (dict(b_stride=1 << 28), -3), (dict(a=None), -1), (dict(be=None), -1), (dict(b=P + 4), -1), (dict(a_stride=24), -1),
    (dict(be_stride=2), -1), (dict(out=None), -1), (dict(out=P + 1), -1), (dict(out_stride=49), -1),
    (dict(m=2, n=50, k=100_000, a_stride=50_000, b_stride=50_000, ae_stride=3128, be_stride=3128, temp=None), -1)])
def test_refused_products(how, code):
    a = dict(a=P, a_stride=64, ae=P, ae_stride=4, b=P, b_stride=64, be=P, be_stride=4, m=40, n=50, k=100, out=P, type=0,
             out_stride=50, temp=P, stream=None)
    assert _lib_().gsx_hip_blocks4_matmul(*dict(a, **how).values()) == code


@pytest.mark.parametrize("how,code", [
    (dict(type=1), -5), (dict(out_type=1), -5), (dict(m=-1), -3), (dict(k=1 << 28), -3), (dict(x_stride=99), -1),
    (dict(out_stride=299), -1), (dict(w=None), -1), (dict(x=None), -1), (dict(x=P + 2), -1), (dict(out=None), -1),
    (dict(temp=None), -1), (dict(temp=P + 8), -1), (dict(w_stride=1 << 28), -3)])
def test_refused_linears(how, code):
    a = dict(x=P, type=0, x_stride=100, w=P, w_stride=64, we=P, we_stride=4, m=400, n=300, k=100, out=P, out_type=0,
             out_stride=300, temp=P, stream=None)
    assert _lib_().gsx_hip_linear4_forward(*dict(a, **how).values()) == code


def test_nothing_to_do():
    lib = _lib_()
    assert lib.gsx_hip_blocks4_quantize(None, 0, 0, 100, 100, None, 64, None, 4, None) == 0
    assert lib.gsx_hip_blocks4_expand(None, 64, None, 4, 0, 100, None, 0, 100, None) == 0
    assert lib.gsx_hip_blocks4_matmul(None, 64, None, 4, P, 64, P, 4, 0, 5, 100, None, 0, 5, None, None) == 0
    assert lib.gsx_hip_linear4_forward(None, 0, 100, P, 64, P, 4, 0, 5, 100, None, 0, 5, None, None) == 0
    assert lib.gsx_hip_linear4_temp_bytes(0, 5, 100) == 0 and lib.gsx_hip_blocks4_matmul_temp_bytes(-1, 5, 100) == 0


@pytest.mark.parametrize("out", TYPES)
def test_products_take_the_kernels_that_the_tests_mean(host, out):  # noqa: F811
    host(f"""
for m, n, k, name in {PRODUCTS!r}:
    before = fake.fake_launches_of(b"product4_kernel")
    one = fake.fake_launches_of(("product4_kernelI{out}" + name).encode())
    row, words = up(up(k, 32) // 2, 16), up(up(k, 32) // 32, 4)
    _lib.check(lib.gsx_hip_blocks4_matmul(P, row, P, words, P, row, P, words, m, n, k, P, {TYPES[out]}, n, P, None), "product")
    assert fake.fake_launches_of(b"product4_kernel") == before + 1
    assert fake.fake_launches_of(("product4_kernelI{out}" + name).encode()) == one + 1, (m, n, k)
""")


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("x", TYPES)
def test_linears_take_the_kernels_that_the_tests_mean(host, x, out):  # noqa: F811
    host(f"""
for m, n, k, wide, name in {LINEARS!r}:
    if wide != ({x!r} == "f") * 2 + 2:
        continue
    name = name.format(x={x!r}, out={out!r}).encode()
    before = fake.fake_launches_of(name)
    row, words = up(up(k, 32) // 2, 16), up(up(k, 32) // 32, 4)
    temp = P if lib.gsx_hip_linear4_temp_bytes(m, n, k) else None
    _lib.check(lib.gsx_hip_linear4_forward(P, {TYPES[x]}, k, P, row, P, words, m, n, k, P, {TYPES[out]}, n, temp, None), "linear")
    assert fake.fake_launches_of(name) == before + 1, (m, n, k, name)
""")
