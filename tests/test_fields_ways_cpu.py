"""Which kernels the label fields' calls launch by their sizes, and what their host code makes of HIP's errors, on a stand-in
for the runtime (fake_hip.c) in a process of its own: no GPU is needed or touched."""
import os
import subprocess
import sys
import textwrap

import pytest

from fields_ways import DISTILLS, LINEARS, PRODUCTS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# HIP's answer to how many workgroups of a kernel a CU takes: what a test says, or a refusal that stays the last error
OCCUPANCY = """
#include "fake_hip.c"
static int each_cu = 3;
void fake_set_each_cu(int n) { each_cu = n; }
int hipOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *f, int threads, size_t lds)
{
    (void)f; (void)threads; (void)lds;
    if(each_cu < 0) return set(INVALID_VALUE);
    *n = each_cu;
    return OK;
}
"""

PRELUDE = """
import ctypes, sys
sys.path.insert(0, {root!r})
sys.path.insert(0, {root!r} + "/tests")
from gsx_amd import _lib
fake = ctypes.CDLL({fake!r})
fake.fake_threads_of.restype = ctypes.c_uint64
lib = _lib.load(require_device=False)
P = 0x7000000000  # an address on the device
up = lambda a, b: -(-a // b) * b
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    at = tmp_path_factory.mktemp("fake")
    source, fake = str(at / "occupancy.c"), str(at / "libfakehip.so")
    with open(source, "w") as f:
        f.write(OCCUPANCY)
    subprocess.run(["gcc", "-std=c11", "-O1", "-fPIC", "-shared", "-Wall", "-I", os.path.join(ROOT, "tests"), "-o", fake, source],
                   check=True)
    preload = ":".join([fake] + ([os.environ["LD_PRELOAD"]] if os.environ.get("LD_PRELOAD") else []))

    def run(code):
        text = PRELUDE.format(root=ROOT, fake=fake) + textwrap.dedent(code)
        res = subprocess.run([sys.executable, "-c", text], env={**os.environ, "LD_PRELOAD": preload}, capture_output=True,
                             text=True, timeout=120)
        assert res.returncode == 0, res.stdout + res.stderr
    return run


TYPES = {"f": 0, "DF16b": 3, "DF16_": 4}


@pytest.mark.parametrize("out", TYPES)
def test_products_take_the_kernels_that_the_tests_mean(host, out):
    host(f"""
for m, n, k, name in {PRODUCTS!r}:
    before = fake.fake_launches_of(b"product_kernel")
    one = fake.fake_launches_of(("product_kernelI{out}" + name).encode())
    row, words = up(k, 128), up(up(k, 128) // 128, 4)
    _lib.check(lib.gsx_hip_blocks_matmul(P, row, P, words, P, row, P, words, m, n, k, P, {TYPES[out]}, n, P, None), "product")
    assert fake.fake_launches_of(b"product_kernel") == before + 1
    assert fake.fake_launches_of(("product_kernelI{out}" + name).encode()) == one + 1, (m, n, k)
""")


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("x", TYPES)
def test_linears_take_the_kernels_that_the_tests_mean(host, x, out):
    host(f"""
for m, n, k, name in {LINEARS!r}:
    name = name.format(x={x!r}, out={out!r}).encode()
    row, words = up(k, 128), up(up(k, 128) // 128, 4)
    _lib.check(lib.gsx_hip_linear_forward(P, {TYPES[x]}, k, P, row, P, words, m, n, k, P, {TYPES[out]}, n, P, None), "linear")
    assert fake.fake_launches_of(name) >= 1, (m, n, k, name)
""")


def test_distillations_take_the_kernels_that_the_tests_mean(host):
    host(f"""
for rows, vocab, top, name in {DISTILLS!r}:
    before, name = fake.fake_launches_of(name.encode()), name.encode()
    _lib.check(lib.gsx_hip_distill_forward(P, 0, vocab, rows, vocab, P, P, top, top, 1.0, None, P, P, P + (1 << 36), vocab, 1.0, P,
                                           None), "distill")
    assert fake.fake_launches_of(name) == before + (2 if b"finish" in name else 1), (rows, vocab, top)
""")


def test_a_refused_occupancy_query_ends_the_call_and_is_not_kept(host):
    """A narrow layer asks how many workgroups a CU takes. If HIP refuses, nothing is launched, the caller gets HIP's error, no error
    is left for later calls, and the next call asks again."""
    host("""
def linear():
    return lib.gsx_hip_linear_forward(P, 0, 128, P, 128, P, 4, 307200, 150, 128, P, 0, 150, None, None)

fake.fake_set_each_cu(-1)
assert linear() == 1  # HIP's code for an invalid value
assert fake.fake_launches_of(b"linear_head") == 0
assert fake.hipGetLastError() == 0
assert b"linear" in lib.gsx_hip_last_error_message()
fake.fake_set_each_cu(3)
_lib.check(linear(), "linear")
assert fake.fake_launches_of(b"linear_head") == 1 and fake.fake_threads_of(b"linear_head") == 3 * 256 * 256
""")


def test_a_weight_whose_rows_lie_too_far_apart_is_refused_before_anything_runs(host):
    """The tiled product takes value rows less than 2^28 bytes apart; other ways of a linear layer have no such limit."""
    host("""
far = 1 << 28
assert lib.gsx_hip_linear_forward(P, 0, 1024, P, far, P, 8, 300, 300, 1024, P, 0, 300, P, None) == -3
assert b"2^28" in lib.gsx_hip_last_error_message()
assert fake.fake_launches() == 0
_lib.check(lib.gsx_hip_linear_forward(P, 0, 1024, P, far - 16, P, 8, 300, 300, 1024, P, 0, 300, P, None), "linear")
_lib.check(lib.gsx_hip_linear_forward(P, 0, 1024, P, far, P, 8, 1, 300, 1024, P, 0, 300, None, None), "linear")
""")
