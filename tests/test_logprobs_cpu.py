"""What the log probabilities' C entries refuse, and which kernels their sizes lead to: nothing runs on a GPU."""
import pytest

from gsx_amd import _lib
from logprobs_ways import WAYS
from test_fields_ways_cpu import host  # noqa: F401  (the stand-in for the runtime)

P = 0x7000000000
FAR = 1 << 36


def _forward(lib=None, **how):
    lib = lib or _lib.load(require_device=False)
    a = dict(logits=P, type=0, stride=100, rows=3, vocab=100, ids=P, temperature=1.0, chosen=P, entropy=P, stats=P, top=5,
             top_ids=P, top_logs=P, grad=None, grad_stride=100, row_grad=None, grad_scale=0.0, entropy_grad=None,
             entropy_scale=0.0, temp=P, stream=None)
    assert not set(how) - set(a)
    return lib.gsx_hip_log_probs_forward(*dict(a, **how).values())


@pytest.mark.parametrize("how,code", [
    (dict(logits=None), -1), (dict(type=1), -5), (dict(stride=99), -1), (dict(rows=-1), -1), (dict(vocab=0, top=0), -3),
    (dict(vocab=1 << 31, stride=1 << 31), -3), (dict(rows=1 << 60), -1), (dict(top=65), -3), (dict(top=-1), -3),
    (dict(vocab=4), -3), (dict(top_ids=None), -1), (dict(top_logs=None), -1), (dict(temperature=0.0), -1),
    (dict(temperature=1e7), -1), (dict(temperature=float("nan")), -1), (dict(logits=P + 2), -1), (dict(ids=P + 2), -1),
    (dict(chosen=P + 1), -1), (dict(grad=P), -1), (dict(grad=P + FAR, grad_stride=99), -1), (dict(grad=P + FAR, stats=None), -1),
    (dict(grad=P + FAR + 2), -1), (dict(row_grad=P + 2), -1),
    (dict(rows=1, vocab=100_000, stride=100_000, temp=None), -1), (dict(rows=1, vocab=100_000, stride=100_000, temp=P + 8), -1)])
def test_refused_calls(how, code):
    assert _forward(**how) == code
    assert b"log probabilities" in _lib.load(require_device=False).gsx_hip_last_error_message()


@pytest.mark.parametrize("how", [dict(stats=None), dict(grad=None), dict(logits=None), dict(type=2), dict(vocab=0),
                                 dict(temperature=-1.0), dict(stats=P + 2), dict(grad_stride=50)])
def test_refused_backward(how):
    a = dict(logits=P, type=3, stride=100, rows=3, vocab=100, ids=None, temperature=1.0, stats=P, row_grad=None, grad_scale=1.0,
             entropy_grad=None, entropy_scale=0.0, grad=P + FAR, grad_stride=100, stream=None)
    assert _lib.load(require_device=False).gsx_hip_log_probs_backward(*dict(a, **how).values()) < 0


def test_no_rows_do_nothing():
    assert _forward(rows=0, logits=None, top_ids=None) == 0


def test_workspaces():
    lib = _lib.load(require_device=False)
    size = lib.gsx_hip_log_probs_temp_bytes
    assert size(1, 131072, 20) > 0 and size(4096, 1000, 20) == 0
    assert size(0, 131072, 20) == 0 and size(1, 1 << 31, 1) == 0 and size(1, 100_000, 65) == 0 and size(1 << 50, 1 << 30, 0) == 0


@pytest.mark.parametrize("kind", {"f": 0, "DF16b": 3, "DF16_": 4}.items())
def test_sizes_take_the_kernels_that_the_tests_mean(host, kind):  # noqa: F811
    host(f"""
for rows, vocab, top, name in {WAYS[kind[0]]!r}:
    name = name.encode()
    before = fake.fake_launches_of(name)
    _lib.check(lib.gsx_hip_log_probs_forward(P, {kind[1]}, vocab, rows, vocab, P, 1.0, P, P, P, top, P, P, P + (1 << 36), vocab,
                                             None, 1.0, None, 0.0, P, None), "log probabilities")
    assert fake.fake_launches_of(name) == before + 1, (rows, vocab, top, name)
""")


def test_more_rows_than_a_grid_has_workgroups(host):  # noqa: F811
    host("""
_lib.check(lib.gsx_hip_log_probs_forward(P, 3, 300, 1 << 33, 300, None, 1.0, P, P, P, 1, P, P, None, 0, None, 0.0, None, 0.0, None,
                                         None), "log probabilities")
assert fake.fake_threads_of(b"logprobs_held") == 256 << 20
""")
