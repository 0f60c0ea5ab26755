"""What AdamW's C entries refuse, and the layout of its structs: nothing is launched, no GPU is needed."""
import ctypes

import pytest

from gsx_amd import _lib

P = 0x7000000000  # an address on the device
FAR = 1 << 32


def _tensor(**how):
    t = _lib.AdamwTensor()
    at = dict(parameter=P, gradient=P + FAR, first=P + 2 * FAR, second=P + 3 * FAR, first_scale=P + 4 * FAR,
              second_scale=P + 5 * FAR, count=1000, parameter_type=0, gradient_type=3, bits=8, group=0)
    at.update(how)
    for k, v in at.items():
        setattr(t, k, v)
    return t


def _fill(*tensors):
    lib = _lib.load(require_device=False)
    arr = (_lib.AdamwTensor * max(1, len(tensors)))(*tensors)
    size = lib.gsx_hip_adamw_table_bytes(arr, len(tensors))
    table = (ctypes.c_int64 * (max(size, 4096) // 8 + 1))()
    chunks = ctypes.c_int64(-1)
    st = lib.gsx_hip_adamw_table_fill(arr, len(tensors), table, ctypes.byref(chunks))
    return st, size, chunks.value


def test_struct_sizes():
    assert ctypes.sizeof(_lib.AdamwTensor) == 7 * 8 + 4 * 4
    assert ctypes.sizeof(_lib.AdamwGroup) == 5 * 8


def test_tables_have_a_chunk_for_every_2048_elements():
    assert _fill() == (0, 16, 0)
    one = _fill(_tensor(count=1))
    assert one[0] == 0 and one[2] == 1
    far = 16 * FAR
    two = _fill(_tensor(count=2049), *[_tensor(**{k: P + (j + 1) * far + i * FAR for i, k in enumerate(
        ("parameter", "gradient", "first", "second", "first_scale", "second_scale"))}, count=n) for j, n in enumerate((0, 2048))])
    assert two[0] == 0 and two[2] == 3 and two[1] == 16 + 3 * 72 + 3 * 8


@pytest.mark.parametrize("how,code,word", [
    (dict(parameter=None), -1, b"null"),
    (dict(gradient=None), -1, b"null"),
    (dict(first=None), -1, b"null"),
    (dict(second_scale=None), -1, b"null"),
    (dict(parameter_type=1), -5, b"f32"),
    (dict(gradient_type=7), -5, b"f32"),
    (dict(bits=16), -5, b"8 bits or 32"),
    (dict(count=-1), -1, b">= 0"),
    (dict(group=16), -1, b"groups"),
    (dict(group=-1), -1, b"groups"),
    (dict(parameter=P + 2), -1, b"aligned"),
    (dict(gradient=P + FAR + 1), -1, b"aligned"),
    (dict(first=P + 2 * FAR + 4), -1, b"aligned"),
    (dict(count=(1 << 24) * 2048, bits=32), -3, b"2^24"),
    (dict(count=1 << 62), -3, b"2^24"),
])
def test_refused_tensors(how, code, word):
    st, size, _ = _fill(_tensor(**how))
    assert st == code and size == 0
    assert word in _lib.load(require_device=False).gsx_hip_last_error_message()


@pytest.mark.parametrize("how", [
    dict(gradient=P),                      # a gradient in the parameter's place
    dict(second=P + 2 * FAR),              # one buffer for both moments
    dict(second=P + 2 * FAR + 1016),       # the last block is whole: 1024 bytes
    dict(first_scale=P + 3996),            # the parameter's last element
    dict(second_scale=P + 4 * FAR + 28),   # the last of eight scales
])
def test_what_a_step_writes_may_not_overlap(how):
    assert _fill(_tensor(**how))[0] == -1


def test_tensors_that_only_touch_or_share_a_gradient():
    a = _tensor()
    b = _tensor(parameter=P + 4000, first=P + 2 * FAR + 1024, second=P + 3 * FAR + 1024, first_scale=P + 4 * FAR + 32,
                second_scale=P + 5 * FAR + 32)
    assert _fill(a, b)[0] == 0
    assert _fill(a, a)[0] == -1
    assert _fill(a, _tensor(count=0))[0] == 0


def _step(groups=None, count=1, chunks=1, table=P, steps=P + 64, factors=P + 128, factor=None, **how):
    lib = _lib.load(require_device=False)
    g = _lib.AdamwGroup(**dict(dict(beta1=0.9, beta2=0.999, learning_rate=1e-3, weight_decay=0.01, epsilon=1e-8), **how))
    arr = (_lib.AdamwGroup * 16)(*[g] * 16)
    return lib.gsx_hip_adamw_step(table, chunks, arr if groups is None else groups, count, 1.0, factor, steps, factors, None)


@pytest.mark.parametrize("how", [
    dict(count=0), dict(count=17), dict(table=None), dict(steps=None), dict(factors=None), dict(table=P + 4),
    dict(factor=P + 2), dict(beta1=1.0), dict(beta2=-0.1), dict(beta1=float("nan")), dict(epsilon=0.0),
    dict(epsilon=1e-60), dict(weight_decay=-1.0), dict(learning_rate=float("inf")), dict(weight_decay=float("nan"))])
def test_refused_steps(how):
    assert _step(**how) == -1


def test_too_many_chunks():
    assert _step(chunks=1 << 24) == -3 and _step(chunks=-1) == -3


def test_refused_moments():
    lib = _lib.load(require_device=False)
    at = [P + i * FAR for i in range(6)]
    assert lib.gsx_hip_moments_hold(at[0], at[1], -1, *at[2:], None) == -3
    assert lib.gsx_hip_moments_hold(None, at[1], 1, *at[2:], None) == -1
    assert lib.gsx_hip_moments_hold(at[0], at[1], 1, at[2] + 4, *at[3:], None) == -1
    assert lib.gsx_hip_moments_read(*at[:4], 1, None, at[5], None) == -1
    assert lib.gsx_hip_moments_read(*at[:4], 1 << 60, *at[4:], None) == -3
    assert lib.gsx_hip_moments_read(None, None, None, None, 0, None, None, None) == 0
