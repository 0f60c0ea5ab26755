"""Label fields over libgsx_hip.so: rows looked up by code, a head in 8-bit or 4-bit blocks, distillation from a teacher's top
logits, log probabilities of given labels.

A field gives each Gaussian or pixel the id of a code. `lookup` fetches the codes' rows, `linear` multiplies them with a head
whose weights are `Blocks` (8-bit values with a power-of-two scale for each block of 128), `distill` compares the logits with
a teacher's top logits and gives their gradient, and `linear_backward` and `lookup_backward` carry it to the weights and the
table, in float32 for `gsx_amd.backend.Adam` or `AdamW`. `log_probs` compares the logits with given labels instead, or gives the
likeliest ones; a head that only answers can be `Blocks4` (4-bit values, a scale for each block of 32). Definitions, rounding and
the treatment of masked ids and rows are those of include/gsx_hip.h.

Tensors are two-dimensional with contiguous rows of any stride (ids and weights one-dimensional and contiguous), all on the
current device. Results and workspaces that a call allocates belong to the stream it runs on: `stream`, or torch's current one.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from ._lib import GsxHipError, check

__all__ = ["Blocks", "Blocks4", "lookup", "lookup_backward", "quantize", "quantize4", "matmul", "linear", "linear_backward", "distill",
           "distill_backward", "LogProbs", "log_probs", "log_probs_backward"]

_TYPES = {torch.float32: 0, torch.bfloat16: 3, torch.float16: 4}  # GSX_HIP_DTYPE_*
BLOCK = 128
BLOCK4 = 32


def _type(dtype) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise GsxHipError(f"label fields take float32, bfloat16 and float16 rows, not {dtype}")
    return code


def _rows(t: torch.Tensor, what: str, dtype=None, shape=None):
    """(address, stride) of a matrix with contiguous rows."""
    if t.get_device() != _device():
        raise GsxHipError(f"{what} must live on the current HIP device")
    if dtype is not None and t.dtype != dtype:
        raise GsxHipError(f"{what} must be {dtype}, not {t.dtype}")
    size = t.shape
    if len(size) != 2 or (shape is not None and size != shape):
        raise GsxHipError(f"{what} must be a matrix{'' if shape is None else f' of shape {shape}'}, not {tuple(size)}")
    rows, cols = size
    step, inner = t.stride()
    stride = step if rows > 1 and cols > 0 else cols
    if (cols > 1 and inner != 1) or stride < cols:
        raise GsxHipError(f"{what} must have contiguous rows that do not overlap")
    return t.data_ptr(), stride


def _vector(t: torch.Tensor | None, what: str, dtype, count: int):
    if t is None:
        return None
    if t.get_device() != _device():
        raise GsxHipError(f"{what} must live on the current HIP device")
    if t.dtype != dtype or t.shape != (count,) or not t.is_contiguous():
        raise GsxHipError(f"{what} must be {count} contiguous {dtype} values")
    return t.data_ptr()


_device = torch.cuda.current_device
# the current stream's handle without a Stream object around it: a quarter of a small call's time
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _run(stream, call):
    """call(stream handle) with what it allocates belonging to the stream that it runs on."""
    if stream is None:
        return call(_current_stream(_device()))
    with torch.cuda.stream(stream):
        return call(stream.cuda_stream)


def _temp(size: int):
    return torch.empty(size, dtype=torch.uint8, device="cuda") if size else None


def _address(t):
    return None if t is None else t.data_ptr()


def lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, out: torch.Tensor | None = None, out_dtype=None,
           out_of_range: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """out[i] = scale * table[ids[i]] (int32 ids). An id outside the table gives zeros; out_of_range, one int32, is set to 1 if
    such an id is not negative."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(table, "table")
    code = _type(table.dtype)
    count, width = ids.numel(), table.shape[1]
    id_ptr = _vector(ids, "ids", torch.int32, count)
    flag = _vector(out_of_range, "out_of_range", torch.int32, 1)

    def call(handle):
        result = out
        if result is None:
            result = torch.empty((count, width), dtype=out_dtype or table.dtype, device=table.device)
        to, to_stride = _rows(result, "out", out_dtype, (count, width))
        check(lib.gsx_hip_lookup_forward(base, code, table.shape[0], stride, id_ptr, count, width, scale, to,
                                         _type(result.dtype), to_stride, flag, handle), "lookup")
        return result

    return _run(stream, call)


def lookup_backward(grad_out: torch.Tensor, ids: torch.Tensor, table_rows: int, scale: float = 1.0,
                    grad_table: torch.Tensor | None = None, accumulate: bool = False, stream=None) -> torch.Tensor:
    """grad_table[v] = scale * the sum of grad_out[i] over the i with ids[i] = v, in float32; accumulate adds it instead."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(grad_out, "grad_out")
    code = _type(grad_out.dtype)
    count, width = grad_out.shape
    id_ptr = _vector(ids, "ids", torch.int32, count)
    if accumulate and grad_table is None:
        raise GsxHipError("accumulate needs a grad_table")

    def call(handle):
        result = grad_table
        if result is None:
            result = torch.empty((table_rows, width), dtype=torch.float32, device=grad_out.device)
        to, to_stride = _rows(result, "grad_table", torch.float32, (table_rows, width))
        temp = _temp(lib.gsx_hip_lookup_backward_temp_bytes(count, table_rows, width))
        check(lib.gsx_hip_lookup_backward(base, code, stride, id_ptr, count, width, scale, to, table_rows, to_stride,
                                          int(accumulate), _address(temp), handle), "lookup backward")
        return result

    return _run(stream, call)


@dataclass
class Blocks:
    """A matrix [rows, cols] in 8-bit blocks: values uint8 [rows, at least cols], exponents uint8 [rows, at least
    ceil(cols / 128)], their rows 16 and 4 bytes aligned."""

    values: torch.Tensor
    exponents: torch.Tensor
    cols: int

    @property
    def rows(self) -> int:
        return int(self.values.shape[0])

    def arguments(self):
        v, v_stride = _rows(self.values, "values", torch.uint8)
        e, e_stride = _rows(self.exponents, "exponents", torch.uint8)
        if self.exponents.shape[0] != self.rows or self.values.shape[1] < self.cols or \
                self.exponents.shape[1] < -(-self.cols // BLOCK):
            raise GsxHipError("values and exponents must cover the same rows and all columns")
        return v, _padded(v_stride, 16, self.rows), e, _padded(e_stride, 4, self.rows)

    def float(self) -> torch.Tensor:
        """The values that the blocks stand for, float32 [rows, cols]."""
        n = -(-self.cols // BLOCK)
        scale = torch.exp2(self.exponents[:, :n].float() - 127).repeat_interleave(BLOCK, 1)[:, : self.cols]
        return self.values[:, : self.cols].view(torch.float8_e4m3fn).float() * scale


def _padded(stride: int, to: int, rows: int) -> int:
    return stride if rows > 1 else -(-stride // to) * to  # a single row's stride is never used


def _blocks_room(kind, block: int, size: int, rows: int, cols: int, out, device):
    """`out`, or new blocks, as `kind` of a matrix [rows, cols] whose rows have room for whole blocks of `size` bytes and whole
    words of exponents, and its arguments."""
    n = -(-cols // block)
    wide, words = n * size, -(-n // 4) * 4
    if out is None:
        values = torch.empty((rows, wide), dtype=torch.uint8, device=device)
        exponents = torch.empty((rows, words), dtype=torch.uint8, device=device)
        return kind(values, exponents, cols), (values.data_ptr(), wide, exponents.data_ptr(), words)
    if not isinstance(out, kind) or out.values.dim() != 2 or out.exponents.dim() != 2 or out.rows != rows or \
            out.cols != cols or out.values.shape[1] < wide or out.exponents.shape[1] < words:
        raise GsxHipError(f"out must be {kind.__name__} of a matrix [{rows}, {cols}] with {wide} values and {words} exponents a row")
    return out, out.arguments()


def quantize(x: torch.Tensor, transpose: bool = False, stream=None, out: Blocks | None = None) -> Blocks:
    """x, or its transpose, in 8-bit blocks along the result's rows. `out`: blocks of a matrix of the same sizes, as an earlier call
    gave them, that are written instead of new ones; what reads their memory, a replayed graph too, finds x there from then on."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(x, "x")
    code = _type(x.dtype)
    rows, cols = (x.shape[1], x.shape[0]) if transpose else x.shape

    def call(handle):
        result, args = _blocks_room(Blocks, BLOCK, BLOCK, rows, cols, out, x.device)
        check(lib.gsx_hip_blocks_quantize(base, code, x.shape[0], x.shape[1], stride, int(transpose), *args, handle), "quantize")
        return result

    return _run(stream, call)


@dataclass
class Blocks4:
    """A matrix [rows, cols] in microscaled 4-bit blocks: values uint8 [rows, at least ceil(cols / 2)], two a byte, exponents uint8
    [rows, at least ceil(cols / 32)], their rows 16 and 4 bytes aligned."""

    values: torch.Tensor
    exponents: torch.Tensor
    cols: int

    @property
    def rows(self) -> int:
        return int(self.values.shape[0])

    def arguments(self):
        v, v_stride = _rows(self.values, "values", torch.uint8)
        e, e_stride = _rows(self.exponents, "exponents", torch.uint8)
        if self.exponents.shape[0] != self.rows or self.values.shape[1] * 2 < self.cols or \
                self.exponents.shape[1] < -(-self.cols // BLOCK4):
            raise GsxHipError("values and exponents must cover the same rows and all columns")
        return v, _padded(v_stride, 16, self.rows), e, _padded(e_stride, 4, self.rows)

    def float(self, out_dtype=torch.float32, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """The values that the blocks stand for, [rows, cols]."""
        lib = _lib.load(require_device=False)
        args = self.arguments()

        def call(handle):
            shape = (self.rows, self.cols)
            result = torch.empty(shape, dtype=out_dtype, device=self.values.device) if out is None else out
            to, to_stride = _rows(result, "out", None, shape)
            check(lib.gsx_hip_blocks4_expand(*args, *shape, to, _type(result.dtype), to_stride, handle), "4-bit blocks")
            return result

        return _run(stream, call)


def quantize4(x: torch.Tensor, stream=None, out: Blocks4 | None = None) -> Blocks4:
    """x in microscaled 4-bit blocks along its rows, written into `out` as `quantize` does if that is given."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(x, "x")
    code = _type(x.dtype)
    rows, cols = x.shape

    def call(handle):
        result, args = _blocks_room(Blocks4, BLOCK4, BLOCK4 // 2, rows, cols, out, x.device)
        check(lib.gsx_hip_blocks4_quantize(base, code, rows, cols, stride, *args, handle), "quantize4")
        return result

    return _run(stream, call)


def matmul(a: Blocks | Blocks4, b: Blocks | Blocks4, out_dtype=torch.float32, out: torch.Tensor | None = None,
           stream=None) -> torch.Tensor:
    """a b^T, [a.rows, b.rows], for operands in blocks of one kind."""
    lib = _lib.load(require_device=False)
    if isinstance(a, Blocks4) != isinstance(b, Blocks4):
        raise GsxHipError("the operands must both be in 8-bit blocks, or both in 4-bit blocks")
    if a.cols != b.cols:
        raise GsxHipError(f"the operands' rows have {a.cols} and {b.cols} values")
    m, n, k = a.rows, b.rows, a.cols
    a_args, b_args = a.arguments(), b.arguments()
    if isinstance(a, Blocks4):
        temp_bytes, product = lib.gsx_hip_blocks4_matmul_temp_bytes, lib.gsx_hip_blocks4_matmul
    else:
        temp_bytes, product = lib.gsx_hip_blocks_matmul_temp_bytes, lib.gsx_hip_blocks_matmul

    def call(handle):
        result = torch.empty((m, n), dtype=out_dtype, device=a.values.device) if out is None else out
        to, to_stride = _rows(result, "out", None, (m, n))
        temp = _temp(temp_bytes(m, n, k))
        check(product(*a_args, *b_args, m, n, k, to, _type(result.dtype), to_stride, _address(temp), handle), "block product")
        return result

    return _run(stream, call)


def linear(x: torch.Tensor, weight: Blocks | Blocks4, out_dtype=None, out: torch.Tensor | None = None,
           stream=None) -> torch.Tensor:
    """x weight^T with the rows of x quantised on the way, to the weight's kind of blocks; the result has x's type unless out_dtype
    or out says otherwise."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(x, "x")
    code = _type(x.dtype)
    m, k = x.shape
    n = weight.rows
    if weight.cols != k:
        raise GsxHipError(f"x has {k} columns, the weight {weight.cols}")
    w_args = weight.arguments()
    if isinstance(weight, Blocks4):
        temp_bytes, forward = lib.gsx_hip_linear4_temp_bytes, lib.gsx_hip_linear4_forward
    else:
        temp_bytes, forward = lib.gsx_hip_linear_temp_bytes, lib.gsx_hip_linear_forward

    def call(handle):
        result = torch.empty((m, n), dtype=out_dtype or x.dtype, device=x.device) if out is None else out
        to, to_stride = _rows(result, "out", out_dtype, (m, n))
        temp = _temp(temp_bytes(m, n, k))
        check(forward(base, code, stride, *w_args, m, n, k, to, _type(result.dtype), to_stride, _address(temp), handle), "linear")
        return result

    return _run(stream, call)


def linear_backward(x: torch.Tensor, grad_out: torch.Tensor, weight_t: Blocks, grad_weight: torch.Tensor | None = None,
                    stream=None):
    """Gradients of linear(x, weight) for the upstream grad_out [m, n]: (grad_x in grad_out's type, grad_weight float32).

    weight_t holds the transposed weight [k, n] in blocks. grad_x = blocks(grad_out) weight_t^T and
    grad_weight = blocks(grad_out^T) blocks(x^T)^T: every operand is quantised along the axis that is summed over."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(x, "x")
    grad_base, grad_stride = _rows(grad_out, "grad_out")
    x_type, grad_type = _type(x.dtype), _type(grad_out.dtype)
    m, k = x.shape
    n = grad_out.shape[1]
    if grad_out.shape[0] != m:
        raise GsxHipError("x and grad_out must have the same number of rows")
    if isinstance(weight_t, Blocks4):
        raise GsxHipError("gradients go through 8-bit blocks: weight_t must be Blocks")
    if weight_t.cols != n or weight_t.rows != k:
        raise GsxHipError(f"weight_t must be [{k}, {n}], not [{weight_t.rows}, {weight_t.cols}]")
    grad_x = linear(grad_out, weight_t, stream=stream)

    def call(handle):
        result = torch.empty((n, k), dtype=torch.float32, device=x.device) if grad_weight is None else grad_weight
        to, to_stride = _rows(result, "grad_weight", torch.float32, (n, k))
        temp = _temp(lib.gsx_hip_linear_backward_weight_temp_bytes(x_type, grad_type, m, n, k))
        check(lib.gsx_hip_linear_backward_weight(base, x_type, stride, grad_base, grad_type, grad_stride, m, n, k, to,
                                                 to_stride, _address(temp), handle), "linear backward")
        return result

    return grad_x, _run(stream, call)


def _teacher(logits, teacher_ids, teacher_logits, row_weight):
    rows = logits.shape[0]
    ids, ids_stride = _rows(teacher_ids, "teacher_ids", torch.int32)
    t, t_stride = _rows(teacher_logits, "teacher_logits", torch.float32, tuple(teacher_ids.shape))
    if teacher_ids.shape[0] != rows or ids_stride != t_stride:
        raise GsxHipError("teacher_ids and teacher_logits must have a row for each row of logits, at the same stride")
    return ids, t, t_stride, teacher_ids.shape[1], _vector(row_weight, "row_weight", torch.float32, rows)


def distill(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, temperature: float = 1.0,
            row_weight: torch.Tensor | None = None, grad_scale: float | None = None, grad: torch.Tensor | None = None,
            stream=None):
    """(loss [rows], row_stats [rows, 2], gradient or None) of the rows of `logits` against the teacher's top entries (int32 ids,
    float32 logits). With grad_scale, the upstream gradient of every row's loss, the logits' gradient comes from the same pass
    (into `grad` if given); row_stats are for `distill_backward`."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(logits, "logits")
    code = _type(logits.dtype)
    rows, vocab = logits.shape
    ids, t, t_stride, top, weight = _teacher(logits, teacher_ids, teacher_logits, row_weight)
    if grad is not None and grad_scale is None:
        raise GsxHipError("a gradient needs a grad_scale")

    def call(handle):
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
        stats = torch.empty((rows, 2), dtype=torch.float32, device=logits.device)
        result, to, to_stride = grad, None, 0
        if grad_scale is not None:
            if result is None:
                result = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
            to, to_stride = _rows(result, "grad", logits.dtype, (rows, vocab))
        temp = _temp(lib.gsx_hip_distill_temp_bytes(rows, vocab))
        check(lib.gsx_hip_distill_forward(base, code, stride, rows, vocab, ids, t, t_stride, top, temperature, weight,
                                          loss.data_ptr(), stats.data_ptr(), to, to_stride, grad_scale or 0.0,
                                          _address(temp), handle), "distill")
        return loss, stats, result

    return _run(stream, call)


def distill_backward(logits: torch.Tensor, row_stats: torch.Tensor, teacher_ids: torch.Tensor,
                     teacher_logits: torch.Tensor, row_grad: torch.Tensor | None = None, temperature: float = 1.0,
                     row_weight: torch.Tensor | None = None, grad_scale: float = 1.0, grad: torch.Tensor | None = None,
                     stream=None) -> torch.Tensor:
    """The logits' gradient for upstream gradients grad_scale * row_grad of the rows' losses, from `distill`'s row_stats."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(logits, "logits")
    code = _type(logits.dtype)
    rows, vocab = logits.shape
    ids, t, t_stride, top, weight = _teacher(logits, teacher_ids, teacher_logits, row_weight)
    stats, stats_stride = _rows(row_stats, "row_stats", torch.float32, (rows, 2))
    if stats_stride != 2:
        raise GsxHipError("row_stats must be contiguous")
    upstream = _vector(row_grad, "row_grad", torch.float32, rows)

    def call(handle):
        result = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device) if grad is None else grad
        to, to_stride = _rows(result, "grad", logits.dtype, (rows, vocab))
        check(lib.gsx_hip_distill_backward(base, code, stride, rows, vocab, ids, t, t_stride, top, temperature, weight,
                                           stats, upstream, grad_scale, to, to_stride, handle), "distill backward")
        return result

    return _run(stream, call)


class LogProbs(NamedTuple):
    """What `log_probs` says of each row; `top_ids` and `top_log_probs` are what `distill` takes as a teacher's entries."""

    chosen: torch.Tensor         # float32 [rows]: log probability of the given label, 0 for a row without one
    entropy: torch.Tensor        # float32 [rows]
    top_ids: torch.Tensor        # int32 [rows, top], -1 where there are fewer alternatives
    top_log_probs: torch.Tensor  # float32 [rows, top]
    row_stats: torch.Tensor      # float32 [rows, 3], for `log_probs_backward`
    grad: torch.Tensor | None    # the logits' gradient


def log_probs(logits: torch.Tensor, ids: torch.Tensor | None = None, top: int = 0, temperature: float = 1.0,
              grad_scale: float | None = None, row_grad: torch.Tensor | None = None, entropy_scale: float | None = None,
              entropy_grad: torch.Tensor | None = None, grad: torch.Tensor | None = None, stream=None) -> LogProbs:
    """Log probabilities of one int32 label a row (what lies outside the logits is no label), entropies and the `top` (at most 64)
    likeliest labels. With grad_scale or entropy_scale, the logits' gradient comes from the same pass (into `grad` if given): for
    upstream gradients grad_scale * row_grad of `chosen` and entropy_scale * entropy_grad of `entropy`."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(logits, "logits")
    code = _type(logits.dtype)
    rows, vocab = logits.shape
    id_ptr = _vector(ids, "ids", torch.int32, rows)
    upstream = _vector(row_grad, "row_grad", torch.float32, rows)
    entropy_upstream = _vector(entropy_grad, "entropy_grad", torch.float32, rows)
    wanted = grad_scale is not None or entropy_scale is not None
    if not wanted and not (grad is None and row_grad is None and entropy_grad is None):
        raise GsxHipError("a gradient needs a grad_scale or an entropy_scale")
    if (row_grad is not None and grad_scale is None) or (entropy_grad is not None and entropy_scale is None):
        raise GsxHipError("row_grad needs a grad_scale, entropy_grad an entropy_scale")
    if top < 0:
        raise GsxHipError("the number of alternatives must be >= 0")

    def call(handle):
        def floats(*shape):
            return torch.empty(shape, dtype=torch.float32, device=logits.device)

        chosen, entropy, stats, top_logs = floats(rows), floats(rows), floats(rows, 3), floats(rows, top)
        top_ids = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
        result, to, to_stride = grad, None, 0
        if wanted:
            if result is None:
                result = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
            to, to_stride = _rows(result, "grad", logits.dtype, (rows, vocab))
        temp = _temp(lib.gsx_hip_log_probs_temp_bytes(rows, vocab, top))
        check(lib.gsx_hip_log_probs_forward(base, code, stride, rows, vocab, id_ptr, temperature, chosen.data_ptr(),
                                            entropy.data_ptr(), stats.data_ptr(), top, top_ids.data_ptr(),
                                            top_logs.data_ptr(), to, to_stride, upstream, grad_scale or 0.0,
                                            entropy_upstream, entropy_scale or 0.0, _address(temp), handle),
              "log probabilities")
        return LogProbs(chosen, entropy, top_ids, top_logs, stats, result)

    return _run(stream, call)


def log_probs_backward(logits: torch.Tensor, row_stats: torch.Tensor, ids: torch.Tensor | None = None,
                       row_grad: torch.Tensor | None = None, entropy_grad: torch.Tensor | None = None,
                       temperature: float = 1.0, grad_scale: float = 1.0, entropy_scale: float | None = None,
                       grad: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The logits' gradient for upstream gradients grad_scale * row_grad of `chosen` and entropy_scale * entropy_grad of `entropy`
    (entropy_scale: 1 if there is an entropy_grad, else 0), from `log_probs`' row_stats."""
    lib = _lib.load(require_device=False)
    base, stride = _rows(logits, "logits")
    code = _type(logits.dtype)
    rows, vocab = logits.shape
    id_ptr = _vector(ids, "ids", torch.int32, rows)
    stats, stats_stride = _rows(row_stats, "row_stats", torch.float32, (rows, 3))
    if stats_stride != 3:
        raise GsxHipError("row_stats must be contiguous")
    upstream = _vector(row_grad, "row_grad", torch.float32, rows)
    entropy_upstream = _vector(entropy_grad, "entropy_grad", torch.float32, rows)
    if entropy_scale is None:
        entropy_scale = 0.0 if entropy_grad is None else 1.0

    def call(handle):
        result = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device) if grad is None else grad
        to, to_stride = _rows(result, "grad", logits.dtype, (rows, vocab))
        check(lib.gsx_hip_log_probs_backward(base, code, stride, rows, vocab, id_ptr, temperature, stats, upstream, grad_scale,
                                             entropy_upstream, entropy_scale, to, to_stride, handle),
              "log probabilities backward")
        return result

    return _run(stream, call)
