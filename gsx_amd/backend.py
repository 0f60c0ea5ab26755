"""Host-side mirror of gsx's renderer / loss / optimizer interface over libgsx_hip.so.

Names and semantics follow the gsx public API (gsx/include/gsx/gsx-render.h, gsx-loss.h,
gsx-optim.h): a render context retains TRAIN state for exactly one backward; gradient sinks
of the render backward are overwritten; loss maps and prediction gradients accumulate; Adam
keeps per-group moments and step counts. Device memory and streams come from PyTorch (ROCm);
every computation runs in the HIP kernels of libgsx_hip.so.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import Camera, GaussianGrads, Gaussians, GsxHipError, check
from .fields import _current_stream

__all__ = ["Camera", "Renderer", "Loss", "Adam", "AdamW", "DensityControl", "GsxHipError", "stream_handle", "ptr"]


def ptr(t: torch.Tensor | None):
    if t is None:
        return None
    if not t.is_cuda:
        raise GsxHipError("gsx_amd tensors must live on the HIP device")
    if not t.is_contiguous():
        raise GsxHipError("gsx_amd tensors must be contiguous")
    if t.dtype not in (torch.float32, torch.int32, torch.uint32, torch.int64, torch.uint64, torch.uint8):
        raise GsxHipError(f"unsupported dtype {t.dtype}")
    return ctypes.c_void_p(t.data_ptr())


def stream_handle(stream: torch.cuda.Stream | None = None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


@dataclass
class GaussianTensors:
    mean3d: torch.Tensor
    rotation: torch.Tensor
    logscale: torch.Tensor
    opacity: torch.Tensor
    sh0: torch.Tensor
    sh_degree: int = 0
    sh1: torch.Tensor | None = None
    sh2: torch.Tensor | None = None
    sh3: torch.Tensor | None = None

    @property
    def count(self) -> int:
        return int(self.mean3d.shape[0])

    def to_struct(self) -> Gaussians:
        g = Gaussians()
        g.count = self.count
        g.sh_degree = self.sh_degree
        for name in ("mean3d", "rotation", "logscale", "opacity", "sh0", "sh1", "sh2", "sh3"):
            setattr(g, name, ptr(getattr(self, name)))
        return g

    @classmethod
    def from_scene(cls, scene, device="cuda") -> "GaussianTensors":
        def t(a):
            return None if a is None else torch.from_numpy(a).to(device)
        return cls(t(scene.mean3d), t(scene.rotation), t(scene.logscale), t(scene.opacity), t(scene.sh0),
                   scene.sh_degree, t(scene.sh1), t(scene.sh2), t(scene.sh3))

    def zeros_like_grads(self) -> "GaussianTensors":
        z = lambda a: None if a is None else torch.zeros_like(a)  # noqa: E731
        return GaussianTensors(z(self.mean3d), z(self.rotation), z(self.logscale), z(self.opacity), z(self.sh0),
                               self.sh_degree, z(self.sh1), z(self.sh2), z(self.sh3))

    def grads_struct(self) -> GaussianGrads:
        g = GaussianGrads()
        for name in ("mean3d", "rotation", "logscale", "opacity", "sh0", "sh1", "sh2", "sh3"):
            setattr(g, name, ptr(getattr(self, name)))
        return g


class Renderer:
    """gsx_renderer + gsx_render_context on the HIP backend (gsx-render.h:148-165)."""

    def __init__(self, width: int, height: int):
        self.lib = _lib.load()
        self.width = int(width)
        self.height = int(height)
        h = ctypes.c_void_p()
        check(self.lib.gsx_hip_render_context_create(ctypes.byref(h)), "render context create")
        self.handle = h

    def close(self):
        if getattr(self, "handle", None) is not None and self.handle.value:
            self.lib.gsx_hip_render_context_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def render(self, camera: Camera, gaussians: GaussianTensors, train: bool = False,
               out_rgb: torch.Tensor | None = None, visible_counter: torch.Tensor | None = None,
               stream=None, borrow_train_state: bool = True) -> torch.Tensor:
        """train=True is GSX_RENDER_FORWARD_TYPE_TRAIN. borrow_train_state (gsx-render.h:101): True
        differentiates the backward at the values the Gaussian tensors hold when backward() is
        called, False at the values of this forward."""
        if camera.width != self.width or camera.height != self.height:
            raise GsxHipError("intrinsics geometry must match the renderer output geometry")
        if out_rgb is None:
            out_rgb = torch.empty((3, self.height, self.width), dtype=torch.float32, device="cuda")
        g = gaussians.to_struct()
        mode = (_lib.FORWARD_TRAIN_BORROW if borrow_train_state else _lib.FORWARD_TRAIN_CLONE) if train else \
            _lib.FORWARD_INFERENCE
        check(self.lib.gsx_hip_render_forward(self.handle, ctypes.byref(camera), ctypes.byref(g), mode,
                                              ptr(out_rgb), ptr(visible_counter), stream_handle(stream)),
              "render forward")
        return out_rgb

    def backward(self, grad_rgb: torch.Tensor, grads: GaussianTensors, stream=None) -> None:
        gg = grads.grads_struct()
        check(self.lib.gsx_hip_render_backward(self.handle, ptr(grad_rgb), ctypes.byref(gg), stream_handle(stream)),
              "render backward")

    def stats(self) -> _lib.RenderStats:
        s = _lib.RenderStats()
        check(self.lib.gsx_hip_render_context_get_stats(self.handle, ctypes.byref(s)), "get stats")
        return s

    def buffers(self) -> _lib.RenderBuffers:
        b = _lib.RenderBuffers()
        check(self.lib.gsx_hip_render_context_get_buffers(self.handle, ctypes.byref(b)), "get buffers")
        return b

    def set_timing(self, capacity: int) -> None:
        """Record per-stage HIP events for the next `capacity` forward/backward pairs (0 = off)."""
        check(self.lib.gsx_hip_render_context_set_timing(self.handle, int(capacity)), "set timing")

    STAGES = ("preprocess", "depth_order", "emit", "sort", "ranges", "blend_forward", "blend_backward", "instance_reduce",
              "projection_backward")

    def timings(self) -> dict:
        arr = (ctypes.c_float * len(self.STAGES))()
        written = ctypes.c_int32(0)
        check(self.lib.gsx_hip_render_context_get_timings(self.handle, arr, len(self.STAGES), ctypes.byref(written)),
              "get timings")
        return {name: float(arr[i]) for i, name in enumerate(self.STAGES[: written.value])}


class Loss:
    """gsx_loss for L1 / MSE / SSIM (gsx-loss.h). grad_normalization 'mean' divides by the
    element count (gsx-tensor-helpers.h:236-244)."""

    def __init__(self, algorithm: str, grad_normalization: str = "mean"):
        if algorithm not in ("l1", "mse", "ssim"):
            raise GsxHipError(f"unknown loss algorithm {algorithm}")
        self.lib = _lib.load()
        self.algorithm = algorithm
        self.mean = grad_normalization == "mean"
        self._pred = None
        self._target = None
        self._workspace = None

    def _grad_scale(self, numel: int, scale: float) -> float:
        s = ctypes.c_float(scale).value
        return ctypes.c_float(s / ctypes.c_float(float(numel)).value).value if self.mean else s

    @staticmethod
    def _image_layout(t: torch.Tensor):
        if t.dim() == 3:
            return 1, t.shape[0], t.shape[1], t.shape[2]
        if t.dim() == 4:
            return t.shape[0], t.shape[1], t.shape[2], t.shape[3]
        raise GsxHipError("ssim expects [C,H,W] or [B,C,H,W]")

    def forward(self, prediction: torch.Tensor, target: torch.Tensor, loss_map: torch.Tensor, scale: float = 1.0,
                train: bool = True, stream=None) -> None:
        n = prediction.numel()
        st = stream_handle(stream)
        if self.algorithm == "ssim":
            outer, c, h, w = self._image_layout(prediction)
            if self._workspace is None or self._workspace.numel() < 3 * n:
                self._workspace = torch.empty(3 * n, dtype=torch.float32, device="cuda")
            check(self.lib.gsx_hip_loss_ssim_chw_f32_forward_kernel_launch(
                ptr(loss_map), ptr(prediction), ptr(target), outer, c, h, w, scale,
                ptr(self._workspace) if train else None, 0.0, 0, st), "ssim forward")
        elif self.algorithm == "l1":
            check(self.lib.gsx_hip_loss_l1_f32_forward_kernel_launch(ptr(loss_map), ptr(prediction), ptr(target), n,
                                                                     scale, st), "l1 forward")
        else:
            check(self.lib.gsx_hip_loss_mse_f32_forward_kernel_launch(ptr(loss_map), ptr(prediction), ptr(target), n,
                                                                      scale, st), "mse forward")
        self._pred, self._target = (prediction, target) if train else (None, None)

    def backward(self, grad_prediction: torch.Tensor, scale: float = 1.0, stream=None) -> None:
        if self._pred is None:
            raise GsxHipError("loss backward requires a train forward on the same context")
        n = self._pred.numel()
        gs = self._grad_scale(n, scale)
        st = stream_handle(stream)
        if self.algorithm == "ssim":
            outer, c, h, w = self._image_layout(self._pred)
            check(self.lib.gsx_hip_loss_ssim_chw_f32_backward_kernel_launch(
                ptr(grad_prediction), ptr(self._pred), ptr(self._target), outer, c, h, w, gs, ptr(self._workspace),
                0.0, 0, st), "ssim backward")
        elif self.algorithm == "l1":
            check(self.lib.gsx_hip_loss_l1_f32_backward_kernel_launch(ptr(grad_prediction), ptr(self._pred),
                                                                      ptr(self._target), n, gs, st), "l1 backward")
        else:
            check(self.lib.gsx_hip_loss_mse_f32_backward_kernel_launch(ptr(grad_prediction), ptr(self._pred),
                                                                       ptr(self._target), n, gs, st), "mse backward")


class Adam:
    """gsx_optim (Adam) over parameter groups, all groups in one launch per step."""

    def __init__(self, groups):
        """groups: list of dicts with parameter, gradient, learning_rate and optional beta1, beta2,
        weight_decay, epsilon, max_grad (defaults 0.9, 0.999, 0, 1e-8, 0)."""
        if len(groups) > _lib.ADAM_MAX_GROUPS:
            raise GsxHipError("too many parameter groups")
        self.lib = _lib.load()
        self.groups = []
        for g in groups:
            p = g["parameter"]
            self.groups.append(dict(parameter=p, gradient=g["gradient"], learning_rate=float(g["learning_rate"]),
                                    beta1=float(g.get("beta1", 0.9)), beta2=float(g.get("beta2", 0.999)),
                                    weight_decay=float(g.get("weight_decay", 0.0)),
                                    epsilon=float(g.get("epsilon", 1e-8)), max_grad=float(g.get("max_grad", 0.0)),
                                    m=torch.zeros_like(p), v=torch.zeros_like(p), step=0))

    def step(self, stream=None) -> None:
        arr = (_lib.AdamGroup * len(self.groups))()
        for i, g in enumerate(self.groups):
            g["step"] += 1
            b1 = ctypes.c_float(g["beta1"]).value
            b2 = ctypes.c_float(g["beta2"]).value
            a = arr[i]
            a.parameter = ptr(g["parameter"])
            a.gradient = ptr(g["gradient"])
            a.first_moment = ptr(g["m"])
            a.second_moment = ptr(g["v"])
            a.count = g["parameter"].numel()
            a.beta1, a.beta2 = b1, b2
            a.learning_rate = g["learning_rate"]
            a.weight_decay = g["weight_decay"]
            a.epsilon = g["epsilon"]
            a.max_grad = g["max_grad"]
            a.bias_correction1 = 1.0 - math.pow(b1, float(g["step"]))
            a.bias_correction2 = 1.0 - math.pow(b2, float(g["step"]))
        check(self.lib.gsx_hip_adam_step_multi_launch(arr, len(self.groups), stream_handle(stream)), "adam step")


class AdamW:
    """AdamW over any number of tensors in one launch, with moments in 32 bits or in 8 (include/gsx_hip.h has the formulas and
    the format). `Adam` is gsx's: up to 16 float32 tensors, steps counted on the host, so that it cannot be replayed.

    groups: up to 16 dicts of `parameters` and `gradients` (lists of contiguous tensors of the same sizes, float32, bfloat16 or
    float16, whose memory stays in use by this optimizer) and of learning_rate, beta1, beta2, weight_decay and epsilon, which may
    be changed in `groups` between steps. All moments lie in one buffer, in the order of the tensors, each from a multiple of 128
    values on (`offsets`). Steps are counted on the device: a step captured into a graph counts at every replay, with the
    rates of its capture."""

    BLOCK = 128
    _TYPES = {torch.float32: 0, torch.bfloat16: 3, torch.float16: 4}  # GSX_HIP_DTYPE_*

    def __init__(self, groups: list[dict], bits: int = 32):
        self.lib = _lib.load()
        if bits not in (8, 32):
            raise GsxHipError(f"moments have 8 bits or 32, not {bits}")
        if not 1 <= len(groups) <= _lib.ADAM_MAX_GROUPS:
            raise GsxHipError(f"1 to {_lib.ADAM_MAX_GROUPS} groups, not {len(groups)}")
        self.bits = bits
        self.device = torch.cuda.current_device()
        self.groups = []
        self.offsets = []
        self._tensors = []  # (group, parameter, gradient)
        total = 0
        for k, g in enumerate(groups):
            parameters, gradients = list(g["parameters"]), list(g["gradients"])
            if len(parameters) != len(gradients):
                raise GsxHipError("a group needs a gradient for each parameter")
            for p, d in zip(parameters, gradients):
                for t in (p, d):
                    if t.get_device() != self.device:
                        raise GsxHipError("parameters and gradients must live on the current HIP device")
                    if t.dtype not in self._TYPES:
                        raise GsxHipError(f"parameters and gradients are float32, bfloat16 or float16, not {t.dtype}")
                    if not t.is_contiguous():
                        raise GsxHipError("parameters and gradients must be contiguous")
                if p.shape != d.shape:
                    raise GsxHipError(f"a gradient of shape {tuple(d.shape)} for a parameter of shape {tuple(p.shape)}")
                self._tensors.append((k, p, d))
                self.offsets.append(total)
                total += -(-p.numel() // self.BLOCK) * self.BLOCK
            self.groups.append(dict(learning_rate=float(g["learning_rate"]), beta1=float(g.get("beta1", 0.9)),
                                    beta2=float(g.get("beta2", 0.999)), weight_decay=float(g.get("weight_decay", 0.01)),
                                    epsilon=float(g.get("epsilon", 1e-8))))
        self.size = total
        kind = torch.uint8 if bits == 8 else torch.float32
        self.first = torch.zeros(total, dtype=kind, device="cuda")
        self.second = torch.zeros(total, dtype=kind, device="cuda")
        self.first_scale = self.second_scale = None
        if bits == 8:
            self.first_scale = torch.full((total // self.BLOCK,), 2.0**-126, device="cuda")
            self.second_scale = torch.full((total // self.BLOCK,), 2.0**-126, device="cuda")
        self.steps = torch.zeros(1, dtype=torch.int64, device="cuda")
        self._factors = torch.zeros(2 * _lib.ADAM_MAX_GROUPS, device="cuda")
        self._lay_out()
        stream = torch.cuda.current_stream()
        stream.synchronize()  # steps may run on any stream
        self._stream = stream.cuda_stream

    def _lay_out(self):
        wide = self.first.element_size()
        entries = (_lib.AdamwTensor * max(1, len(self._tensors)))()
        for e, at, (k, p, d) in zip(entries, self.offsets, self._tensors):
            e.parameter, e.gradient, e.count, e.group, e.bits = p.data_ptr(), d.data_ptr(), p.numel(), k, self.bits
            e.parameter_type, e.gradient_type = self._TYPES[p.dtype], self._TYPES[d.dtype]
            e.first, e.second = self.first.data_ptr() + at * wide, self.second.data_ptr() + at * wide
            if self.bits == 8:
                e.first_scale = self.first_scale.data_ptr() + at // self.BLOCK * 4
                e.second_scale = self.second_scale.data_ptr() + at // self.BLOCK * 4
        size = self.lib.gsx_hip_adamw_table_bytes(entries, len(self._tensors))
        table = torch.empty(max(size, 16) // 8, dtype=torch.int64)
        chunks = ctypes.c_int64(0)
        check(self.lib.gsx_hip_adamw_table_fill(entries, len(self._tensors), table.data_ptr(), ctypes.byref(chunks)),
              "adamw table")
        self._table, self._chunks = table.cuda(), chunks.value

    def _on(self, stream):
        """The handle of a call's stream, whose use of this optimizer's memory the allocator is told of."""
        if torch.cuda.current_device() != self.device:
            raise GsxHipError("the optimizer's device must be the current one")
        handle = _current_stream(self.device) if stream is None else stream.cuda_stream
        if handle != self._stream:
            s = torch.cuda.current_stream() if stream is None else stream
            for t in (self.first, self.second, self.first_scale, self.second_scale, self.steps, self._factors, self._table):
                if t is not None:
                    t.record_stream(s)
        return handle

    def step(self, grad_scale: float = 1.0, grad_factor: torch.Tensor | None = None, stream=None) -> None:
        """One step. Gradients are multiplied by grad_scale and by what grad_factor, one float32 on the device, holds then."""
        if grad_factor is not None and (grad_factor.get_device() != self.device or grad_factor.dtype != torch.float32 or
                                        grad_factor.numel() != 1):
            raise GsxHipError("grad_factor must be one float32 on the current HIP device")
        handle = self._on(stream)
        arr = (_lib.AdamwGroup * len(self.groups))()
        for a, g in zip(arr, self.groups):
            a.beta1, a.beta2, a.learning_rate = g["beta1"], g["beta2"], g["learning_rate"]
            a.weight_decay, a.epsilon = g["weight_decay"], g["epsilon"]
        check(self.lib.gsx_hip_adamw_step(self._table.data_ptr(), self._chunks, arr, len(self.groups), grad_scale,
                                          None if grad_factor is None else grad_factor.data_ptr(), self.steps.data_ptr(),
                                          self._factors.data_ptr(), handle), "adamw step")

    def moments(self, stream=None):
        """(first, second) moments in float32, each [size]; tensor i's from offsets[i] on, 0 between the tensors. With 32 bits
        they are the optimizer's own."""
        if self.bits == 32:
            return self.first, self.second
        handle = self._on(stream)
        with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
            first, second = (torch.empty(self.size, device="cuda") for _ in range(2))
        check(self.lib.gsx_hip_moments_read(self.first.data_ptr(), self.first_scale.data_ptr(), self.second.data_ptr(),
                                            self.second_scale.data_ptr(), self.size // self.BLOCK, first.data_ptr(),
                                            second.data_ptr(), handle), "moments")
        return first, second

    def load(self, first: torch.Tensor, second: torch.Tensor, steps: int, stream=None) -> None:
        """Goes on from moments laid out as `moments` gives them (0 between the tensors, second ones >= 0) after `steps` steps."""
        for t in (first, second):
            if t.get_device() != self.device or t.dtype != torch.float32 or t.shape != (self.size,) or not t.is_contiguous():
                raise GsxHipError(f"moments are {self.size} contiguous float32 values on the current HIP device")
        if steps < 0:
            raise GsxHipError("the number of steps must be >= 0")
        handle = self._on(stream)
        with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
            self.steps.fill_(int(steps))
            if self.bits == 32:
                self.first.copy_(first)
                self.second.copy_(second)
            else:
                check(self.lib.gsx_hip_moments_hold(first.data_ptr(), second.data_ptr(), self.size // self.BLOCK,
                                                    self.first.data_ptr(), self.first_scale.data_ptr(),
                                                    self.second.data_ptr(), self.second_scale.data_ptr(), handle), "moments")


FIELD_WIDTHS = {"mean3d": 3, "rotation": 4, "logscale": 3, "opacity": 1, "sh0": 3, "sh1": 9, "sh2": 15, "sh3": 21}
PARAM_FIELDS = ("mean3d", "rotation", "logscale", "opacity", "sh0", "sh1", "sh2", "sh3")
AUX_FIELDS = ("grad_acc", "absgrad_acc", "visible_counter", "max_screen_radius")


class DensityControl:
    """gsx_adc (DEFAULT / ABSGS) on the HIP backend (gsx-adc.h). Rows live in capacity-sized
    device buffers: growth appends in place, pruning compacts into a second buffer set."""

    def __init__(self, params: dict, seed: int = 0):
        self.lib = _lib.load()
        p = _lib.AdcParams()
        for name, _ in _lib.AdcParams._fields_:
            if name in params:
                setattr(p, name, params[name])
        self.params = p
        h = ctypes.c_void_p()
        check(self.lib.gsx_hip_adc_context_create(ctypes.byref(h), int(seed)), "adc context create")
        self.handle = h

    def close(self):
        if getattr(self, "handle", None) is not None and self.handle.value:
            self.lib.gsx_hip_adc_context_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def rows_struct(count: int, sh_degree: int, fields: dict, moments: dict | None) -> _lib.GsRows:
        r = _lib.GsRows()
        r.count = count
        r.sh_degree = sh_degree
        for name in PARAM_FIELDS + AUX_FIELDS:
            setattr(r, name, ptr(fields.get(name)))
        if moments is not None:
            for k, name in enumerate(PARAM_FIELDS):
                if name in moments:
                    r.first_moment[k] = ptr(moments[name][0])
                    r.second_moment[k] = ptr(moments[name][1])
        return r

    def step(self, global_step: int, count: int, sh_degree: int, fields: dict, moments: dict | None,
             capacity: int, out_fields: dict, out_moments: dict | None, stream=None):
        """Returns (new_count, result_in_out, counts[pruned, duplicated, grown, reset])."""
        rows = self.rows_struct(count, sh_degree, fields, moments)
        out = self.rows_struct(0, sh_degree, out_fields, out_moments)
        in_out = ctypes.c_int32(0)
        counts = (ctypes.c_int64 * 4)()
        check(self.lib.gsx_hip_adc_step(self.handle, ctypes.byref(self.params), int(global_step), ctypes.byref(rows),
                                        int(capacity), ctypes.byref(out), ctypes.byref(in_out), counts,
                                        stream_handle(stream)), "adc step")
        new_count = out.count if in_out.value else rows.count
        return int(new_count), bool(in_out.value), list(counts)
