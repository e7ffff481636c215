"""Microscaled 4- and 8-bit tensors around the LoRA linear.

A frozen base weight in 4 bits, an activation kept for the backward pass in 8:

``mx_quantize`` / ``mx_dequantize``
    to and from ``mxfp4`` (E2M1 codes, a power of two per 32 values), ``nvfp4``
    (E2M1, an E4M3 scale per 16 values and one fp32 scale a tensor) and
    ``mxfp8`` (E4M3, a power of two per 32 values).
``mx_lora_linear``
    the LoRA linear with W and the quantised input in 4 bits (block-scaled
    tcgen05 MMAs) and the adapter in 16.
``mx_lora_forward`` / ``mx_lora_backward``
    the same with an 8-bit checkpoint of its input, and the gradients from it.
``MXLoRALinear``
    all of it as a module: a base frozen in 4 bits under a trainable adapter.

Everything runs in the sm_100a kernels behind ``include/lora_b200.h``; CPU
tensors raise.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_FORMATS = {"mxfp4": _lib.LORA_MXFP4, "nvfp4": _lib.LORA_NVFP4, "mxfp8": _lib.LORA_MXFP8}
_BLOCK = {"mxfp4": 32, "nvfp4": 16, "mxfp8": 32}
_HALF = (torch.float16, torch.bfloat16)
_DTYPE = {torch.float16: _lib.LORA_F16, torch.bfloat16: _lib.LORA_BF16}


# A call of a few tokens takes the GPU a few microseconds: the wrappers below pass
# plain integers to the C ABI, look the raw stream up directly and keep sizes by shape.
# (None in builds of PyTorch without CUDA, where no tensor gets that far)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


@functools.cache
def _entry(name: str):
    return getattr(_lib.load(), name)


@functools.lru_cache(maxsize=4096)
def _linear_bytes(m, n, k, r, code):
    return _entry("lora_mx_linear_workspace_size")(m, n, k, r, code)


@functools.lru_cache(maxsize=4096)
def _backward_bytes(m, n, k, r, flags):
    return _entry("lora_mx_backward_workspace_size")(m, n, k, r, flags)


def _need_cuda(where, *tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            _lib.require_cuda(t, where=where)


def _need_one_device(where, *tensors):
    _need_cuda(where, *tensors)
    devices = {str(t.device) for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"{where}: operands lie on different devices ({', '.join(sorted(devices))})")


def _elsewhere(device_index: int) -> bool:
    """Whether that GPU (-1: none) is not the current one, on which kernels launch."""
    return device_index >= 0 and device_index != _current_device()


def _format(fmt: str, where: str) -> int:
    code = _FORMATS.get(fmt)
    if code is None:
        raise ValueError(f"{where}: unknown format {fmt!r} (one of {', '.join(_FORMATS)})")
    return code


@functools.lru_cache(maxsize=4096)
def _sizes(m: int, k: int, fmt: str) -> tuple[int, int]:
    """Bytes of a row of codes, and of all scales, of an [m, k] tensor."""
    kp = (k + 31) // 32 * 32
    chunks = (kp // _BLOCK[fmt] + 3) // 4
    return (kp if fmt == "mxfp8" else kp // 2), (m + 127) // 128 * chunks * 512


class MXTensor:
    """An [M, K] tensor in a microscaled format.

    ``codes``: uint8 ``[M, Kp / 2]`` (4 bits, the even column in the low half of a
    byte) or ``[M, Kp]`` (8 bits), Kp = K rounded up to 32, zeros beyond K.
    ``scales``: uint8, flat, in 512-byte chunks of 128 rows x 4 blocks -- row r,
    block g of a chunk at byte ``16 (r % 32) + 4 (r / 32) + g``, the chunks of 128
    rows next to one another -- zeros beyond the tensor.  A value is
    ``code * scale * global_scale``; ``global_scale`` is 1 except for nvfp4.
    """

    __slots__ = ("codes", "scales", "shape", "fmt", "global_scale", "_code")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, fmt: str, global_scale: float = 1.0):
        self._code = _format(fmt, "MXTensor")
        m, k = shape
        m, k = int(m), int(k)
        pitch, nscales = _sizes(m, k, fmt)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("MXTensor: codes and scales are uint8")
        if codes.shape != (m, pitch) or scales.numel() != nscales:
            raise ValueError(f"MXTensor: a {fmt} tensor of shape {(m, k)} has codes {(m, pitch)} and {nscales} scale "
                             f"bytes, got {tuple(codes.shape)} and {scales.numel()}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("MXTensor: codes and scales must be contiguous")
        if codes.device != scales.device:
            raise ValueError("MXTensor: codes and scales lie on different devices")
        self.codes, self.scales, self.shape, self.fmt = codes, scales, (m, k), fmt
        self.global_scale = float(global_scale)

    @classmethod
    def _of(cls, codes, scales, shape, fmt, global_scale, code):
        """An MXTensor of buffers that the caller has laid out itself."""
        t = object.__new__(cls)
        t.codes, t.scales, t.shape, t.fmt, t.global_scale, t._code = codes, scales, shape, fmt, global_scale, code
        return t

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self):
        return f"MXTensor({self.fmt}, shape={self.shape}, global_scale={self.global_scale:g}, device={self.device})"


def nvfp4_global_scale(amax: float) -> float:
    """The nvfp4 tensor scale that maps ``amax`` to the largest code times the largest block scale."""
    return float(torch.tensor(max(float(amax), 2.0 ** -50) / (448.0 * 6.0), dtype=torch.float32))


def _rows(x: torch.Tensor, where: str) -> torch.Tensor:
    if x.dtype not in _HALF:
        raise TypeError(f"{where}: expected float16/bfloat16, got {x.dtype}")
    if x.dim() == 2 and x.is_contiguous():
        return x
    return _lib.row_major(x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4", global_scale: float = 1.0) -> MXTensor:
    """``x`` [..., K] (16-bit) in the format, as an [M, K] tensor.

    mxfp4 / mxfp8: scale ``2^(floor(log2 amax) - top)`` per 32 values (top = 2 / 8);
    nvfp4: ``E4M3(amax / (6 global_scale))`` per 16.  Codes round to nearest even
    and saturate; a block with an infinity or a NaN reads back as NaN.
    """
    code = _format(fmt, "mx_quantize")
    if _elsewhere(x.get_device()):
        with torch.cuda.device(x.device):
            return mx_quantize(x, fmt, global_scale)
    _need_cuda("mx_quantize", x)
    x = _rows(x, "mx_quantize")
    m, k = x.shape
    pitch, nscales = _sizes(m, k, fmt)
    device, dtype = x.device, x.dtype
    codes = x.new_empty((m, pitch), dtype=torch.uint8)
    scales = x.new_empty(nscales, dtype=torch.uint8)
    global_scale = float(global_scale)
    rc = _entry("lora_mx_quantize")(x.data_ptr(), _ld(x), codes.data_ptr(), scales.data_ptr(), m, k, code, global_scale,
                                    _DTYPE[dtype], _raw_stream(device.index))
    if rc:
        _lib.check(rc, "lora_mx_quantize")
    return MXTensor._of(codes, scales, (m, k), fmt, global_scale, code)


def mx_dequantize(q: MXTensor, dtype: torch.dtype = torch.bfloat16, transpose: bool = False) -> torch.Tensor:
    """The values of ``q`` in ``dtype`` (rounded once), [M, K] or, transposed, [K, M]."""
    if _elsewhere(q.codes.get_device()):
        with torch.cuda.device(q.codes.device):
            return mx_dequantize(q, dtype, transpose)
    _need_cuda("mx_dequantize", q.codes)
    if dtype not in _HALF:
        raise TypeError(f"mx_dequantize: expected float16/bfloat16, got {dtype}")
    m, k = q.shape
    device = q.codes.device
    out = q.codes.new_empty((k, m) if transpose else (m, k), dtype=dtype)
    rc = _entry("lora_mx_dequantize")(q.codes.data_ptr(), q.scales.data_ptr(), out.data_ptr(), m if transpose else k, m,
                                      k, q._code, q.global_scale, int(transpose), _DTYPE[dtype],
                                      _raw_stream(device.index))
    if rc:
        _lib.check(rc, "lora_mx_dequantize")
    return out


# --------------------------------------------------------------------- linear
def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """Row-major with 16-byte rows where the width allows it (copies only when needed)."""
    if not t.is_contiguous():
        t = _lib.row_major(t)
    if t.shape[1] % 8 == 0 and (_ld(t) % 8 != 0 or t.data_ptr() % 16 != 0):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _refuse_linear(x, weight, bias, a, b, where):
    """The error of a call that ``_linear``'s one check found wrong."""
    _need_one_device(where, x, weight.codes, bias, a, b)
    n, k = weight.shape
    if weight.fmt not in ("mxfp4", "nvfp4"):
        raise ValueError(f"{where}: the weight must be in a 4-bit format, got {weight.fmt}")
    if x.dtype not in _HALF:
        raise TypeError(f"{where}: expected float16/bfloat16, got {x.dtype}")
    if x.shape[-1] != k:
        raise ValueError(f"{where}: x {tuple(x.shape)} and the weight {weight.shape} disagree on K")
    if bias is not None and (bias.shape != (n,) or bias.dtype != x.dtype):
        raise ValueError(f"{where}: bias must be [{n}] in x's dtype")
    if a.dtype != x.dtype or b.dtype != x.dtype:
        raise TypeError(f"{where}: x, a and b must share one dtype")
    r = a.shape[0]
    if a.shape != (r, k) or b.shape != (n, r):
        raise ValueError(f"{where}: a {tuple(a.shape)} / b {tuple(b.shape)} do not match [{r}, {k}] / [{n}, {r}]")
    raise ValueError(f"{where}: ranks up to 256, got {r}")


def _linear(x, weight, bias, a, b, scale, x_global_scale, keep_z, where):
    dev = x.get_device()  # (-1: not on a GPU)
    if _elsewhere(dev):
        with torch.cuda.device(x.device):
            return _linear(x, weight, bias, a, b, scale, x_global_scale, keep_z, where)
    shape, dtype, codes, code = x.shape, x.dtype, weight.codes, weight._code
    n, k = weight.shape
    r = 0 if a is None or b is None or (scale == 0 and not keep_z) else a.shape[0]
    dt = _DTYPE.get(dtype)
    if (dt is None or code == _lib.LORA_MXFP8 or dev < 0 or codes.get_device() != dev or shape[-1] != k
            or (bias is not None and (bias.get_device() != dev or bias.dtype != dtype or bias.shape != (n,)))
            or (r and (r > 256 or a.dtype != dtype or b.dtype != dtype or a.get_device() != dev or b.get_device() != dev
                       or a.shape != (r, k) or b.shape != (n, r)))):
        _refuse_linear(x, weight, bias, a, b, where)
    if len(shape) != 2 or not x.is_contiguous():
        x = _rows(x, where)
    m = x.shape[0]
    xp, ap, bp, lda, ldb = x.data_ptr(), None, None, 0, 0
    ldx = _ld(x)
    if r:
        # TMA reads rows of 16-byte multiples: copies only where the layout is another
        if (xp | 2 * ldx) & 15 and k % 8 == 0:
            x = _aligned_rows(x)
            xp, ldx = x.data_ptr(), _ld(x)
        ap, bp, lda, ldb = a.data_ptr(), b.data_ptr(), k, r
        if not a.is_contiguous() or (ap | 2 * k) & 15:
            a = _aligned_rows(a)
            ap, lda = a.data_ptr(), _ld(a)
        if not b.is_contiguous() or (bp | 2 * r) & 15:
            b = _aligned_rows(b)
            bp, ldb = b.data_ptr(), _ld(b)
    if bias is not None:
        bias = bias.contiguous()
    out = x.new_empty((m, n))
    z = x.new_empty((m, 2 * ((r + 15) // 16 * 16))) if keep_z and r else None
    if m and n:
        device = x.device
        stream = _raw_stream(device.index)
        ws = _lib.WORKSPACE.get(_linear_bytes(m, n, k, r, code), device, "mx_linear", stream)
        rc = _entry("lora_mx_linear")(xp, ldx, codes.data_ptr(), weight.scales.data_ptr(), weight.global_scale,
                                      None if bias is None else bias.data_ptr(), ap, lda, bp, ldb, out.data_ptr(), n,
                                      None if z is None else z.data_ptr(), m, n, k, r, float(scale), float(x_global_scale),
                                      code, dt, ws.data_ptr(), ws.numel(), stream)
        if rc:
            _lib.check(rc, "lora_mx_linear")
    return (out if len(shape) == 2 else out.view(*shape[:-1], n)), z


def mx_lora_linear(x: torch.Tensor, weight: MXTensor, bias: torch.Tensor | None, a: torch.Tensor | None,
                   b: torch.Tensor | None, scale: float = 1.0, x_global_scale: float = 1.0) -> torch.Tensor:
    """``q(x) @ W.T + bias + scale * (x @ a.T) @ b.T`` with W (mxfp4 or nvfp4) and q(x) in 4 bits.

    x [..., K] is quantised to the weight's format (``x_global_scale``: its nvfp4
    tensor scale); the adapter a [r, K], b [N, r] (r <= 256) takes x itself.
    ``a`` / ``b`` None, or scale 0, leave the adapter out.
    """
    return _linear(x, weight, bias, a, b, scale, x_global_scale, False, "mx_lora_linear")[0]


# ------------------------------------------------------------------- training
def _refuse_backward(dy, x8, z, a, b, weight, where):
    """The error of a call that ``mx_lora_backward``'s one check found wrong."""
    _need_one_device(where, dy, x8.codes, z, a, b, weight.codes if weight is not None else None)
    m, n = dy.shape
    r, k = a.shape
    if dy.dtype not in _HALF:
        raise TypeError(f"{where}: expected float16/bfloat16, got {dy.dtype}")
    if x8.fmt != "mxfp8" or x8.shape != (m, k):
        raise ValueError(f"{where}: x8 must be an mxfp8 tensor of shape {(m, k)}, got {x8.fmt} {x8.shape}")
    if a.dtype != dy.dtype or b.dtype != dy.dtype or z.dtype != dy.dtype:
        raise TypeError(f"{where}: dy, z, a and b must share one dtype")
    if b.shape != (n, r) or not 1 <= r <= 256:
        raise ValueError(f"{where}: b {tuple(b.shape)} does not match [{n}, {r}] (1 <= r <= 256)")
    if z.shape != (m, 2 * ((r + 15) // 16 * 16)) or not z.is_contiguous():
        raise ValueError(f"{where}: z must be the contiguous [M, 2 * round_up(r, 16)] pair, got {tuple(z.shape)}")
    raise ValueError(f"{where}: the weight must be a 4-bit tensor of shape {(n, k)}, got {weight.fmt} {weight.shape}")


def mx_lora_backward(dy: torch.Tensor, x8: MXTensor, z: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                     scale: float = 1.0, weight: MXTensor | None = None, z_scale: float = 1.0):
    """Gradients ``(dx, da, db)`` of the LoRA linear from the 8-bit checkpoint of its input.

    ``g = scale * dy @ b``;  ``da = g.T @ X`` [r, K];  ``db = z_scale * dy.T @ z`` [N, r];
    ``dx = dy @ W + g @ a`` [..., K], or None without ``weight``.  ``x8`` is the mxfp8
    checkpoint of x, ``z`` the [M, 2 r16] pair [hi | lo] of the forward pass, W an mxfp4 /
    nvfp4 tensor.  W is frozen; rounding to 4 or 8 bits counts as the identity.
    """
    dev = dy.get_device()  # (-1: not on a GPU)
    if _elsewhere(dev):
        with torch.cuda.device(dy.device):
            return mx_lora_backward(dy, x8, z, a, b, scale, weight, z_scale)
    shape, dtype = dy.shape, dy.dtype
    wc = weight.codes if weight is not None else None
    if len(shape) != 2 or not dy.is_contiguous():
        _need_cuda("mx_lora_backward", dy)
        dy = _rows(dy, "mx_lora_backward")
    m, n = dy.shape
    r, k = a.shape
    dt = _DTYPE.get(dtype)
    if (dt is None or x8.fmt != "mxfp8" or x8.shape != (m, k) or a.dtype != dtype or b.dtype != dtype
            or z.dtype != dtype or b.shape != (n, r) or not 1 <= r <= 256
            or z.shape != (m, 2 * ((r + 15) // 16 * 16)) or not z.is_contiguous()
            or dev < 0 or x8.codes.get_device() != dev or z.get_device() != dev or a.get_device() != dev
            or b.get_device() != dev
            or (weight is not None and (weight._code == _lib.LORA_MXFP8 or weight.shape != (n, k)
                                        or wc.get_device() != dev))):
        _refuse_backward(dy, x8, z, a, b, weight, "mx_lora_backward")
    if not a.is_contiguous():
        a = _lib.row_major(a)
    if not b.is_contiguous():
        b = _lib.row_major(b)
    device = dy.device
    da, db = dy.new_empty((r, k)), dy.new_empty((n, r))
    dx = wp = sp = dxp = None
    wg, wcode = 1.0, 0
    dyp, lddy, bp, ldb = dy.data_ptr(), _ld(dy), b.data_ptr(), _ld(b)
    flags = _lib.LORA_MX_ONLY_BF16 if dtype == torch.bfloat16 else 0
    if (dyp | 2 * lddy) & 15 == 0:
        flags |= _lib.LORA_MX_DY_ALIGNED
    if (bp | 2 * ldb) & 15 == 0:
        flags |= _lib.LORA_MX_B_ALIGNED
    if weight is not None:
        flags |= _lib.LORA_MX_NEED_DX
        dx = dy.new_empty((m, k))
        dxp = dx.data_ptr()
        wp, sp, wg, wcode = wc.data_ptr(), weight.scales.data_ptr(), weight.global_scale, weight._code
    stream = _raw_stream(device.index)
    ws = _lib.WORKSPACE.get(_backward_bytes(m, n, k, r, flags), device, "mx_backward", stream)
    rc = _entry("lora_mx_backward")(dyp, lddy, x8.codes.data_ptr(), x8.scales.data_ptr(), z.data_ptr(),
                                    float(z_scale), a.data_ptr(), _ld(a), bp, ldb, wp, sp, wg, wcode,
                                    dxp, k, da.data_ptr(), k, db.data_ptr(), r, m, n, k, r, float(scale), dt,
                                    ws.data_ptr(), ws.numel(), stream)
    if rc:
        _lib.check(rc, "lora_mx_backward")
    return (dx if dx is None or len(shape) == 2 else dx.view(*shape[:-1], k)), da, db


def mx_lora_forward(x: torch.Tensor, weight: MXTensor, bias: torch.Tensor | None, a: torch.Tensor, b: torch.Tensor,
                    scale: float = 1.0, x_global_scale: float = 1.0):
    """The linear with what its backward pass keeps: ``(y, x8, z, z_scale)``.

    ``y`` as ``mx_lora_linear``; ``x8`` the mxfp8 checkpoint of x (half its bytes),
    ``z`` the [M, 2 r16] pair with ``z_scale * (hi + lo) = scale * x @ a.T``.
    """
    if a is None or b is None or a.shape[0] == 0:
        raise ValueError("mx_lora_forward: an adapter (rank >= 1) is required")
    y, z = _linear(x, weight, bias, a, b, scale, x_global_scale, True, "mx_lora_forward")
    z_scale = _entry("lora_mx_linear_z_scale")(float(x_global_scale), weight.global_scale, weight._code)
    return y, mx_quantize(x, "mxfp8"), z, z_scale


class _MXLoRAFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, weight, bias, scale, x_global_scale):
        a, b = a.detach(), b.detach()
        y, x8, z, ctx.z_scale = mx_lora_forward(x, weight, bias, a, b, scale, x_global_scale)
        ctx.save_for_backward(x8.codes, x8.scales, z, a, b)
        ctx.x_shape, ctx.weight, ctx.scale = x8.shape, weight, scale
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return (None,) * 7
        codes, scales, z, a, b = ctx.saved_tensors
        x8 = MXTensor(codes, scales, ctx.x_shape, "mxfp8")
        need_x, need_a, need_b = ctx.needs_input_grad[:3]
        dx, da, db = mx_lora_backward(dy, x8, z, a, b, ctx.scale, ctx.weight if need_x else None, ctx.z_scale)
        return dx, da if need_a else None, db if need_b else None, None, None, None, None


class MXLoRALinear(torch.nn.Module):
    """An ``nn.Linear`` frozen in 4 bits with a trainable LoRA adapter.

    ``y = q(x) @ W.T + bias + scale * (x @ lora_a.T) @ lora_b.T``.  W is quantised
    once (``fmt`` mxfp4 or nvfp4) and frozen; ``lora_a`` [r, K] and ``lora_b`` [N, r]
    are parameters.  While gradients are recorded the input is kept for the backward
    pass in 8 bits (mxfp8) with the [M, r] product, and nothing else of its size;
    without them the call is ``mx_lora_linear``.  ``x_amax``, for nvfp4: the largest
    magnitude expected of the input (its calibration).  ``state_dict`` holds codes, scales,
    both tensor-wide scales and the format; a state of the other format is refused.
    """

    def __init__(self, base: torch.nn.Linear, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0,
                 fmt: str = "mxfp4", x_amax: float = 32.0):
        super().__init__()
        if fmt not in ("mxfp4", "nvfp4"):
            raise ValueError(f"MXLoRALinear: fmt must be mxfp4 or nvfp4, got {fmt!r}")
        if a.shape[1] != base.in_features or b.shape[0] != base.out_features or a.shape[0] != b.shape[1]:
            raise ValueError(
                f"LoRA factors {tuple(a.shape)}/{tuple(b.shape)} do not match "
                f"Linear({base.in_features}, {base.out_features})"
            )
        weight = base.weight.detach()
        self.in_features, self.out_features = base.in_features, base.out_features
        self.scale, self.fmt = float(scale), fmt
        nv = fmt == "nvfp4"
        self.w_global_scale = nvfp4_global_scale(weight.abs().max()) if nv else 1.0
        self.x_global_scale = nvfp4_global_scale(x_amax) if nv else 1.0
        q = mx_quantize(weight, fmt, self.w_global_scale)
        self.register_buffer("w_codes", q.codes)
        self.register_buffer("w_scales", q.scales)
        self.register_buffer("bias", None if base.bias is None else base.bias.detach())
        self.lora_a = torch.nn.Parameter(a.detach().to(weight).contiguous().clone())
        self.lora_b = torch.nn.Parameter(b.detach().to(weight).contiguous().clone())

    # The codes mean nothing without the tensor-wide scales, which stay on the host (a call
    # passes them by value): they travel in the state as one small CPU tensor.
    def get_extra_state(self) -> torch.Tensor:
        return torch.tensor([_FORMATS[self.fmt], self.w_global_scale, self.x_global_scale], dtype=torch.float64)

    def set_extra_state(self, state: torch.Tensor) -> None:
        code, w_global_scale, x_global_scale = state.tolist()
        if code != _FORMATS[self.fmt]:
            names = {v: k for k, v in _FORMATS.items()}
            raise RuntimeError(
                f"MXLoRALinear: the state is of a {names.get(int(code), code)} layer, this one is {self.fmt}")
        self.w_global_scale, self.x_global_scale = w_global_scale, x_global_scale

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        key = prefix + "_extra_state"
        if self.fmt == "mxfp4" and key not in state_dict:  # nothing to restore: both scales are 1
            state_dict = {**state_dict, key: self.get_extra_state()}
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)

    @property
    def rank(self) -> int:
        return self.lora_a.shape[0]

    @property
    def weight(self) -> MXTensor:
        return MXTensor(self.w_codes, self.w_scales, (self.out_features, self.in_features), self.fmt,
                        self.w_global_scale)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"rank={self.rank}, scale={self.scale}, fmt={self.fmt}")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        learns = torch.is_grad_enabled() and (
            x.requires_grad or self.lora_a.requires_grad or self.lora_b.requires_grad)
        if learns:
            return _MXLoRAFunction.apply(x, self.lora_a, self.lora_b, self.weight, self.bias, self.scale,
                                         self.x_global_scale)
        return mx_lora_linear(x, self.weight, self.bias, self.lora_a, self.lora_b, self.scale, self.x_global_scale)
