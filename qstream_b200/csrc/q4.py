"""Matrix products with weights held in 4 bits, a scale for each row and group of columns.

A weight is (code - 8) * scale with a code of 0 .. 15 and a bfloat16 scale, so a matrix takes 4 + 16 / group bits a weight.
`quantize` rounds a matrix once, when a model is loaded; `linear` multiplies by it as `parts.linear.linear` does by a matrix.
The reference engine holds its weights in blocks of 4 bits with a scale each as well (QStream src/quant.c:95-286); the
order of the codes here is the one in which the tensor cores take them.
"""
from __future__ import annotations

import functools
from ctypes import c_int, c_longlong, c_void_p
from dataclasses import dataclass

import torch

from ..errors import QsError, QStreamError
from . import gemm_tc, ops

GROUPS = (32, 64, 128)
TYPES = (torch.float32, torch.bfloat16)
MAX_COLUMNS = 32768

_quantize = _linear = _scratch = _kernels = None


def _bind():
    global _quantize, _linear, _scratch, _kernels
    if _linear is None:
        _quantize = ops.bind("qs_q4_quantize", [c_void_p, c_void_p, c_void_p, c_int, c_longlong, c_int, c_int, c_int, c_void_p])
        _scratch = functools.lru_cache(maxsize=4096)(ops.bind("qs_q4_linear_scratch", [c_int, c_int, c_int, c_int, c_int], c_longlong))
        _kernels = functools.lru_cache(maxsize=4096)(ops.bind("qs_q4_linear_kernels", [c_int, c_int, c_int, c_int, c_int], c_int))
        _linear = ops.bind("qs_q4_linear", [c_void_p, c_int, c_longlong, c_void_p, c_int, c_longlong, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int,
                                            c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p])


def _refuse(text, code=QsError.INVALID_INPUT):
    raise QStreamError(code, text)


@dataclass(frozen=True)
class Weight4:
    """A matrix [out_features, in_features] in 4 bits.

    codes: uint8 [ceil(out / 16)][ceil(in / 64)][32][16].  Entry 4 g + t of a tile is four little-endian words of eight codes; word
    2 h + u holds row g + 8 u of the tile, columns 32 h + 8 t + (0, 2, 4, 6, 1, 3, 5, 7), lowest four bits first.
    scales: bfloat16 [ceil(out / 16)][groups][8][2], entry (g, u) for row g + 8 u; groups cover the columns rounded up to 64.
    What fills up the last rows and columns are codes of 8 and scales of 0."""
    codes: torch.Tensor
    scales: torch.Tensor
    out_features: int
    in_features: int
    group: int

    def __post_init__(self):
        n, k, g = self.out_features, self.in_features, self.group
        if n < 1 or k < 1 or g not in GROUPS:
            _refuse(f"4-bit weights: a matrix [{n}, {k}] in groups of {g} (groups: {GROUPS})", QsError.QUANT_MISMATCH)
        tiles, chunks = -(-n // 16), -(-k // 64)
        want = (tiles, chunks, 32, 16), (tiles, -(-chunks * 64 // g), 8, 2)
        for name, t, shape, dtype in (("codes", self.codes, want[0], torch.uint8), ("scales", self.scales, want[1], torch.bfloat16)):
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
                _refuse(f"4-bit weights: {name} of [{n}, {k}] in groups of {g} are contiguous {dtype} {shape}, got {t.dtype} {tuple(t.shape)}", QsError.QUANT_MISMATCH)
        if self.codes.device != self.scales.device or self.codes.data_ptr() % 16 or self.scales.data_ptr() % 4:
            _refuse("4-bit weights: codes and scales lie on one device, the codes on a 16-byte boundary")

    @property
    def shape(self):
        return (self.out_features, self.in_features)

    @property
    def device(self):
        return self.codes.device

    def numel(self) -> int:
        return self.out_features * self.in_features

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()


def sizes(out_features: int, in_features: int, group: int):
    """Shapes of the codes and the scales of a matrix."""
    tiles, chunks = -(-out_features // 16), -(-in_features // 64)
    return (tiles, chunks, 32, 16), (tiles, -(-chunks * 64 // group), 8, 2)


def _on_current_device(*tensors):
    """All operands on the device whose stream the kernels are launched on."""
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        _refuse(f"operands on several devices: {sorted(map(str, devices))}")
    device = devices.pop()
    if device.type == "cuda" and device.index != torch.cuda.current_device():
        _refuse(f"operands on {device}, but the current device is cuda:{torch.cuda.current_device()}")


def quantize(weight: torch.Tensor, group: int = 64) -> Weight4:
    """Round a float32 or bfloat16 matrix (any row stride) to 4 bits.  Of each row's group, the element m of the largest magnitude sets the
    scale s = bfloat16(-m / 8); a weight w becomes the nearest (ties to even) of the numbers -8 s .. 7 s."""
    if weight.dim() != 2 or weight.stride(1) != 1 or weight.dtype not in TYPES or 0 in weight.shape:
        _refuse(f"4-bit weights: need a float32 or bfloat16 matrix with contiguous rows, got {weight.dtype} {tuple(weight.shape)} strides {weight.stride()}")
    if group not in GROUPS:
        _refuse(f"4-bit weights: groups of {group} columns (groups: {GROUPS})", QsError.QUANT_MISMATCH)
    ops.ptr(weight)
    _on_current_device(weight)
    _bind()
    N, K = weight.shape
    shapes = sizes(N, K, group)
    codes = torch.empty(shapes[0], dtype=torch.uint8, device=weight.device)
    scales = torch.zeros(shapes[1], dtype=torch.bfloat16, device=weight.device)
    ops.check(_quantize(ops.ptr(codes), ops.ptr(scales), ops.ptr(weight), ops.dtype_code(weight), weight.stride(0), N, K, group, ops.stream()))
    return Weight4(codes, scales, N, K, group)


def linear(x, weight: Weight4, bias=None, activation=None, residuals=(), out_dtype=None, out=None, settled=False) -> torch.Tensor:
    """act(x W^T + bias) + residuals for rows x [M, in_features] of float32 or bfloat16, accumulated in 32 bits.  Arguments and
    result as for `parts.linear.linear`: up to two residuals of x's type; `out_dtype` float32 for a 32-bit result; `out`: a view to
    write into (contiguous rows, any row stride).  `settled`: the weight was complete before the previous kernel of the stream began
    (a model's is); the kernel then fetches it while that kernel still runs."""
    M, K, ldx = ops._rows(x)
    N = weight.out_features
    if K != weight.in_features:
        _refuse(f"linear: x is [{M}, {K}] but weight is {weight.shape}")
    if x.dtype not in TYPES:
        _refuse(f"linear: rows of {x.dtype}; 4-bit weights take float32 or bfloat16")
    if activation not in ops.ACTIVATIONS:
        _refuse(f"linear: activation '{activation}' has no kernel")
    if bias is not None and (bias.dim() != 1 or bias.numel() != N or bias.stride(0) != 1 or bias.dtype not in TYPES):
        _refuse(f"linear: a bias for {N} results, got {bias.dtype} {tuple(bias.shape)}")
    want = out.dtype if out is not None else out_dtype or x.dtype
    if want not in ((torch.float32,) if x.dtype == torch.float32 else TYPES) or (out is not None and out_dtype not in (None, out.dtype)):
        _refuse(f"linear: a result of {want} from rows of {x.dtype}")
    if K > MAX_COLUMNS:
        _refuse(f"linear: {K} columns, the kernels take {MAX_COLUMNS}")
    out, res, ldr = ops._product_views(x, M, N, [r for r in residuals if r is not None], want, out)
    if M == 0:
        return out
    _on_current_device(x, weight.codes, bias, out, *res[:2])
    _bind()
    code, element = ops.dtype_code(x), x.element_size()
    aligned = x.data_ptr() % 16 == 0 and ldx * element % 16 == 0
    nbytes = _scratch(M, N, K, code, int(aligned))          # rows laid out anew, for many rows the operands' powers of two
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes else None
    if nbytes:
        ops.count_launches(_kernels(M, N, K, code, int(aligned)) - 1)
    ops.check(_linear(ops.ptr(out), ops.dtype_code(out), out.stride(0), ops.ptr(x), code, ldx, int(aligned), ops.ptr(weight.codes), ops.ptr(weight.scales),
                      ops.ptr(bias), ops.dtype_code(bias) if bias is not None else 0, ops.ACTIVATIONS[activation], ops.ptr(res[0]), ops.ptr(res[1]), ldr,
                      M, N, K, weight.group, int(bool(settled)), ops.ptr(scratch),
                      ops.ptr(gemm_tc.status_word(x.device)), ops.stream()))
    return out
