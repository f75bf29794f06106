"""Matrix products with weights held in 4 bits, a scale for each row and group of columns.

A weight is (code - 8) * scale with a code of 0 .. 15 and a bfloat16 scale, so a matrix takes 4 + 16 / group bits a weight.
`quantize` rounds a matrix once, when a model is loaded; `linear` multiplies by it as `parts.linear.linear` does by a matrix.
The reference engine holds its weights in blocks of 4 bits with a scale each as well (QStream src/quant.c:95-286); the
order of the codes here is the one in which the tensor cores take them.
"""
from __future__ import annotations

import functools
from ctypes import c_int, c_longlong, c_void_p
from operator import attrgetter

import torch

from ..errors import QsError, QStreamError
from . import gemm_tc, ops

GROUPS = (32, 64, 128)
TYPES = (torch.float32, torch.bfloat16)
MAX_COLUMNS = 32768
MAX_ROWS = 65408                    # of a call to the library: what the kernels' grids hold, in whole tiles of 128

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


class Weight4:
    """A matrix [out_features, in_features] in 4 bits.

    codes: uint8 [ceil(out / 16)][ceil(in / 64)][32][16].  Entry 4 g + t of a tile is four little-endian words of eight codes; word
    2 h + u holds row g + 8 u of the tile, columns 32 h + 8 t + (0, 2, 4, 6, 1, 3, 5, 7), lowest four bits first.
    scales: bfloat16 [ceil(out / 16)][groups][8][2], entry (g, u) for row g + 8 u; groups cover the columns rounded up to 64.
    What fills up the last rows and columns are codes of 8 and scales of 0.
    The two tensors are checked once, here, so they stay: their contents may change, another tensor takes another matrix."""
    __slots__ = ("_codes", "_scales", "_n", "_k", "_group")
    codes, scales, out_features, in_features, group = (property(attrgetter(name)) for name in __slots__)

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, out_features: int, in_features: int, group: int):
        n, k, g = self._n, self._k, self._group = out_features, in_features, group
        self._codes, self._scales = codes, scales
        if n < 1 or k < 1 or g not in GROUPS:
            _refuse(f"4-bit weights: a matrix [{n}, {k}] in groups of {g} (groups: {GROUPS})", QsError.QUANT_MISMATCH)
        tiles, chunks = -(-n // 16), -(-k // 64)
        if codes.shape != (tiles, chunks, 32, 16) or codes.dtype is not torch.uint8 or not codes.is_contiguous() \
                or scales.shape != (tiles, -(-chunks * 64 // g), 8, 2) or scales.dtype is not torch.bfloat16 or not scales.is_contiguous():
            _refuse(f"4-bit weights: [{n}, {k}] in groups of {g} are contiguous uint8 codes and bfloat16 scales of {sizes(n, k, g)}, got {codes.dtype} "
                    f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}", QsError.QUANT_MISMATCH)
        if scales.get_device() != codes.get_device() or codes.data_ptr() % 16 or scales.data_ptr() % 4:
            _refuse("4-bit weights: codes and scales lie on one device, the codes on a 16-byte boundary")

    def __reduce__(self):
        return Weight4, (self.codes, self.scales, self.out_features, self.in_features, self.group)

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


def launch_stream(device: int, *tensors) -> int:
    """The stream to launch on, for operands that all lie on the current device (`device`: the first one's index, -1 on the host)."""
    for t in tensors:
        if t is not None and t.get_device() != device:
            _refuse(f"operands on several devices: one on {t.device}, others on {'cuda:%d' % device if device >= 0 else 'the host'}")
    if device < 0:
        _refuse("kernels run on CUDA tensors only; there is no CPU path")
    if device != torch.cuda.current_device():
        _refuse(f"operands on cuda:{device}, but the current device is cuda:{torch.cuda.current_device()}")
    return ops.stream()


def quantize(weight: torch.Tensor, group: int = 64) -> Weight4:
    """Round a float32 or bfloat16 matrix (any row stride) to 4 bits.  Of each row's group, the element m of the largest magnitude sets the
    scale s = bfloat16(-m / 8); a weight w becomes the nearest (ties to even) of the numbers -8 s .. 7 s.  Up to 32,768 columns, as `linear` takes them."""
    if weight.dim() != 2 or weight.stride(1) != 1 or weight.dtype not in TYPES or 0 in weight.shape:
        _refuse(f"4-bit weights: need a float32 or bfloat16 matrix with contiguous rows, got {weight.dtype} {tuple(weight.shape)} strides {weight.stride()}")
    if group not in GROUPS:
        _refuse(f"4-bit weights: groups of {group} columns (groups: {GROUPS})", QsError.QUANT_MISMATCH)
    if weight.shape[1] > MAX_COLUMNS:
        _refuse(f"4-bit weights: a matrix of {weight.shape[1]} columns, the products take {MAX_COLUMNS}", QsError.QUANT_MISMATCH)
    stream = launch_stream(weight.get_device())
    _bind()
    N, K = weight.shape
    shapes = sizes(N, K, group)
    codes = torch.empty(shapes[0], dtype=torch.uint8, device=weight.device)
    scales = torch.zeros(shapes[1], dtype=torch.bfloat16, device=weight.device)
    ops.check(_quantize(ops.ptr(codes), ops.ptr(scales), ops.ptr(weight), ops.dtype_code(weight), weight.stride(0), N, K, group, stream))
    return Weight4(codes, scales, N, K, group)


def linear(x, weight: Weight4, bias=None, activation=None, residuals=(), out_dtype=None, out=None, settled=False) -> torch.Tensor:
    """act(x W^T + bias) + residuals for rows x [M, in_features] of float32 or bfloat16, accumulated in 32 bits.  Arguments and
    result as for `parts.linear.linear`: up to two residuals of x's type; `out_dtype` float32 for a 32-bit result; `out`: a view to
    write into (contiguous rows, any row stride).  `settled`: the weight was complete before the previous kernel of the stream began
    (a model's is); the kernel then fetches it while that kernel still runs.

    Products are exact and summed in 32 bits, but for one limit: more than 16 bfloat16 rows in a large product are taken as 16-bit floats over a power of
    two for each row, and so are the scales of a row of the matrix.  A number is off by 2^-25 of its row's largest at most (bfloat16 numbers down to 2^-17
    of it not at all), a weight by eight times 2^-25 of the largest scale in its row."""
    M, K, ldx = ops._rows(x)
    N, dtype = weight.out_features, x.dtype
    wide = dtype is torch.float32
    if K != weight.in_features:
        _refuse(f"linear: x is [{M}, {K}] but weight is {weight.shape}")
    if not wide and dtype is not torch.bfloat16:
        _refuse(f"linear: rows of {dtype}; 4-bit weights take float32 or bfloat16")
    if K > MAX_COLUMNS:
        _refuse(f"linear: {K} columns, the kernels take {MAX_COLUMNS}")
    act = ops.ACTIVATIONS.get(activation)
    if act is None:
        _refuse(f"linear: activation '{activation}' has no kernel")
    if bias is not None and (bias.shape != (N,) or bias.stride(0) != 1 or bias.dtype not in TYPES):
        _refuse(f"linear: a bias for {N} results, got {bias.dtype} {tuple(bias.shape)}")
    want = out.dtype if out is not None else out_dtype or dtype
    if want not in TYPES or (wide and want is not torch.float32) or (out is not None and out_dtype not in (None, want)):
        _refuse(f"linear: a result of {want} from rows of {dtype}")
    if residuals or out is not None:
        out, res, ldr = ops._product_views(x, M, N, [r for r in residuals if r is not None], want, out)
        r0, r1 = res[:2]
    else:
        out, r0, r1, ldr = torch.empty((M, N), dtype=want, device=x.device), None, None, N
    if M == 0:
        return out
    if M > MAX_ROWS:
        for a in range(0, M, MAX_ROWS):
            part = [None if t is None else t[a:a + MAX_ROWS] for t in (x, out, r0, r1)]
            linear(part[0], weight, bias, activation, part[2:], out=part[1], settled=settled)
        return out
    codes, scales = weight._codes, weight._scales
    stream = launch_stream(codes.get_device(), x, bias, out, r0, r1)
    if _linear is None:
        _bind()
    code, at = (ops.F32, x.data_ptr()) if wide else (ops.BF16, x.data_ptr())
    aligned = int(at % 16 == 0 and ldx % (4 if wide else 8) == 0)
    scratch = None
    if wide or M > 16 or K % 64 or not aligned:             # rows laid out anew; for many rows the operands' powers of two
        nbytes = _scratch(M, N, K, code, aligned)
        if nbytes:
            scratch = torch.empty((nbytes,), dtype=torch.uint8, device=x.device)
            ops.count_launches(_kernels(M, N, K, code, aligned) - 1)
    ops.check(_linear(out.data_ptr(), ops.F32 if want is torch.float32 else ops.BF16, out.stride(0), at, code, ldx, aligned, codes.data_ptr(), scales.data_ptr(),
                      None if bias is None else bias.data_ptr(), 0 if bias is None else ops.dtype_code(bias), act, None if r0 is None else r0.data_ptr(),
                      None if r1 is None else r1.data_ptr(), ldr, M, N, K, weight.group, 1 if settled else 0, None if scratch is None else scratch.data_ptr(),
                      gemm_tc.status_word(x.device).data_ptr(), stream))
    return out
