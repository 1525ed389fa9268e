"""Linear layers in 8 bits: e4m3 codes with a scale per block of 128 (gfx950).

A row of a hidden state is e4m3 codes (``torch.float8_e4m3fn``) with an fp32
scale per 128 channels, a weight codes with a scale per 128 x 128: a code stands
for code * scale.  Rows of codes are as long as whole blocks, zeros behind the
last channel, so ``codes`` is [M, ceil(K / 128) * 128].

  * ``rms_norm_quant``: the residual's addition, RMS norm and the codes of the
    normed rows in one launch; ``quantize_rows`` the codes alone (an attention's
    output on its way into the o-projection).
  * ``quantize_weight``: a weight, once, when it is loaded.
  * ``linear``: rows times weight, with a residual added on the way out where
    there is one, for any number of rows (``decode_step.decode_linear`` is the
    bf16 counterpart, for at most 16).
  * ``gated_linear``: both projections of a gated feed-forward block, silu(gate)
    * up, and the result as codes and scales for the down projection.

The scale of a block is its largest magnitude / 448 (the largest e4m3 value) and
not below 2^-100; the code is value / scale rounded to nearest even.  A block
that holds an infinity or a NaN has a NaN scale and NaN codes.  Sums, norms and
activations are fp32, and nothing is rounded to 16 bits between the codes of the
inputs and the one rounding of the result.  (The product of a row's and a
weight's scale is formed first: it should stay within fp32's range.)

Each function checks its arguments on every call; the ``*Plan`` classes check
once for fixed buffers and then make one C-ABI call per ``run()``.

The reference's projections are bf16 (Z/model_hub/qwen.py:439-604).
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from ._lib import check, device_stream, lib, packed_args, ptr, require_gpu
from .paged import _launch, _nothing, _Plan, _same_device, _strides

BLOCK = 128
MAX_K = 16384          # of a product (what the choice of kernels and the bounds on errors are measured for)
MAX_NORM_K = 65536     # of a normed row
E4M3 = torch.float8_e4m3fn
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class _PackedPlan(_Plan):
    """A plan whose arguments are packed once: a run passes their address and the
    stream (17 arguments converted per run took 1.3 us more)."""

    def __init__(self, name: str, rows: torch.Tensor, args, result, keep):
        packed = packed_args(name, args)
        super().__init__(getattr(lib(), name + "_call") if rows.shape[0] else _nothing, rows.device,
                         (ctypes.addressof(packed),), result, (packed, *keep))
        self._index, self._at = rows.device.index, ctypes.addressof(packed)

    def run(self):
        if torch.cuda.current_device() == self._index:
            rc = self._fn(self._at, device_stream(self._device))
            if rc:
                check(rc)
        else:
            _launch(self._fn, self._device, self._args)
        return self.out


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def _check_type(name: str, dtype: torch.dtype) -> int:
    if dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32; got {dtype}")
    return _TYPES[dtype]


def _row_stride(name: str, t: torch.Tensor, shape: tuple) -> int:
    """The row stride of a 2-D tensor with contiguous rows that do not overlap
    (0 where there is one row)."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}; got {list(t.shape)}")
    ld, one = _strides(t)
    if (shape[1] > 1 and one != 1) or (shape[0] > 1 and ld < shape[1]):
        raise ValueError(f"the rows of {name} must be contiguous and apart; got strides {t.stride()}")
    return ld if shape[0] > 1 else shape[1]


def _check_codes(name: str, codes: torch.Tensor, rows: int, K: int, align: int) -> int:
    if codes.dtype != E4M3:
        raise TypeError(f"{name} must be float8_e4m3fn; got {codes.dtype}")
    ld = _row_stride(name, codes, (rows, blocks(K) * BLOCK))
    if codes.data_ptr() % align or ld % align:
        raise ValueError(f"the rows of {name} must start on {align} bytes")
    return ld


def _check_scales(name: str, scales: torch.Tensor, rows: int, K: int, apart: bool) -> tuple[int, int]:
    if scales.dtype != torch.float32 or tuple(scales.shape) != (rows, blocks(K)):
        raise ValueError(f"{name} must be float32 [{rows}, {blocks(K)}]; got {scales.dtype} {list(scales.shape)}")
    s = _strides(scales)
    if apart and scales.numel() > 1:
        # two of them share a place if i rows and j blocks are as far apart for some i, j
        # in the shape, the least of which are the other's stride over the common divisor
        common = math.gcd(*s)
        if common < 1 or s[1] // common < rows and s[0] // common < blocks(K):
            raise ValueError(f"{name} must have a place for every scale; got strides {scales.stride()}")
    return s


def _new_codes(rows: int, K: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(rows, blocks(K) * BLOCK, dtype=E4M3, device=like.device)


def _new_scales(rows: int, K: int, like: torch.Tensor) -> torch.Tensor:
    """Scales as columns of `rows` (neighbouring rows' scales of one block lie
    together, as a product reads them)."""
    return torch.empty(blocks(K), rows, dtype=torch.float32, device=like.device).t()


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """The bytes that a tensor's elements lie in."""
    if not t.numel():
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _runs(t: torch.Tensor) -> tuple[int, int, int]:
    """A contiguous or 2-D tensor as runs of bytes of one length: (the length, how
    many, the bytes from one to the next).  Where no dim is contiguous, a run spans
    what lies between its elements too."""
    size = t.element_size()
    if t.is_contiguous():
        return t.numel() * size, 1, 1
    (inner, n), (outer, count) = sorted((s, n) if n > 1 else (0, 1) for s, n in zip(t.stride(), t.shape))
    length = (inner * (n - 1) + 1) * size
    if outer * size > length:
        return length, count, outer * size
    return length + outer * (count - 1) * size, 1, 1


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share memory.  Runs that lie equally far apart (columns of
    one buffer) and one run among others are told apart; else by the extents."""
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if a0 >= b1 or b0 >= a1:
        return False
    (a_len, a_n, a_step), (b_len, b_n, b_step) = _runs(a), _runs(b)
    if a_n > 1 and b_n > 1 and a_step != b_step:
        return True
    # run j of b lies over run i of a where -b_len < b0 - a0 + (j - i) step < a_len
    step, apart = a_step if a_n > 1 else b_step, b0 - a0
    least, most = (-b_len - apart) // step + 1, -((apart - a_len) // step) - 1
    return max(least, 1 - a_n) <= min(most, b_n - 1)


def _check_apart(name: str, out: torch.Tensor, *others) -> None:
    """`out` is written while other workgroups still read the inputs."""
    for t in others:
        if t is not None and _overlap(out, t):
            raise ValueError(f"{name} must lie apart from the inputs and the other outputs")


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
def _rows_args(x, weight, eps, residual, sum_out, codes, scales):
    kind = _check_type("x", x.dtype)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [rows, channels]; got {list(x.shape)}")
    M, K = x.shape
    if M >= 1 << 27 or K >= 1 << 30:
        raise ValueError(f"{M} rows of {K} channels in one call")
    x_ld = _row_stride("x", x, (M, K))
    res_ld = sum_ld = 0
    if weight is not None:
        if weight.dtype != x.dtype or tuple(weight.shape) != (K,) or (K > 1 and weight.stride(0) != 1):
            raise ValueError(f"the norm's weight must be contiguous {x.dtype} [{K}]; got {weight.dtype} "
                             f"{list(weight.shape)}")
        if K > MAX_NORM_K:
            raise ValueError(f"normed rows have at most {MAX_NORM_K} channels; got {K}")
    if residual is not None:
        if residual.dtype != x.dtype:
            raise TypeError(f"the residual must be {x.dtype}; got {residual.dtype}")
        res_ld = _row_stride("residual", residual, (M, K))
        sum_out = torch.empty(M, K, dtype=x.dtype, device=x.device) if sum_out is None else sum_out
        if sum_out.dtype != x.dtype:
            raise TypeError(f"sum_out must be {x.dtype}; got {sum_out.dtype}")
        sum_ld = _row_stride("sum_out", sum_out, (M, K))
        for name, t in (("x", x), ("residual", residual)):
            if sum_out.data_ptr() != t.data_ptr() and _overlap(sum_out, t) or \
                    sum_out.data_ptr() == t.data_ptr() and _strides(sum_out) != _strides(t):
                raise ValueError(f"sum_out must be {name} itself or lie apart from it")
    elif sum_out is not None:
        raise ValueError("sum_out goes with a residual")
    codes = _new_codes(M, K, x) if codes is None else codes
    scales = _new_scales(M, K, x) if scales is None else scales
    codes_ld = _check_codes("codes", codes, M, K, 8)
    s_m, s_b = _check_scales("scales", scales, M, K, apart=True)
    _same_device(x, weight=weight, residual=residual, sum_out=sum_out, codes=codes, scales=scales)
    for name, t in (("codes", codes), ("scales", scales)):
        _check_apart(name, t, x, weight, residual, sum_out)
    _check_apart("scales", scales, codes)
    if sum_out is not None:
        _check_apart("sum_out", sum_out, weight)
    require_gpu(x)
    args = (ptr(x), x_ld, M, K, kind, ptr(weight), float(eps), ptr(residual), res_ld, ptr(sum_out), sum_ld,
            ptr(codes), codes_ld, ptr(scales), s_m, s_b)
    result = (codes, scales) if residual is None else (codes, scales, sum_out)
    return args, result, (x, weight, residual, sum_out, codes, scales)


class RmsNormQuantPlan(_PackedPlan):
    """``rms_norm_quant`` with its checks done once for fixed buffers."""

    def __init__(self, x, weight, eps, residual=None, sum_out=None, codes=None, scales=None):
        if weight is None:
            raise ValueError("the norm needs its weight")
        args, result, keep = _rows_args(x, weight, eps, residual, sum_out, codes, scales)
        super().__init__("zkv_fp8_rows", x, args, result, keep)


class QuantizeRowsPlan(_PackedPlan):
    """``quantize_rows`` with its checks done once for fixed buffers."""

    def __init__(self, x, codes=None, scales=None):
        args, result, keep = _rows_args(x, None, 0.0, None, None, codes, scales)
        super().__init__("zkv_fp8_rows", x, args, result, keep)


def _fresh_rows(x, weight, eps, residual):
    """The call over contiguous inputs, with outputs of its own: what _rows_args
    checks in fewer steps, or None where it has to be asked (which names what is
    wrong)."""
    kind = _TYPES.get(x.dtype)
    if kind is None or x.dim() != 2 or not x.is_contiguous() or not x.is_cuda:
        return None
    M, K = shape = x.shape
    device = x.device
    if not 0 < M < 1 << 27 or not 0 < K <= MAX_NORM_K:
        return None
    if weight is not None and (weight.dtype != x.dtype or weight.shape != shape[1:] or not weight.is_contiguous() or
                               weight.device != device):
        return None
    total = None
    if residual is not None:
        if residual.dtype != x.dtype or residual.shape != shape or not residual.is_contiguous() or \
                residual.device != device:
            return None
        total = torch.empty(shape, dtype=x.dtype, device=device)
    kb = -(-K // BLOCK)
    codes = torch.empty((M, kb * BLOCK), dtype=E4M3, device=device)
    scales = torch.empty_strided((M, kb), (1, M), dtype=torch.float32, device=device)
    _launch(lib().zkv_fp8_rows, device,
            (x.data_ptr(), K, M, K, kind, None if weight is None else weight.data_ptr(), float(eps),
             None if total is None else residual.data_ptr(), K, None if total is None else total.data_ptr(), K,
             codes.data_ptr(), kb * BLOCK, scales.data_ptr(), 1, M))
    return (codes, scales) if total is None else (codes, scales, total)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
                   sum_out: torch.Tensor | None = None, codes: torch.Tensor | None = None,
                   scales: torch.Tensor | None = None):
    """h = x [+ residual]; h * rsqrt(mean(h^2) + eps) * weight per row of x [M,
    K] (bf16, fp16 or fp32; residual and weight [K] alike), as codes [M,
    ceil(K / 128) * 128] and scales float32 [M, ceil(K / 128)].

    fp32 throughout; the norm goes by the unrounded sum, which is rounded to x's
    type where it is stored.  Returns (codes, scales), and with a residual (codes,
    scales, sum_out); sum_out may be x or residual.  New scales are laid out as
    columns of M."""
    if sum_out is None and codes is None and scales is None and weight is not None:
        got = _fresh_rows(x, weight, eps, residual)
        if got is not None:
            return got
    return RmsNormQuantPlan(x, weight, eps, residual, sum_out, codes, scales).run()


def quantize_rows(x: torch.Tensor, codes: torch.Tensor | None = None, scales: torch.Tensor | None = None):
    """The rows of x [M, K] (bf16, fp16 or fp32) as codes [M, ceil(K / 128) *
    128] and scales float32 [M, ceil(K / 128)]."""
    if codes is None and scales is None:
        got = _fresh_rows(x, None, 0.0, None)
        if got is not None:
            return got
    return QuantizeRowsPlan(x, codes, scales).run()


# ---------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------
@dataclass
class Fp8Weight:
    """A weight of codes [rows, ceil(K / 128) * 128] (zeros behind K) and scales
    float32 [blocks of rows, ceil(K / 128)], contiguous.  parts: the rows are
    that many matrices, one behind the other, with blocks of their own (a gate /
    up weight has 2)."""

    codes: torch.Tensor
    scales: torch.Tensor
    parts: int = 1

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    def dequantize(self) -> torch.Tensor:
        """float32 [rows, ceil(K / 128) * 128]."""
        n = self.rows // self.parts
        s = self.scales.view(self.parts, blocks(n), -1).repeat_interleave(BLOCK, 1)[:, :n].reshape(self.rows, -1, 1)
        return (self.codes.float().view(self.rows, -1, BLOCK) * s).view(self.rows, -1)


def quantize_weight(w: torch.Tensor, parts: int = 1) -> Fp8Weight:
    """A weight [rows, K] (bf16, fp16 or fp32; the rows of `parts` matrices of
    one size) as codes with a scale per 128 x 128."""
    kind = _check_type("w", w.dtype)
    parts = int(parts)
    if w.dim() != 2 or min(w.shape) < 1 or parts < 1 or w.shape[0] % parts:
        raise ValueError(f"w must be [rows, channels], rows a multiple of {parts}; got {list(w.shape)}")
    N, K = w.shape
    nb = parts * blocks(N // parts)
    if nb > 65535 or K >= 1 << 30:
        raise ValueError(f"a weight of {N} x {K} in one call")
    ld = _row_stride("w", w, (N, K))
    require_gpu(w)
    codes = _new_codes(N, K, w)
    scales = torch.empty(nb, blocks(K), dtype=torch.float32, device=w.device)
    _launch(lib().zkv_fp8_weight, w.device, (ptr(w), ld, N, K, kind, parts, ptr(codes), codes.shape[1], ptr(scales)))
    return Fp8Weight(codes, scales, parts)


def _check_product(codes, scales, weight: Fp8Weight, parts: int):
    """(M, rows of a part of the weight, K, the operands' arguments)."""
    if codes.dim() != 2 or weight.codes.dim() != 2 or codes.shape[1] != weight.codes.shape[1] or \
            codes.shape[1] % BLOCK or not codes.shape[1]:
        raise ValueError(f"codes and weight must have one length, a multiple of {BLOCK}; got {list(codes.shape)}, "
                         f"{list(weight.codes.shape)}")
    if weight.parts != parts:
        raise ValueError(f"a weight in {weight.parts} part(s), not {parts}")
    M, K = codes.shape
    rows = weight.rows
    if K > MAX_K:
        raise ValueError(f"a product over {K} channels, at most {MAX_K}")
    if rows < parts or rows % parts or rows >= parts << 22 or M >= 1 << 20 or M * (rows // parts) > 1 << 37:
        raise ValueError(f"a product of {M} rows with a weight of {rows} rows in {parts} part(s)")
    x_ld = _check_codes("codes", codes, M, K, 16)
    if max(x_ld, weight.codes.stride(0)) >= 1 << 23:
        raise ValueError("rows of codes must lie less than 8 MiB apart")
    s_m, s_b = _check_scales("scales", scales, M, K, apart=False)
    w_ld = _check_codes("the weight's codes", weight.codes, rows, K, 16)
    nb = parts * blocks(rows // parts)
    ws = weight.scales
    if ws.dtype != torch.float32 or tuple(ws.shape) != (nb, K // BLOCK) or not ws.is_contiguous():
        raise ValueError(f"the weight's scales must be contiguous float32 [{nb}, {K // BLOCK}]; got {ws.dtype} "
                         f"{list(ws.shape)}")
    _same_device(codes, scales=scales, weight=weight.codes, weight_scales=ws)
    n = rows // parts
    return M, n, K, (ptr(codes), x_ld, ptr(scales), s_m, s_b, ptr(weight.codes), w_ld, ptr(ws), M, n, K)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _workspace(need: int, given: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    """The workspace of a call, whose content does not matter: of its own unless
    one is given (so calls on other streams, and graphs, never share one)."""
    ws = torch.empty(need, dtype=torch.uint8, device=like.device) if given is None else given
    if ws.dtype != torch.uint8 or ws.numel() < need or not ws.is_contiguous() or (need and ws.data_ptr() % 16):
        raise ValueError(f"workspace must be contiguous uint8 of at least {need} bytes on 16 bytes")
    _same_device(like, workspace=ws)
    return ws


def _linear_args(codes, scales, weight, out, out_dtype, residual, workspace):
    M, N, K, operands = _check_product(codes, scales, weight, 1)
    if out is None:
        _check_type("out_dtype", out_dtype)
        out = torch.empty(M, N, dtype=out_dtype, device=codes.device)
    kind = _check_type("out", out.dtype)
    out_ld = _row_stride("out", out, (M, N))
    res_ld = 0
    if residual is not None:
        if residual.dtype != out.dtype:
            raise TypeError(f"the residual must be {out.dtype}; got {residual.dtype}")
        res_ld = _row_stride("residual", residual, (M, N))
        if out.data_ptr() != residual.data_ptr() and _overlap(out, residual) or \
                out.data_ptr() == residual.data_ptr() and _strides(out) != _strides(residual):
            raise ValueError("out must be the residual itself or lie apart from it")
    _same_device(codes, out=out, residual=residual)
    inputs = codes, scales, weight.codes, weight.scales
    _check_apart("out", out, *inputs)
    ws = _workspace(lib().zkv_fp8_linear_workspace_size(M, N, K), workspace, codes)
    _check_apart("workspace", ws, *inputs, residual, out)
    require_gpu(codes)
    args = (*operands, ptr(residual), res_ld, ptr(out), out_ld, kind, ptr(ws), ws.numel())
    return args, out, (codes, scales, weight.codes, weight.scales, residual, out, ws)


class LinearPlan(_PackedPlan):
    """``linear`` with its checks done once for fixed buffers.  A plan has a
    workspace of its own unless one is given; runs of one plan must not overlap on
    the device."""

    def __init__(self, codes, scales, weight, out=None, out_dtype=torch.bfloat16, residual=None, workspace=None):
        args, result, keep = _linear_args(codes, scales, weight, out, out_dtype, residual, workspace)
        super().__init__("zkv_fp8_linear", codes, args, result, keep)


def _fresh_operands(codes, scales, weight: Fp8Weight, parts: int):
    """_check_product of contiguous operands in fewer steps, or None where it has
    to be asked."""
    w, ws = weight.codes, weight.scales
    if codes.dtype != E4M3 or w.dtype != E4M3 or codes.dim() != 2 or w.dim() != 2 or weight.parts != parts or \
            not codes.is_contiguous() or not w.is_contiguous() or not codes.is_cuda:
        return None
    (M, K), (rows, wide), device = codes.shape, w.shape, codes.device
    if wide != K or K % BLOCK or not 0 < K <= MAX_K or not 0 < M < 1 << 20 or not parts <= rows < parts << 22 or \
            rows % parts or M * rows > 1 << 37:
        return None
    n, kb = rows // parts, K // BLOCK
    if scales.dtype != torch.float32 or scales.shape != (M, kb) or ws.dtype != torch.float32 or \
            ws.shape != (parts * -(-n // BLOCK), kb) or not ws.is_contiguous():
        return None
    if scales.device != device or w.device != device or ws.device != device:
        return None
    x_ptr, w_ptr = codes.data_ptr(), w.data_ptr()
    if (x_ptr | w_ptr) % 16:
        return None
    s_m, s_b = scales.stride()
    return M, n, K, (x_ptr, K, scales.data_ptr(), s_m, s_b, w_ptr, K, ws.data_ptr(), M, n, K)


def _fresh_linear(codes, scales, weight, out_dtype, residual):
    """The call over contiguous inputs, with an output of its own; None where
    _linear_args has to be asked."""
    operands, kind = _fresh_operands(codes, scales, weight, 1), _TYPES.get(out_dtype)
    if operands is None or kind is None:
        return None
    M, N, K, args = operands
    if residual is not None and (residual.dtype != out_dtype or residual.shape != (M, N) or
                                 not residual.is_contiguous() or residual.device != codes.device):
        return None
    device = codes.device
    out = torch.empty((M, N), dtype=out_dtype, device=device)
    L = lib()
    need = L.zkv_fp8_linear_workspace_size(M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _launch(L.zkv_fp8_linear, device,
            (*args, None if residual is None else residual.data_ptr(), N, out.data_ptr(), N, kind,
             None if ws is None else ws.data_ptr(), need))
    return out


def _fresh_gated(codes, scales, weight):
    operands = _fresh_operands(codes, scales, weight, 2)
    if operands is None:
        return None
    M, F, K, args = operands
    device, nb = codes.device, -(-F // BLOCK)
    out_codes = torch.empty((M, nb * BLOCK), dtype=E4M3, device=device)
    out_scales = torch.empty_strided((M, nb), (1, M), dtype=torch.float32, device=device)
    L = lib()
    need = L.zkv_fp8_gated_workspace_size(M, F, K)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _launch(L.zkv_fp8_gated_linear, device,
            (*args, out_codes.data_ptr(), nb * BLOCK, out_scales.data_ptr(), 1, M,
             None if ws is None else ws.data_ptr(), need))
    return out_codes, out_scales


def linear(codes: torch.Tensor, scales: torch.Tensor, weight: Fp8Weight, out: torch.Tensor | None = None,
           out_dtype: torch.dtype = torch.bfloat16, residual: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Rows (codes [M, K], scales float32 [M, K / 128] of any strides) times
    weight.T [+ residual]: [M, rows of the weight] in bf16, fp16 or fp32, rounded
    once.  out may be the residual.  The workspace (uint8,
    zkv_fp8_linear_workspace_size(M, N, K) bytes: where few tiles meet a long K)
    needs no clearing; calls that overlap on one race."""
    if out is None and workspace is None:
        got = _fresh_linear(codes, scales, weight, out_dtype, residual)
        if got is not None:
            return got
    return LinearPlan(codes, scales, weight, out, out_dtype, residual, workspace).run()


def _gated_args(codes, scales, weight, out_codes, out_scales, workspace):
    M, F, K, operands = _check_product(codes, scales, weight, 2)
    out_codes = _new_codes(M, F, codes) if out_codes is None else out_codes
    out_scales = _new_scales(M, F, codes) if out_scales is None else out_scales
    codes_ld = _check_codes("out_codes", out_codes, M, F, 8)
    s_m, s_b = _check_scales("out_scales", out_scales, M, F, apart=True)
    inputs = codes, scales, weight.codes, weight.scales
    _check_apart("out_codes", out_codes, *inputs)
    _check_apart("out_scales", out_scales, *inputs, out_codes)
    _same_device(codes, out_codes=out_codes, out_scales=out_scales)
    ws = _workspace(lib().zkv_fp8_gated_workspace_size(M, F, K), workspace, codes)
    _check_apart("workspace", ws, *inputs, out_codes, out_scales)
    require_gpu(codes)
    args = (*operands, ptr(out_codes), codes_ld, ptr(out_scales), s_m, s_b, ptr(ws), ws.numel())
    return args, (out_codes, out_scales), (codes, scales, weight.codes, weight.scales, out_codes, out_scales, ws)


class GatedLinearPlan(_PackedPlan):
    """``gated_linear`` with its checks done once for fixed buffers.  A plan has
    a workspace of its own unless one is given; runs of one plan must not overlap
    on the device."""

    def __init__(self, codes, scales, weight, out_codes=None, out_scales=None, workspace=None):
        args, result, keep = _gated_args(codes, scales, weight, out_codes, out_scales, workspace)
        super().__init__("zkv_fp8_gated_linear", codes, args, result, keep)


def gated_linear(codes: torch.Tensor, scales: torch.Tensor, weight: Fp8Weight, out_codes: torch.Tensor | None = None,
                 out_scales: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """silu(gate) * up of a gated feed-forward block: gate and up are the rows
    (codes, scales) times the two parts of the weight ([2 F, K], parts = 2); returns
    codes [M, ceil(F / 128) * 128] and scales float32 [M, ceil(F / 128)] (new ones as
    columns of M), what ``linear`` takes for the down projection.  The workspace
    (uint8, zkv_fp8_gated_workspace_size(M, F, K) bytes) needs no clearing; calls
    that overlap on one race."""
    if out_codes is None and out_scales is None and workspace is None:
        got = _fresh_gated(codes, scales, weight)
        if got is not None:
            return got
    return GatedLinearPlan(codes, scales, weight, out_codes, out_scales, workspace).run()
