"""Block-scaled FP8 products: dense, grouped by expert, and the experts' FFN.

Operands are e4m3 codes with fp32 scales in blocks of 128 columns:

* ``a`` [rows, K] with ``a_scale`` [rows, ceil(K / 128)], one scale per 1 x 128
  block: what :func:`kiwi_b200.ops.quant_fp8` returns and what the FP8 dispatch
  delivers;
* ``b`` [N, K] with ``b_scale`` [ceil(N / 128), ceil(K / 128)], one scale per
  128 x 128 block (:func:`quant_fp8_weights`); grouped: [G * N, K] and
  [G * N / 128, ceil(K / 128)], group g's weights in rows g*N .. g*N+N-1.

``out[r, n] = sum over blocks of a_scale * b_scale * (a block . b block)``, summed
in fp32 and rounded once to bf16.  K is a multiple of 16 (a short last block has
a scale of its own), a dense N is any, a grouped N a multiple of 128 (256 with
SwiGLU, whose gate and up rows are interleaved in blocks of 128:
:func:`kiwi_b200.models.moe.interleave_gate_up`).

CUDA tensors run the sm_100a kernel (``kiwi_b200._C.ops.fp8_gemm``: tcgen05 8-bit
MMAs, scales applied in fp32) on the current stream; nothing synchronises, row
counts that are on the device stay there, and such a call can be captured into a
CUDA graph.  The kernel is chosen by the call's sizes, so the order of a row's
fp32 sum, and with it the last bit, can change with the number of rows beside it;
a buffer much larger than the rows in it costs time (8 rows in one of 2048: 74 us
against 53), so pass only as many rows as may be in use.

A result that a call allocates has zeros in the rows past ``sum(counts)``; of an
``out`` that is passed in, those rows are left as they were.  It must not overlap
an input, the counts included.  Counts that are negative or add up to more than
the rows are clamped and reported, like a wait that ran out, by
:func:`check_gemm` (a call without rows reports nothing).  CPU tensors run
:func:`fp8_gemm_reference`, the fp32 restatement.  No gradients: FP8 codes are
not differentiable.
"""
import torch

from ..models import moe as _moe
from .grouped_gemm import _swiglu_tiles

_BLOCK = 128
_FP8 = torch.float8_e4m3fn
_MAX_COLUMNS = 2 ** 31 - 257  # the kernels count blocks of columns in 32 bits
_ops = None


def _native_ops():
    """The native extension's ops, looked up once: a call of a few microseconds pays for every lookup."""
    global _ops
    if _ops is None:
        from .. import native

        _ops = native().ops
    return _ops


def _check_operand(x, s, scale_rows, what):
    if x.dtype != _FP8 or x.dim() != 2:
        raise ValueError(f"{what} must be float8_e4m3fn [rows, K]")
    if x.shape[1] < 16 or x.shape[1] % 16:
        raise ValueError("K must be a positive multiple of 16")
    if x.shape[1] > _MAX_COLUMNS:
        raise ValueError("K must be below 2^31 - 256")
    want = (scale_rows, -(-x.shape[1] // _BLOCK))
    if s.dtype != torch.float32 or tuple(s.shape) != want:
        raise ValueError(f"{what}'s scales must be fp32 {list(want)}")
    if x.device != s.device:
        raise ValueError(f"{what} and its scales must be on one device")


def _check(a, a_scale, b, b_scale, counts, out, swiglu, row_scale):
    """The CPU path's argument checks (the native op makes the same ones)."""
    groups = 1 if counts is None else counts.numel()
    if counts is not None and (counts.dim() != 1 or not 1 <= groups <= 1024):
        raise ValueError("counts must hold 1 to 1024 groups")
    if b.dim() != 2 or b.shape[0] < 1 or b.shape[0] % groups:
        raise ValueError("B must be [groups * N, K]")
    n = b.shape[0] // groups
    if a.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError("A and B must share K")
    if counts is not None and n % _BLOCK:
        raise ValueError("a grouped product needs N to be a multiple of 128")
    _check_operand(a, a_scale, a.shape[0], "A")
    _check_operand(b, b_scale, groups * -(-n // _BLOCK), "B")
    if a.device != b.device:
        raise ValueError("A and B must be on one device")
    if swiglu and n % 256:
        raise ValueError("SwiGLU needs N to be a multiple of 256")
    if row_scale is not None and (row_scale.dtype != torch.float32 or tuple(row_scale.shape) != (a.shape[0],)):
        raise ValueError("row_scale must be fp32 [rows]")
    cols = n // 2 if swiglu else n
    if out is not None and (out.dtype != torch.bfloat16 or tuple(out.shape) != (a.shape[0], cols)):
        raise ValueError(f"out must be bf16 [{a.shape[0]}, {cols}]")


def _as_counts(counts, device):
    """int32 row counts on the rows' device (a host list is copied there).  What
    32 bits cannot hold is saturated to a count that is reported, not wrapped."""
    if torch.is_tensor(counts) and counts.dtype == torch.int32 and counts.device == device:
        return counts
    counts = torch.as_tensor(counts)
    if counts.is_floating_point() and counts.numel():
        raise ValueError("counts must be whole numbers")
    if counts.element_size() > 2 and counts.dtype != torch.int32:
        counts = counts.to(torch.int64).clamp(-1, 2 ** 31 - 1)
    return counts.to(device=device, dtype=torch.int32)


def dequant_fp8(codes, scales, rows_per_scale=1):
    """fp32 values of FP8 codes in blocks of ``rows_per_scale`` x 128 (1 or 128)."""
    s = scales if rows_per_scale == 1 else scales.repeat_interleave(rows_per_scale, 0)[:codes.shape[0]]
    return codes.float() * s.repeat_interleave(_BLOCK, 1)[:, :codes.shape[1]]


def fp8_gemm_reference(a, a_scale, b, b_scale, counts=None, swiglu=False, row_scale=None):
    """fp32 reference of the products; returns fp32 [rows, N or N / 2], zeros past sum(counts)."""
    counts = [a.shape[0]] if counts is None else [int(c) for c in torch.as_tensor(counts).tolist()]
    n = b.shape[0] // len(counts)
    nb = -(-n // _BLOCK)
    af = dequant_fp8(a, a_scale)
    out = torch.zeros(a.shape[0], n // 2 if swiglu else n, device=a.device)
    off = 0
    for g, c in enumerate(counts):
        y = af[off:off + c] @ dequant_fp8(b[g * n:(g + 1) * n], b_scale[g * nb:(g + 1) * nb], _BLOCK).t()
        if swiglu:
            y = _swiglu_tiles(y)
        if row_scale is not None:
            y = y * row_scale[off:off + c, None]
        out[off:off + c] = y
        off += c
    return out


def _checked_sum(counts, rows):
    c = counts.tolist()
    if min(c) < 0 or sum(c) > rows:
        raise ValueError("counts must be non-negative and add up to at most the rows")
    return sum(c)


def fp8_gemm(a, a_scale, b, b_scale, out=None):
    """bf16 [M, N] = a . b^T of block-scaled FP8 operands; see the module docstring."""
    if not a.is_cuda:
        _check(a, a_scale, b, b_scale, None, out, False, None)
        res = fp8_gemm_reference(a, a_scale, b, b_scale).bfloat16()
        return res if out is None else out.copy_(res)
    return _native_ops().fp8_gemm(a, a_scale, b, b_scale, None, out)


def grouped_fp8_gemm(a, a_scale, b, b_scale, counts, out=None, swiglu=False, row_scale=None):
    """The product of each group's rows with its weights, as
    :func:`kiwi_b200.ops.grouped_gemm` on FP8 operands: bf16 [rows, N], or
    [rows, N / 2] with the SwiGLU epilogue, times ``row_scale`` (fp32 [rows])."""
    counts = _as_counts(counts, a.device)
    if not a.is_cuda:
        _check(a, a_scale, b, b_scale, counts, out, swiglu, row_scale)
        total = _checked_sum(counts, a.shape[0])
        res = fp8_gemm_reference(a, a_scale, b, b_scale, counts, swiglu, row_scale).bfloat16()
        if out is None:
            return res
        out[:total] = res[:total]
        return out
    return _native_ops().fp8_gemm(a, a_scale, b, b_scale, counts, out, bool(swiglu), row_scale)


def grouped_fp8_swiglu(a, a_scale, b, b_scale, counts):
    """:func:`grouped_fp8_gemm` with SwiGLU whose rows come back quantised, ready
    for the next product: (codes [rows, N / 2], scales [rows, N / 256]).  The
    fp32 activations are quantised as :func:`kiwi_b200.ops.quant_fp8` does, in
    the product's epilogue; they are never stored."""
    counts = _as_counts(counts, a.device)
    if not a.is_cuda:
        _check(a, a_scale, b, b_scale, counts, None, True, None)
        _checked_sum(counts, a.shape[0])
        return _moe.quant_fp8_codes(fp8_gemm_reference(a, a_scale, b, b_scale, counts, True))
    return _native_ops().fp8_swiglu(a, a_scale, b, b_scale, counts)


def expert_ffn_fp8(x, x_scale, w13, w13_scale, w2, w2_scale, counts, row_scale=None, out=None):
    """The experts' SwiGLU FFN in FP8: ``row_scale * (quant(swiglu(x . w13^T)) . w2^T)``
    for expert-sorted rows ``x`` [rows, H], ``w13`` [E * 2F, H] (gate and up
    interleaved) and ``w2`` [E * H, F]; bf16 [rows, H].  Two launches."""
    return _expert_ffn_fp8(x, x_scale, w13, w13_scale, w2, w2_scale, counts, row_scale, out, None)


def _expert_ffn_fp8(x, x_scale, w13, w13_scale, w2, w2_scale, counts, row_scale, out, error):
    """expert_ffn_fp8 with an error word (int32 [1] on the device) of the caller's own, or None."""
    counts = _as_counts(counts, x.device)
    if not x.is_cuda:
        e = counts.numel()
        if (w13.dim() != 2 or w2.dim() != 2 or w13.shape[0] % (2 * e) or
                tuple(w2.shape) != (e * x.shape[1], w13.shape[0] // (2 * e))):
            raise ValueError("w13 must be [E * 2F, H] and w2 [E * H, F]")
        h, hs = grouped_fp8_swiglu(x, x_scale, w13, w13_scale, counts)
        return grouped_fp8_gemm(h, hs, w2, w2_scale, counts, out, False, row_scale)
    return _native_ops().expert_ffn_fp8(x, x_scale, w13, w13_scale, w2, w2_scale, counts, row_scale, out, error)


def quant_fp8_weights(w):
    """(codes float8_e4m3fn [R, K], fp32 scales [ceil(R / 128), ceil(K / 128)]) of a
    bf16 matrix in 128 x 128 blocks, scale = amax / 448 (1 for an all-zero block;
    2^-128 where 448 / amax would overflow, amax < 1.4e-36).
    Grouped weights [G * N, K] with N a multiple of 128 quantise group by group."""
    if not w.is_cuda:
        if w.dtype != torch.bfloat16 or w.dim() != 2:
            raise ValueError("w must be a bf16 [rows, K] tensor")
        r, c = w.shape
        rb, cb = -(-r // _BLOCK), -(-c // _BLOCK)
        t = torch.zeros(rb * _BLOCK, cb * _BLOCK)
        t[:r, :c] = w.float()
        t = t.view(rb, _BLOCK, cb, _BLOCK).permute(0, 2, 1, 3).reshape(rb * cb, -1)
        codes, scales = _moe.quant_fp8_codes(t, _BLOCK * _BLOCK)
        codes = codes.view(rb, cb, _BLOCK, _BLOCK).permute(0, 2, 1, 3).reshape(rb * _BLOCK, cb * _BLOCK)
        return codes[:r, :c].contiguous(), scales.view(rb, cb)
    return _native_ops().quant_fp8_weights(w)


def check_gemm(device=None):
    """Raises RuntimeError if a product of this module or of
    :mod:`kiwi_b200.ops.grouped_linear` on ``device`` (the current one) reported
    an error since the last check (synchronises the current stream).  There is one
    error word a device for all callers of these functions, and a check clears it
    for all; an :class:`kiwi_b200.ops.ExpertFFN` has its own."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    if dev is None:
        dev = torch.cuda.current_device()
    _raise_error(_native_ops().gemm_error(dev))


def _raise_error(e):
    if e:
        what = [n for b, n in ((1, "a wait ran out"), (2, "counts negative or past the rows")) if e & b]
        raise RuntimeError("expert products: " + " and ".join(what))


__all__ = ["fp8_gemm", "grouped_fp8_gemm", "grouped_fp8_swiglu", "expert_ffn_fp8", "quant_fp8_weights",
           "fp8_gemm_reference", "dequant_fp8", "check_gemm"]
