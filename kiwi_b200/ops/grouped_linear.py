"""The experts' bf16 product with its gradients, SwiGLU, and the FFN for training.

``grouped_linear(x, w, counts)`` multiplies each group's consecutive rows of
``x`` [rows, K] with that group's weights (``w`` [G * N, K], group g's in rows
g*N .. g*N+N-1) into bf16 [rows, N]; ``counts`` [G] are the groups' row counts,
on the device for CUDA tensors.  It is differentiable in ``x`` and ``w``:

    dx[rows of g] = dy[rows of g] @ w[g]          (:func:`grouped_linear_dgrad`)
    dw[g]         = dy[rows of g].T @ x[rows of g] (:func:`grouped_linear_wgrad`)

both also callable by themselves; the second writes bf16 or fp32 and can add to
what its ``out`` holds (gradients kept over several micro-batches).  N and K are
multiples of 64.  Sums are fp32, each result is rounded once, and no result
depends on the order in which anything ran.  Rows past ``sum(counts)`` are zero
in a result that the call allocates, left as they were in an ``out`` that is
passed in, and never read; a group without rows has a zero ``dw`` (with
``accumulate``: an unchanged one).

``swiglu(y, row_scale)`` is ``row_scale * silu(gate) * up`` of rows laid out in
blocks of 128 gate and 128 up columns, differentiable in ``y`` and
``row_scale``.  A routing weight applied here is the same as one applied to the
second product's rows, and its gradient needs no product.  ``expert_ffn`` is the
three together: the experts' FFN for training.  On CUDA tensors the sigmoid is
made of the approximate exponential and reciprocal, which stay far below a bf16
rounding; the fp32 gradient of ``row_scale`` is off by up to 0.30 steps of 2^-23 of
the sum of its terms' magnitudes, with exact functions by 0.24.

CUDA tensors run the sm_100a kernels on the current stream: nothing
synchronises, and the calls can be captured into a CUDA graph (a captured
backward needs, as in any PyTorch program, a warm-up on the capturing stream and
leaves that no live eager graph still accumulates into).  Counts that are
negative or add up to more than the rows are clamped and reported by
:func:`kiwi_b200.ops.check_gemm` (a call without rows reports nothing).  CPU
tensors run the same sums in fp32.  Gradients are once differentiable.
"""
import torch

from .fp8_gemm import _MAX_COLUMNS, _as_counts, _checked_sum, _native_ops
from .grouped_gemm import grouped_gemm_reference


def _check(x, w_rows, w_cols, groups, what):
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise ValueError(f"{what} must be bf16 [rows, columns]")
    n = w_rows // groups
    if n < 64 or n % 64 or w_cols < 64 or w_cols % 64:
        raise ValueError("N and K must be multiples of 64")
    if w_cols > _MAX_COLUMNS:
        raise ValueError("K must be below 2^31 - 256")


def _check_counts(counts):
    if counts.dim() != 1 or not 1 <= counts.numel() <= 1024:
        raise ValueError("counts must hold 1 to 1024 groups")


def _check_out(out, shape, types):
    if out is not None and (tuple(out.shape) != tuple(shape) or out.dtype not in types):
        raise ValueError(f"out must be {list(shape)} of {' or '.join(str(t) for t in types)}")


def _fill(out, res, total):
    """`res`, or `out` with its first `total` rows set."""
    if out is None:
        return res
    out[:total] = res[:total]
    return out


def _forward(x, w, counts, out=None):
    _check_counts(counts)
    if w.dtype != torch.bfloat16 or w.dim() != 2 or w.shape[1] != x.shape[-1] or w.shape[0] % counts.numel():
        raise ValueError("w must be bf16 [groups * N, K] with x's K")
    _check(x, w.shape[0], w.shape[1], counts.numel(), "x")
    _check_out(out, (x.shape[0], w.shape[0] // counts.numel()), (torch.bfloat16,))
    total = _checked_sum(counts, x.shape[0])
    res = torch.zeros(x.shape[0], w.shape[0] // counts.numel(), dtype=torch.bfloat16)
    res[:total] = grouped_gemm_reference(x[:total], w, counts).bfloat16()
    return _fill(out, res, total)


def grouped_linear_dgrad(dy, w, counts, out=None):
    """dx [rows, K] of :func:`grouped_linear` for dy [rows, N]."""
    counts = _as_counts(counts, dy.device)
    if dy.is_cuda:
        return _native_ops().grouped_linear_dgrad(dy, w, counts, out)
    _check_counts(counts)
    if w.dtype != torch.bfloat16 or w.dim() != 2 or w.shape[0] != counts.numel() * dy.shape[-1]:
        raise ValueError("w must be bf16 [groups * N, K] with dy's N")
    _check(dy, w.shape[0], w.shape[1], counts.numel(), "dy")
    _check_out(out, (dy.shape[0], w.shape[1]), (torch.bfloat16,))
    total = _checked_sum(counts, dy.shape[0])
    n = dy.shape[1]
    res = torch.zeros(dy.shape[0], w.shape[1], dtype=torch.bfloat16)
    off = 0
    for g, c in enumerate(counts.tolist()):
        res[off:off + c] = (dy[off:off + c].float() @ w[g * n:(g + 1) * n].float()).bfloat16()
        off += c
    return _fill(out, res, total)


def grouped_linear_wgrad(dy, x, counts, out=None, accumulate=False):
    """dw [G * N, K] of :func:`grouped_linear`: bf16, or of ``out``'s type (bf16 or
    fp32); with ``accumulate`` it is added to ``out``."""
    counts = _as_counts(counts, dy.device)
    if dy.is_cuda:
        return _native_ops().grouped_linear_wgrad(dy, x, counts, out, bool(accumulate))
    _check_counts(counts)
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[0] != dy.shape[0]:
        raise ValueError("x must be bf16 [rows, K] with dy's rows")
    n, k = dy.shape[-1], x.shape[1]
    _check(dy, counts.numel() * n, k, counts.numel(), "dy")
    if accumulate and out is None:
        raise ValueError("accumulate needs an out to add to")
    _check_out(out, (counts.numel() * n, k), (torch.bfloat16, torch.float32))
    _checked_sum(counts, dy.shape[0])
    res = torch.zeros(counts.numel() * n, k)
    off = 0
    for g, c in enumerate(counts.tolist()):
        res[g * n:(g + 1) * n] = dy[off:off + c].float().t() @ x[off:off + c].float()
        off += c
    if out is None:
        return res.bfloat16()
    return out.copy_(out.float() + res if accumulate else res)


class _GroupedLinear(torch.autograd.Function):  # CPU tensors; the native op has its own
    @staticmethod
    def forward(ctx, x, w, counts):
        ctx.save_for_backward(x, w, counts)
        return _forward(x, w, counts)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, counts = ctx.saved_tensors
        dx = grouped_linear_dgrad(dy, w, counts) if ctx.needs_input_grad[0] else None
        dw = grouped_linear_wgrad(dy, x, counts) if ctx.needs_input_grad[1] else None
        return dx, dw, None


def grouped_linear(x, w, counts, out=None):
    """bf16 [rows, N]: each group's rows times its weights; see the module
    docstring.  Without ``out`` it is differentiable in x and w."""
    counts = _as_counts(counts, x.device)
    if out is not None:
        if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
            raise ValueError("out is not differentiable: leave it out, or call under torch.no_grad()")
    if x.is_cuda:
        o = _native_ops()
        return o.grouped_linear(x, w, counts) if out is None else o.grouped_linear_out(x, w, counts, out)
    return _GroupedLinear.apply(x, w, counts) if out is None else _forward(x, w, counts, out)


def _swiglu_halves(y):
    t = y.reshape(y.shape[0], y.shape[1] // 256, 2, 128)
    return t[:, :, 0].flatten(1), t[:, :, 1].flatten(1)


def _check_swiglu(y, row_scale):
    if y.dtype != torch.bfloat16 or y.dim() != 2 or y.shape[1] < 256 or y.shape[1] % 256:
        raise ValueError("y must be bf16 [rows, 2F] with a multiple of 256 columns (128 gate, 128 up, ...)")
    if row_scale is not None and (row_scale.dtype != torch.float32 or tuple(row_scale.shape) != (y.shape[0],)):
        raise ValueError("row_scale must be fp32 [rows]")


def swiglu_grad(dh, y, row_scale=None, need_scale_grad=None):
    """(dy, drow_scale) of :func:`swiglu`; drow_scale is None without row_scale
    (or with ``need_scale_grad=False``)."""
    need = row_scale is not None if need_scale_grad is None else bool(need_scale_grad)
    if y.is_cuda:
        return _native_ops().swiglu_grad(dh, y, row_scale, need)
    _check_swiglu(y, row_scale)
    if dh.dtype != torch.bfloat16 or dh.dim() != 2 or tuple(dh.shape) != (y.shape[0], y.shape[1] // 2):
        raise ValueError("dh must be bf16 [rows, F] for y [rows, 2F]")
    if need and row_scale is None:
        raise ValueError("without row_scale there is no gradient of it")
    g, u = _swiglu_halves(y.float())
    d = dh.float()
    s = torch.ones(y.shape[0], 1) if row_scale is None else row_scale[:, None]
    sig = torch.sigmoid(g)
    dg, du = d * s * u * sig * (1 + g * (1 - sig)), d * s * g * sig
    dy = torch.stack([t.view(len(d), d.shape[1] // 128, 128) for t in (dg, du)], 2).reshape(y.shape).bfloat16()
    return dy, ((d * g * sig * u).sum(1) if need else None)


class _SwiGLU(torch.autograd.Function):  # CPU tensors; the native op has its own
    @staticmethod
    def forward(ctx, y, row_scale):
        ctx.save_for_backward(y, row_scale)
        _check_swiglu(y, row_scale)
        g, u = _swiglu_halves(y.float())
        h = g * torch.sigmoid(g) * u
        return (h if row_scale is None else h * row_scale[:, None]).bfloat16()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        y, row_scale = ctx.saved_tensors
        return swiglu_grad(dh, y, row_scale, row_scale is not None and ctx.needs_input_grad[1])


def swiglu(y, row_scale=None):
    """bf16 [rows, F] of y [rows, 2F] (blocks of 128 gate and 128 up columns),
    times ``row_scale`` (fp32 [rows]); differentiable in both."""
    if y.is_cuda:
        return _native_ops().swiglu(y, row_scale)
    return _SwiGLU.apply(y, row_scale)


def expert_ffn(x, w13, w2, counts, row_scale=None):
    """The experts' SwiGLU FFN on expert-sorted rows, differentiable in x, both
    weights and the routing weights: ``grouped_linear(swiglu(grouped_linear(x,
    w13), row_scale), w2)``, bf16 [rows, H].  ``w13`` [E * 2F, H] has gate and up
    rows interleaved in blocks of 128, ``w2`` is [E * H, F]."""
    counts = _as_counts(counts, x.device)
    return grouped_linear(swiglu(grouped_linear(x, w13, counts), row_scale), w2, counts)


__all__ = ["grouped_linear", "grouped_linear_dgrad", "grouped_linear_wgrad", "swiglu", "swiglu_grad", "expert_ffn"]
