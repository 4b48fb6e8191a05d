"""The FP8 products, the experts' differentiable product and SwiGLU on CPU
tensors: their fp32 restatements, refusals and gradients."""
import pytest
import torch

from kiwi_b200 import ops

BF16, F32 = 2.0 ** -8, 2.0 ** -23


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(0)


def _fp8(groups, n, k, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(rows, k, generator=g).mul(50).to(torch.float8_e4m3fn)
    b = torch.randn(groups * n, k, generator=g).mul(50).to(torch.float8_e4m3fn)
    sa = torch.rand(rows, -(-k // 128), generator=g) + 0.1
    sb = (torch.rand(groups * -(-n // 128), -(-k // 128), generator=g) + 0.1) * 1e-3
    return a, sa, b, sb


def _f64(codes, s, rows_per_scale=1):
    s = s.double().repeat_interleave(rows_per_scale, 0)[:len(codes)]
    return codes.double() * s.repeat_interleave(128, 1)[:, :codes.shape[1]]


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (5, 200, 272), (3, 128, 128)])
def test_dense_fp8_product(m, n, k):
    a, sa, b, sb = _fp8(1, n, k, m)
    x, w = _f64(a, sa), _f64(b, sb, 128)
    ref, mag = x @ w.T, x.abs() @ w.abs().T
    out = ops.fp8_gemm(a, sa, b, sb)
    assert out.dtype == torch.bfloat16
    assert bool(((out.double() - ref).abs() <= BF16 * ref.abs() + F32 * (k + 2) * mag).all())
    into = torch.empty(m, n, dtype=torch.bfloat16)
    assert torch.equal(ops.fp8_gemm(a, sa, b, sb, out=into), out) and torch.equal(into, out)


def test_grouped_fp8_products_and_ffn():
    a, sa, w13, s13 = _fp8(3, 512, 256, 12)
    _, _, w2, s2 = _fp8(3, 256, 256, 1, seed=1)
    counts = torch.tensor([4, 0, 6])
    scale = torch.rand(12)
    codes, scales = ops.grouped_fp8_swiglu(a, sa, w13, s13, counts)
    assert tuple(codes.shape) == (12, 256) and tuple(scales.shape) == (12, 2)
    h = ops.grouped_fp8_gemm(a, sa, w13, s13, counts, swiglu=True)
    d = ops.dequant_fp8(codes, scales)
    s = scales.repeat_interleave(128, 1)
    assert bool(((d - h.float()).abs() <= (2.0 ** -4 + BF16) * h.float().abs() + 2.0 ** -10 * s).all())
    y = ops.expert_ffn_fp8(a, sa, w13, s13, w2, s2, counts, row_scale=scale)
    assert torch.equal(y, ops.grouped_fp8_gemm(codes, scales, w2, s2, counts, row_scale=scale))
    assert bool((y[10:] == 0).all())
    out = torch.full_like(y, 7.0)
    ops.expert_ffn_fp8(a, sa, w13, s13, w2, s2, counts, scale, out)
    assert torch.equal(out[:10], y[:10]) and bool((out[10:] == 7).all())


def test_weight_quantisation_round_trip():
    w = (torch.randn(200, 272) * 0.02).bfloat16()
    w[:128, :128] = 0
    codes, scales = ops.quant_fp8_weights(w)
    assert tuple(codes.shape) == (200, 272) and tuple(scales.shape) == (2, 3)
    assert scales[0, 0] == 1 and bool((codes[:128, :128].float() == 0).all())
    back = ops.dequant_fp8(codes, scales, 128)
    s = scales.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :272]
    assert bool(((back - w.float()).abs() <= (2.0 ** -4 + 4 * F32) * w.float().abs() + 2.0 ** -10 * s).all())


def test_fp8_refusals():
    a, sa, b, sb = _fp8(2, 256, 256, 8)
    cnt = torch.tensor([4, 4])
    bad = [
        lambda: ops.fp8_gemm(a.float(), sa, b, sb),
        lambda: ops.fp8_gemm(a, sa[:, :1], b, sb),
        lambda: ops.fp8_gemm(a, sa.double(), b, sb),
        lambda: ops.fp8_gemm(a, sa, b, sb[:1]),
        lambda: ops.fp8_gemm(a[:, :40], sa[:, :1], b[:, :40], sb[:, :1]),
        lambda: ops.fp8_gemm(a, sa, b[:, :128], sb[:, :1]),
        lambda: ops.fp8_gemm(a, sa, b, sb, out=torch.empty(8, 512)),
        lambda: ops.grouped_fp8_gemm(a, sa, b[:400], sb, cnt),
        lambda: ops.grouped_fp8_gemm(a, sa, b[:256], sb[:2], cnt, swiglu=True),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, cnt, row_scale=torch.ones(7)),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, torch.tensor([5, 4])),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, torch.tensor([-1, 4])),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, [1.5, 2.0]),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, torch.zeros(0, dtype=torch.int32)),
        lambda: ops.expert_ffn_fp8(a, sa, b, sb, b, sb, cnt),
        lambda: ops.quant_fp8_weights(a),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()


COUNTS = [[5], [0, 3, 1], [0, 0], [2, 0, 9]]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
def test_grouped_linear_and_its_gradients(counts):
    n, k, spare = 64, 128, 2
    rows = sum(counts) + spare
    x = torch.randn(rows, k).bfloat16().requires_grad_()
    w = (torch.randn(len(counts) * n, k) * 0.1).bfloat16().requires_grad_()
    dy = torch.randn(rows, n).bfloat16()
    cnt = torch.tensor(counts)
    y = ops.grouped_linear(x, w, cnt)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    off = 0
    for e, c in enumerate(counts):
        xe, de, we = x[off:off + c].double(), dy[off:off + c].double(), w[e * n:(e + 1) * n].double()
        for got, a, b in ((y[off:off + c], xe, we.T), (dx[off:off + c], de, we), (dw[e * n:(e + 1) * n], de.T, xe)):
            ref = a @ b
            assert bool(((got.double() - ref).abs() <= BF16 * ref.abs() + F32 * (a.shape[1] + 1) * (a.abs() @ b.abs())).all())
        off += c
    assert bool((y[off:] == 0).all()) and bool((dx[off:] == 0).all())


def test_weight_gradient_accumulates():
    x, dy = torch.randn(9, 64).bfloat16(), torch.randn(9, 64).bfloat16()
    cnt = torch.tensor([4, 0, 5])
    one = ops.grouped_linear_wgrad(dy, x, cnt, out=torch.empty(192, 64))
    two = ops.grouped_linear_wgrad(dy, x, cnt, out=one.clone(), accumulate=True)
    assert torch.equal(two, 2 * one) and bool((one[64:128] == 0).all())
    assert ops.grouped_linear_wgrad(dy, x, cnt).dtype == torch.bfloat16


@pytest.mark.parametrize("rows", [0, 1, 6])
def test_ffn_gradients_against_autograd(rows):
    """The chain's gradients against autograd of the 64-bit formula: at most three
    roundings of rows to bf16 and one of the gradient, 2^-8 of a value each.

    A routing weight's gradient is one sum, sum_j dh_j a_j u_j with a = silu(g),
    which may cancel, so it is bounded term by term: dh, g and u are each off by
    2^-8 of a value (|silu'| <= 1.1), hence by 2^-8 sum_j |dh_j| (|a_j u_j| +
    1.1 |g_j u_j| + |a_j u_j|), and 5 % for products of errors."""
    torch.manual_seed(rows)
    h, f = 64, 128
    counts = [rows // 2, rows - rows // 2]
    x = torch.randn(rows, h).bfloat16()
    w13 = (torch.randn(2 * 2 * f, h) * 0.1).bfloat16()
    w2 = (torch.randn(2 * h, f) * 0.1).bfloat16()
    s = torch.rand(rows) + 0.5
    d = torch.randn(rows, h).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2, s)]
    out = ops.expert_ffn(leaves[0], leaves[1], leaves[2], counts, leaves[3])
    grads = torch.autograd.grad(out, leaves, d)
    auto = [t.double().requires_grad_() for t in (x, w13, w2, s)]
    outs, off = [], 0
    slack = torch.zeros(rows, dtype=torch.float64)
    for e, c in enumerate(counts):
        y = auto[0][off:off + c] @ auto[1][e * 2 * f:(e + 1) * 2 * f].T
        gate, up = y[:, :128], y[:, 128:]
        a = gate * torch.sigmoid(gate)
        outs.append((a * up * auto[3][off:off + c, None]) @ auto[2][e * h:(e + 1) * h].T)
        dh = d[off:off + c].double() @ auto[2][e * h:(e + 1) * h]
        slack[off:off + c] = 1.05 * BF16 * (dh.abs() * (2 * (a * up).abs() + 1.1 * (gate * up).abs())).sum(1).detach()
        off += c
    ref = torch.cat(outs)
    assert (out.double() - ref).norm() <= 3 * BF16 * ref.norm()
    want = torch.autograd.grad(ref, auto, d.double())
    for g, r in zip(grads[:3], want[:3]):
        assert (g.double() - r).norm() <= 4 * BF16 * r.norm()
    assert bool(((grads[3].double() - want[3]).abs() <= slack).all())


def test_grouped_linear_refusals():
    x, w, dy = torch.zeros(8, 128).bfloat16(), torch.zeros(256, 128).bfloat16(), torch.zeros(8, 128).bfloat16()
    cnt = torch.tensor([4, 4])
    bad = [
        lambda: ops.grouped_linear(x.float(), w, cnt),
        lambda: ops.grouped_linear(x[:, :64], w, cnt),
        lambda: ops.grouped_linear(x[:, :32], w[:, :32], cnt),
        lambda: ops.grouped_linear(x, w[:100], cnt),
        lambda: ops.grouped_linear(x, w, torch.tensor([5, 4])),
        lambda: ops.grouped_linear_dgrad(dy, w[:128], cnt),
        lambda: ops.grouped_linear_wgrad(dy[:5], x, cnt),
        lambda: ops.grouped_linear_wgrad(dy, x, cnt, accumulate=True),
        lambda: ops.grouped_linear_wgrad(dy, x, cnt, out=torch.empty(256, 128).half()),
        lambda: ops.grouped_linear(x.clone().requires_grad_(), w, cnt, out=torch.empty(8, 128).bfloat16()),
        lambda: ops.swiglu(x),
        lambda: ops.swiglu(x.repeat(1, 2).float()),
        lambda: ops.swiglu(x.repeat(1, 2), torch.ones(7)),
        lambda: ops.swiglu_grad(x, x.repeat(1, 4)),
        lambda: ops.swiglu_grad(x, x.repeat(1, 2), None, True),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()


# ---------------------------------------------------------------- the layers that use them


@pytest.mark.parametrize("quant", ["none", "fp8", "nvfp4"])
def test_fp8_experts_in_the_collective_layer(quant):
    """The layer with FP8 experts equals its own pieces: the dispatched rows, FP8
    weights, the FFN's reference and the routing-weighted sum."""
    from kiwi_b200.models import moe
    from kiwi_b200.parallel.ep_collective import CollectiveMoE

    cfg = moe.MoEConfig(hidden=256, ffn=128, num_experts=3, topk=2, tokens_per_rank=20, quant=quant, name="t")
    layer = CollectiveMoE(cfg, device="cpu", weight_format="fp8")
    assert layer.w13.dtype == torch.float8_e4m3fn
    x, logits = moe.synthetic_inputs(cfg, 0, "cpu", tokens=17)
    out = layer(x, logits)
    layer.check()
    idx, w = moe.route_reference(logits, cfg.topk)
    codes, scales = moe.quant_fp8_codes(x) if quant == "fp8" else moe.quant_fp8_codes(
        moe.dispatch_reference(x, quant).bfloat16())
    ref = torch.zeros(17, 256)
    for e in range(3):
        t, s = (idx == e).nonzero(as_tuple=True)
        a, b, c = moe.expert_weights(cfg, e, "cpu")
        w13, s13 = ops.quant_fp8_weights(moe.interleave_gate_up(a, b))
        w2, s2 = ops.quant_fp8_weights(c)
        y = ops.expert_ffn_fp8(codes[t], scales[t], w13, s13, w2, s2, [len(t)], row_scale=w[t, s].float().contiguous())
        ref.index_add_(0, t, y.float())
    # The layer sums bf16 rows in fp32 and rounds once more.
    assert bool(((out.float() - ref).abs() <= BF16 * ref.abs() + 1e-6).all())


def test_fp8_expert_ffn_object():
    from kiwi_b200.models import moe

    cfg = moe.MoEConfig(hidden=256, ffn=128, num_experts=3, topk=1, tokens_per_rank=8, quant="none", name="t")
    w13, w2 = moe.local_expert_weights(cfg, 0, 1, "cpu")
    ffn = ops.ExpertFFN(w13, w2, 3, 16, weight_format="fp8")
    x = torch.randn(10, 256).bfloat16()
    ffn.input_buffer()[:10].copy_(x)
    counts, scale = torch.tensor([4, 0, 6]), torch.rand(16)
    y = ffn(counts, scale)
    assert tuple(y.shape) == (16, 256)
    rows = ops.quant_fp8(x)
    want = ops.expert_ffn_fp8(*rows, ffn.w13, ffn.w13_scale, ffn.w2, ffn.w2_scale, counts, row_scale=scale[:10])
    assert torch.equal(y[:10], want) and torch.equal(ffn(counts, scale, rows=rows), want)
    ffn.check()
    # And near the bf16 experts: e4m3 rows, weights and hidden rows are each off
    # by at most 2^-4 of a value, which a norm over many sees well below 3 * 2^-4.
    ref = ops.ExpertFFN(w13, w2, 3, 16)
    ref.input_buffer()[:10].copy_(x)
    full = ref(counts, scale)[:10].float()
    assert (want.float() - full).norm() <= 3 * 2.0 ** -4 * full.norm()
    for bad in (lambda: ops.ExpertFFN(w13, w2, 3, 16, weight_format="int8"), lambda: ref(counts, scale, rows=rows),
                lambda: ffn(counts, scale, rows=ops.quant_fp8(torch.zeros(17, 256).bfloat16()))):
        with pytest.raises(ValueError):
            bad()
