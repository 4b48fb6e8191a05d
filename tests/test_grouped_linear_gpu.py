"""The experts' bf16 product, its gradients and SwiGLU on the GPU against 64 bits.

Tolerance of a product: one rounding to bf16 (2^-8 of the value) and one fp32
rounding or truncation (2^-23) a summed product, relative to the sum of the
products' magnitudes.
"""
import pytest
import torch

from kiwi_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -23


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _data(g, counts, n, k, spare=0):
    rows = sum(counts) + spare
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(len(counts) * n, k, generator=g, device="cuda") * 0.1).bfloat16()
    dy = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    return x, w, dy, torch.tensor(counts, dtype=torch.int32, device="cuda")


def _close(got, a, b, extra=None, rounding=BF16):
    """got == a @ b within the bound; `extra` is a term added before rounding."""
    a, b = a.double(), b.double()
    ref, mag = a @ b, a.abs() @ b.abs()
    if extra is not None:
        ref, mag = ref + extra.double(), mag + extra.double().abs()
    bad = ~((got.double() - ref).abs() <= rounding * ref.abs() + F32 * (a.shape[1] + 1) * mag)  # a NaN is bad
    assert not bool(bad.any()), (int(bad.sum()), got.double()[bad][:4], ref[bad][:4])


def _groups(counts):
    off = 0
    for e, c in enumerate(counts):
        yield e, off, off + c
        off += c


CASES = [([5], 64, 64), ([0, 0, 130, 1], 128, 192), ([256, 0, 77], 320, 448), ([1] * 9, 64, 320), ([0, 0], 128, 256),
         ([64, 65, 128, 129, 63], 192, 64), ([1000, 3], 256, 512), ([31, 33, 2], 1024, 128),
         ([257, 513, 255], 320, 448), ([300, 0, 33, 770, 256, 1], 64, 576), ([2000, 700, 95], 2560, 1024)]


@pytest.mark.parametrize("counts,n,k", CASES, ids=str)
def test_product_and_gradients_match_64_bits(counts, n, k):
    x, w, dy, cnt = _data(_gen(n + k), counts, n, k, spare=4)
    x.requires_grad_(), w.requires_grad_()
    y = ops.grouped_linear(x, w, cnt)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ops.check_gemm()
    with torch.no_grad():
        for e, i, j in _groups(counts):
            we = w[e * n:(e + 1) * n]
            _close(y[i:j], x[i:j], we.t())
            _close(dx[i:j], dy[i:j], we)
            _close(dw[e * n:(e + 1) * n], dy[i:j].t(), x[i:j])
        total = sum(counts)
        assert bool((y[total:] == 0).all()) and bool((dx[total:] == 0).all())
        assert torch.equal(dw, ops.grouped_linear_wgrad(dy, x, cnt))
        assert torch.equal(dx, ops.grouped_linear_dgrad(dy, w, cnt))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weight_gradient_into_a_buffer(dtype, accumulate):
    counts, n, k = [70, 0, 129], 192, 320
    x, _, dy, cnt = _data(_gen(1), counts, n, k, spare=2)
    held = torch.randn(3 * n, k, generator=_gen(2), device="cuda").to(dtype)
    out = held.clone()
    ops.grouped_linear_wgrad(dy, x, cnt, out=out, accumulate=accumulate)
    ops.check_gemm()
    for e, i, j in _groups(counts):
        s = slice(e * n, (e + 1) * n)
        _close(out[s], dy[i:j].t(), x[i:j], held[s] if accumulate else None, BF16 if dtype == torch.bfloat16 else F32)
    if accumulate:
        assert torch.equal(out[n:2 * n], held[n:2 * n])
    else:
        assert bool((out[n:2 * n] == 0).all())


def test_infinities_and_nan_outside_a_group_stay_outside():
    counts, n, k = [37, 0, 70, 5], 128, 128
    x, w, dy, cnt = _data(_gen(3), counts, n, k, spare=90)
    y0, dx0 = ops.grouped_linear(x, w, cnt), ops.grouped_linear_dgrad(dy, w, cnt)
    dw0 = ops.grouped_linear_wgrad(dy, x, cnt)
    x[112:], dy[112:] = float("nan"), float("inf")   # behind the last group
    x[107:112], dy[107:112] = float("inf"), float("nan")  # the last group's own rows
    w[n:2 * n] = float("nan")                        # the empty group's weights
    y, dx, dw = ops.grouped_linear(x, w, cnt), ops.grouped_linear_dgrad(dy, w, cnt), ops.grouped_linear_wgrad(dy, x, cnt)
    ops.check_gemm()
    assert torch.equal(y[:107], y0[:107]) and torch.equal(dx[:107], dx0[:107])
    assert torch.equal(dw[:3 * n], dw0[:3 * n]) and bool(dw[3 * n:].isnan().all())
    assert bool((y[112:] == 0).all()) and bool((dx[112:] == 0).all())


def test_rows_behind_the_last_group_of_an_out_are_left():
    counts, n, k = [10, 20], 64, 128
    x, w, dy, cnt = _data(_gen(4), counts, n, k, spare=7)
    y, dx = torch.full((37, n), 5.0, device="cuda").bfloat16(), torch.full((37, k), 5.0, device="cuda").bfloat16()
    assert ops.grouped_linear(x, w, cnt, out=y).data_ptr() == y.data_ptr()
    ops.grouped_linear_dgrad(dy, w, cnt, out=dx)
    assert torch.equal(y[:30], ops.grouped_linear(x, w, cnt)[:30]) and bool((y[30:] == 5).all())
    assert torch.equal(dx[:30], ops.grouped_linear_dgrad(dy, w, cnt)[:30]) and bool((dx[30:] == 5).all())


def test_writing_an_out_is_seen_by_autograd():
    x, w, dy, cnt = _data(_gen(18), [8, 8], 64, 64)
    buf = torch.zeros(16, 64, device="cuda", dtype=torch.bfloat16)
    scale = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    z = buf * scale  # saves buf
    ops.grouped_linear(x, w, cnt, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    held = torch.zeros(128, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError):
        ops.grouped_linear_wgrad(dy, x, cnt, out=held)
    with torch.no_grad():
        ops.grouped_linear_wgrad(dy, x, cnt, out=held)
    assert torch.equal(held, ops.grouped_linear_wgrad(dy, x, cnt))


def test_no_rows_at_all():
    w = torch.ones(128, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    cnt = torch.zeros(2, dtype=torch.int32, device="cuda")
    y = ops.expert_ffn(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16),
                       torch.ones(512, 64, device="cuda", dtype=torch.bfloat16),
                       torch.ones(128, 128, device="cuda", dtype=torch.bfloat16), cnt)
    assert tuple(y.shape) == (0, 64)
    y = ops.grouped_linear(x, w, cnt)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert tuple(y.shape) == (0, 64) and tuple(dx.shape) == (0, 64) and bool((dw == 0).all())
    acc = torch.ones(128, 64, device="cuda")
    ops.grouped_linear_wgrad(torch.empty_like(y), x.detach(), cnt, out=acc, accumulate=True)
    assert bool((acc == 1).all())


def test_strided_operands():
    counts, n, k = [33, 50], 128, 192
    x, w, dy, cnt = _data(_gen(5), counts, n, k)
    y, dx, dw = ops.grouped_linear(x, w, cnt), ops.grouped_linear_dgrad(dy, w, cnt), ops.grouped_linear_wgrad(dy, x, cnt)

    def wide(t, pad):
        b = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), device="cuda", dtype=t.dtype)
        b[:, pad // 2:pad // 2 + t.shape[1]] = t
        return b[:, pad // 2:pad // 2 + t.shape[1]]

    for pad in (16, 6):  # rows on 16-byte boundaries, and off them
        assert torch.equal(ops.grouped_linear(wide(x, pad), wide(w, pad), cnt), y)
        assert torch.equal(ops.grouped_linear_dgrad(wide(dy, pad), wide(w, pad), cnt), dx)
        assert torch.equal(ops.grouped_linear_wgrad(wide(dy, pad), wide(x, pad), cnt), dw)
    t = dy.t().contiguous().t()  # column-major
    assert torch.equal(ops.grouped_linear_dgrad(t, w, cnt), dx)
    one = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(83, n)  # the gradient of a sum
    assert torch.equal(ops.grouped_linear_dgrad(one, w, cnt), ops.grouped_linear_dgrad(one.contiguous(), w, cnt))


def test_bad_counts_are_reported():
    x, w, dy, _ = _data(_gen(6), [50, 50], 64, 64)
    ops.check_gemm()
    for counts in ([80, 80], [-1, 100]):
        cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
        for f in (lambda: ops.grouped_linear(x, w, cnt), lambda: ops.grouped_linear_dgrad(dy, w, cnt),
                  lambda: ops.grouped_linear_wgrad(dy, x, cnt)):
            f()
            with pytest.raises(RuntimeError, match="counts"):
                ops.check_gemm()


def test_offsets_past_32_bits():
    rows, n, k = 66000, 32768, 64
    g = _gen(7)
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(n, k, generator=g, device="cuda").bfloat16()
    cnt = torch.tensor([rows], dtype=torch.int32, device="cuda")
    y = ops.grouped_linear(x, w, cnt)
    ops.check_gemm()
    assert y.numel() > 2 ** 31
    for r in (slice(0, 2), slice(65534, 65538), slice(rows - 2, rows)):
        _close(y[r], x[r], w.t())
    # dy of more than 2^31 elements read back in the gradients' products.
    dx = ops.grouped_linear_dgrad(y, w, cnt)
    _close(dx[-2:], y[-2:], w)


def test_runs_on_the_current_stream_behind_its_inputs():
    counts, n, k = [33, 50], 128, 192
    x, w, dy, cnt = _data(_gen(19), counts, n, k)
    want = ops.grouped_linear(x, w, cnt), ops.grouped_linear_dgrad(dy, w, cnt), ops.grouped_linear_wgrad(dy, x, cnt)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    late = [torch.zeros_like(t) for t in (x, w, dy, cnt)]
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        for t, v in zip(late, (x, w, dy, cnt)):
            t.copy_(v)
        x2, w2, dy2, c2 = late
        got = ops.grouped_linear(x2, w2, c2), ops.grouped_linear_dgrad(dy2, w2, c2), ops.grouped_linear_wgrad(dy2, x2, c2)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- SwiGLU


def _halves(y):
    t = y.view(len(y), y.shape[1] // 256, 2, 128)
    return t[:, :, 0].flatten(1), t[:, :, 1].flatten(1)


@pytest.mark.parametrize("rows,ffn", [(1, 128), (7, 256), (8, 384), (9, 1152), (300, 2048), (1000, 128)])
@pytest.mark.parametrize("scaled", [True, False])
def test_swiglu_and_gradients_match_64_bits(rows, ffn, scaled):
    """Each result is a product of a few factors, each good to a few fp32 steps
    (the exponential's error grows with |gate|), rounded once; the routing
    weight's gradient is a sum of ffn of them.  Where exp(-gate) overflows fp32
    (gate < -88.7) the sigmoid is 0 instead of something below 2^-128: a factor
    that is off by at most 2^-128, so a result by that times its other factors."""
    g = _gen(rows + ffn)
    y = (torch.randn(rows, 2 * ffn, generator=g, device="cuda") * 3).bfloat16()
    y[0, :128] = torch.linspace(-100, 100, 128, device="cuda").bfloat16()
    dh = torch.randn(rows, ffn, generator=g, device="cuda").bfloat16()
    s = (torch.rand(rows, generator=g, device="cuda") + 0.1) if scaled else None
    y.requires_grad_()
    leaves = (y,) if s is None else (y, s.requires_grad_())
    h = ops.swiglu(y, s)
    grads = torch.autograd.grad(h, leaves, dh)
    gate, up = (t.double() for t in _halves(y.detach()))
    d, sc = dh.double(), torch.ones(rows, 1, device="cuda").double() if s is None else s.detach().double()[:, None]
    sig = torch.sigmoid(gate)
    steps = (24 + 4 * gate.abs()) * F32
    want = gate * sig * up * sc
    tiny = 2.0 ** -128 * (1 + gate.abs()) ** 2 * (1 + d.abs()) * (1 + up.abs()) * sc + 1e-38  # and bf16's own underflow
    assert bool(((h.double() - want).abs() <= (BF16 + steps) * want.abs() + tiny).all())
    dg, du = _halves(grads[0].double())
    wdu = d * sc * gate * sig
    assert bool(((du - wdu).abs() <= (BF16 + steps) * wdu.abs() + tiny).all())
    # 1 + g (1 - sig) cancels where it is near zero: its error is relative to its terms.
    wdg = d * sc * up * sig * (1 + gate * (1 - sig))
    mag = (d * sc * up * sig).abs() * (1 + (gate * (1 - sig)).abs())
    assert bool(((dg - wdg).abs() <= BF16 * wdg.abs() + steps * mag + tiny).all())
    if scaled:
        t = d * gate * sig * up
        assert bool(((grads[1].double() - t.sum(1)).abs() <= ((steps + ffn * F32) * t.abs() + tiny / sc).sum(1)).all())


def test_swiglu_offsets_past_32_bits():
    rows, ffn = 550_000, 2048
    y = torch.full((rows, 2 * ffn), 0.5, device="cuda", dtype=torch.bfloat16)
    g = _gen(20)
    y[-3:] = torch.randn(3, 2 * ffn, generator=g, device="cuda").bfloat16()
    assert y.numel() > 2 ** 31
    s = torch.rand(rows, generator=g, device="cuda")
    h = ops.swiglu(y, s)
    assert torch.equal(h[-3:], ops.swiglu(y[-3:].clone(), s[-3:].clone()))
    dy, ds = ops.swiglu_grad(h, y, s)
    want = ops.swiglu_grad(h[-3:].clone(), y[-3:].clone(), s[-3:].clone())
    assert torch.equal(dy[-3:], want[0]) and torch.equal(ds[-3:], want[1])


def test_swiglu_strides_and_expanded_gradients():
    g = _gen(12)
    big = torch.randn(40, 530, generator=g, device="cuda").bfloat16()
    for o in (8, 3):
        y = big[:, o:o + 512]
        assert torch.equal(ops.swiglu(y), ops.swiglu(y.contiguous()))
    y = big[:, 8:520].clone().requires_grad_()
    ops.swiglu(y).sum().backward()
    dy, ds = ops.swiglu_grad(torch.ones(40, 256, device="cuda", dtype=torch.bfloat16), y.detach())
    assert torch.equal(y.grad, dy) and ds is None


# ---------------------------------------------------------------- together


def _ffn64(x, w13, w2, s, counts):
    outs = []
    h, f = x.shape[1], w2.shape[1]
    for e, i, j in _groups(counts):
        gate, up = _halves(x[i:j] @ w13[e * 2 * f:(e + 1) * 2 * f].T)
        outs.append((gate * torch.sigmoid(gate) * up * s[i:j, None]) @ w2[e * h:(e + 1) * h].T)
    return torch.cat(outs)


def test_ffn_gradients_against_differences():
    """Directional derivatives of the 64-bit FFN by central differences against
    the kernels' gradients.  Each gradient passes through at most three bf16
    roundings of rows (y, h, dh or dy13) and one of its own: 2^-8 of a value
    each, which in a norm over many independent values stays below 4 * 2^-8."""
    counts, h, f = [30, 0, 41], 128, 256
    g = _gen(13)
    rows = sum(counts)
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
    x = torch.randn(rows, h, generator=g, device="cuda").bfloat16()
    w13 = (torch.randn(3 * 2 * f, h, generator=g, device="cuda") * 0.1).bfloat16()
    w2 = (torch.randn(3 * h, f, generator=g, device="cuda") * 0.1).bfloat16()
    s = torch.rand(rows, generator=g, device="cuda") + 0.5
    dout = torch.randn(rows, h, generator=g, device="cuda").bfloat16()
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2, s)]
    out = ops.expert_ffn(leaves[0], leaves[1], leaves[2], cnt, leaves[3])
    grads = torch.autograd.grad(out, leaves, dout)
    ops.check_gemm()
    d64 = [t.double() for t in (x, w13, w2, s)]
    ref = _ffn64(d64[0], d64[1], d64[2], d64[3], counts)
    assert (out.double() - ref).norm() <= 3 * BF16 * ref.norm()
    auto = [t.clone().requires_grad_() for t in d64]
    formula = torch.autograd.grad(_ffn64(auto[0], auto[1], auto[2], auto[3], counts), auto, dout.double())
    for i, (got, want) in enumerate(zip(grads, formula)):
        assert (got.double() - want).norm() <= 4 * BF16 * want.norm(), i
        v = torch.randn(got.shape, generator=g, device="cuda", dtype=torch.float64)
        eps = 1e-5
        lo, hi = list(d64), list(d64)
        lo[i], hi[i] = d64[i] - eps * v, d64[i] + eps * v
        diff = ((_ffn64(*hi, counts) - _ffn64(*lo, counts)) * dout.double()).sum() / (2 * eps)
        assert abs(float((want * v).sum() - diff)) <= 1e-6 * float((want * v).abs().sum())
        assert abs(float((got.double() * v).sum() - diff)) <= 4 * BF16 * float(want.norm() * v.norm())


def test_gradients_are_once_differentiable_and_only_those_asked_for():
    x, w, dy, cnt = _data(_gen(16), [9, 5], 128, 256)
    x.requires_grad_()
    y = ops.grouped_linear(x, w, cnt)
    dx, = torch.autograd.grad(y, x, dy.clone().requires_grad_(), create_graph=True)
    assert torch.equal(dx, ops.grouped_linear_dgrad(dy, w, cnt))
    with pytest.raises(RuntimeError, match="once differentiable"):
        dx.float().sum().backward()
    s = torch.ones(14, device="cuda", requires_grad=True)
    ds, = torch.autograd.grad(ops.swiglu(x.detach(), s).float().sum(), s, create_graph=True)
    with pytest.raises(RuntimeError, match="once differentiable"):
        ds.sum().backward()
    assert not ops.grouped_linear(x.detach(), w, cnt).requires_grad
    with torch.no_grad():
        assert not ops.swiglu(x).requires_grad


def test_captured_step_follows_counts_and_data():
    """Forward and both gradients in one graph, next to live eager graphs of other leaves."""
    counts, n, k = [20, 30], 128, 128
    x, w, dy, cnt = _data(_gen(14), counts, n, k, spare=6)

    def step():
        return (ops.grouped_linear(x, w, cnt), ops.grouped_linear_dgrad(dy, w, cnt),
                ops.grouped_linear_wgrad(dy, x, cnt), ops.swiglu(dy.repeat(1, 2)))

    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        held = step()
    for c in ([20, 30], [0, 56], [1, 0]):
        cnt.copy_(torch.tensor(c))
        x.mul_(0.5)
        gr.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
    ops.check_gemm()


def test_captured_training_step():
    """Forward and backward of the FFN in one graph, warmed up on the capturing
    stream; replays follow the counts, the data and the weights."""
    counts, h, f = [30, 0, 41], 128, 256
    g = _gen(17)
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
    x = torch.randn(80, h, generator=g, device="cuda").bfloat16().requires_grad_()
    w13 = (torch.randn(3 * 2 * f, h, generator=g, device="cuda") * 0.1).bfloat16().requires_grad_()
    w2 = (torch.randn(3 * h, f, generator=g, device="cuda") * 0.1).bfloat16().requires_grad_()
    s = torch.rand(80, generator=g, device="cuda").requires_grad_()
    d = torch.randn(80, h, generator=g, device="cuda").bfloat16()

    def step():
        y = ops.expert_ffn(x, w13, w2, cnt, s)
        return (y.detach(),) + torch.autograd.grad(y, (x, w13, w2, s), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        held = step()
    for c in ([30, 0, 41], [1, 79, 0], [0, 0, 0]):
        cnt.copy_(torch.tensor(c))
        with torch.no_grad():
            x.mul_(0.9), w2.mul_(1.1)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)
    ops.check_gemm()


def test_refusals():
    x, w, dy, cnt = _data(_gen(15), [4, 4], 128, 128)
    bad = [
        lambda: ops.grouped_linear(x.float(), w, cnt),
        lambda: ops.grouped_linear(x, w.cpu(), cnt),
        lambda: ops.grouped_linear(x[:, :64], w, cnt),
        lambda: ops.grouped_linear(x[:, :32], w[:, :32], cnt),
        lambda: ops.grouped_linear(x, w[:100], cnt),
        lambda: ops.grouped_linear(x, w[:-1], cnt),
        lambda: ops.grouped_linear_dgrad(dy, w[:128], cnt),
        lambda: ops.grouped_linear_wgrad(dy[:5], x, cnt),
        lambda: ops.grouped_linear_wgrad(dy, x, cnt, accumulate=True),
        lambda: ops.grouped_linear_wgrad(dy, x, cnt, out=torch.empty(256, 128, device="cuda", dtype=torch.float16)),
        lambda: ops.grouped_linear(x, w, cnt, out=torch.empty(8, 129, device="cuda", dtype=torch.bfloat16)[:, 1:]),
        lambda: ops.grouped_linear(x, w, cnt, out=x),
        lambda: ops.grouped_linear(x.clone().requires_grad_(), w, cnt, out=torch.empty_like(x)),
        lambda: ops.grouped_linear(x, w, torch.zeros(1025, dtype=torch.int32, device="cuda")),
        lambda: ops.swiglu(x),
        lambda: ops.swiglu(x.repeat(1, 2).float()),
        lambda: ops.swiglu(x.repeat(1, 2), torch.ones(8, device="cuda").double()),
        lambda: ops.swiglu_grad(x, x.repeat(1, 4)),
        lambda: ops.swiglu_grad(x, x.repeat(1, 2), None, True),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
