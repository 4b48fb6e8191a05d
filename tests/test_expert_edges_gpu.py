"""Edges of the experts' operators on the GPU: blocks too small for a finite
factor, refusals before a launch, error words, strides and counts that other
tests do not have."""
import pytest
import torch

from kiwi_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -23
FLOOR = float.fromhex("0x1.c00002p-120")  # the smallest amax whose 448 / amax is finite in fp32


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _fp8(g, rows, k, mag=1.0):
    """Quantised bf16 rows and their 64-bit values."""
    x = (torch.randn(rows, k, generator=g, device="cuda") * mag).bfloat16()
    codes, s = ops.quant_fp8(x)
    return codes, s, codes.double() * s.double().repeat_interleave(128, 1)


def _fp8_weights(g, rows, k, mag=0.02):
    codes, s = ops.quant_fp8_weights((torch.randn(rows, k, generator=g, device="cuda") * mag).bfloat16())
    return codes, s, codes.double() * s.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :k]


def _e4m3_close(codes, scale, x, slack=0.0):
    """Quantised values against x (64 bits): half a step is 2^-4 of a value, and
    2^-10 of the scale below e4m3's normal range.  2^-20 of a value is for the
    factor's and the scale's own rounding: 2^-24 each, and 2^-22 where the scale
    is subnormal (2^-128 with steps of 2^-149)."""
    got = codes.double() * scale
    assert bool(((got - x).abs() <= (2.0 ** -4 + 2.0 ** -20) * x.abs() + 2.0 ** -10 * scale + slack).all())


@pytest.mark.parametrize("amax", [2.0 ** -133, 1e-37, 1.3e-36, FLOOR, 1e-35, 1e-30], ids=lambda a: f"{a:.3g}")
def test_tiny_blocks(amax):
    x = torch.zeros(200, 512, device="cuda")
    x[0, 0], x[0, 5], x[0, 200], x[1, 300], x[150, 400] = amax, -amax / 3, 1.0, -amax, amax
    x = x.bfloat16()
    codes, scales = ops.quant_fp8(x)
    assert bool((codes[x == 0].float() == 0).all()) and scales[2, 0] == 1
    _e4m3_close(codes, scales.double().repeat_interleave(128, 1), x.double())
    codes, scales = ops.quant_fp8_weights(x)
    assert bool((codes[x == 0].float() == 0).all())
    _e4m3_close(codes, scales.double().repeat_interleave(128, 0)[:200].repeat_interleave(128, 1), x.double())


@pytest.mark.parametrize("magnitude", [1e-18, 1e-19, 1e-20, 1e-21, 1e-22, 1e-37])
@pytest.mark.parametrize("rows", [3, 2000])  # both kernels
def test_hidden_rows_of_a_tiny_block(rows, magnitude):
    g = _gen(rows)
    k, f = 256, 256
    a, sa, x = _fp8(g, rows, k, magnitude)
    b, sb, w = _fp8_weights(g, 2 * f, k)
    b[:1] = 0  # a zero gate row: a zero hidden column in each block
    w[:1] = 0
    cnt = torch.tensor([rows], dtype=torch.int32, device="cuda")
    codes, scales = ops.grouped_fp8_swiglu(a, sa, b, sb, cnt)
    # gate and up: fp32 sums of K products; the approximate exponential and
    # division cost 16 steps at such gates, underflow 4 steps of 2^-149.
    y, e = x @ w.T, k * F32 * (x.abs() @ w.abs().T)
    y, e = (t.view(rows, f // 128, 2, 128) for t in (y, e))
    gate, up = y[:, :, 0], y[:, :, 1]
    silu = gate * torch.sigmoid(gate)
    h = silu * up
    d = 1.1 * e[:, :, 0] * (up.abs() + e[:, :, 1]) + silu.abs() * e[:, :, 1] + 16 * F32 * h.abs() + 4 * 2.0 ** -149
    _e4m3_close(codes, scales.double().repeat_interleave(128, 1), h.flatten(1), 1.1 * d.flatten(1))
    assert bool((codes[:, 0].float() == 0).all())
    w2, s2, _ = _fp8_weights(g, 256, f)
    out = ops.expert_ffn_fp8(a, sa, b, sb, w2, s2, cnt)
    assert bool(torch.isfinite(out).all())
    assert torch.equal(out, ops.grouped_fp8_gemm(codes, scales, w2, s2, cnt))
    ops.check_gemm()


def test_rows_too_long_for_32_bits():
    """Refused before anything is allocated or launched (the operands are one element each)."""
    k = 2 ** 31 - 16
    a = torch.zeros(1, 1, device="cuda").to(torch.float8_e4m3fn).expand(1, k)
    s = torch.ones(1, 1, device="cuda").expand(1, -(-k // 128))
    with pytest.raises(ValueError, match="2\\^31"):
        ops.fp8_gemm(a, s, a, s)
    x = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(64, 2 ** 31 - 64)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.grouped_linear(x, x, torch.tensor([64], dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="2\\^31"):
        ops.swiglu(x[:1, :1].expand(1, 2 ** 31 - 256))


def test_ffn_refuses_an_out_over_its_row_scale_before_it_launches():
    g = _gen(3)
    a, sa, _ = _fp8(g, 8, 256)
    w13, s13, _ = _fp8_weights(g, 256, 256)
    w2, s2, _ = _fp8_weights(g, 256, 128)
    buf = torch.zeros(8 * 256 + 16, device="cuda", dtype=torch.bfloat16)
    out, scale = buf[:8 * 256].view(8, 256), buf[-24:-8].view(torch.float32)
    # Counts that a launched product reports: nothing may have run.
    cnt = torch.tensor([9], dtype=torch.int32, device="cuda")
    ops.check_gemm()
    with pytest.raises(ValueError, match="overlap"):
        ops.expert_ffn_fp8(a, sa, w13, s13, w2, s2, cnt, row_scale=scale, out=out)
    ops.check_gemm()


def test_out_over_the_counts_is_refused():
    """Every CTA reads the counts for itself: an out written over them would
    change the schedule under the CTAs that start later."""
    g = _gen(6)
    a, sa, _ = _fp8(g, 8, 256)
    w13, s13, _ = _fp8_weights(g, 256, 256)
    w2, s2, _ = _fp8_weights(g, 256, 128)
    x, w = torch.zeros(8, 256, device="cuda").bfloat16(), torch.zeros(256, 256, device="cuda").bfloat16()
    buf = torch.zeros(256 * 256, device="cuda", dtype=torch.bfloat16)
    out, cnt = buf[:8 * 256].view(8, 256), buf[:2].view(torch.int32)
    for f in (lambda: ops.grouped_fp8_gemm(a, sa, w13, s13, cnt, out=out),
              lambda: ops.grouped_fp8_gemm(a, sa, w13, s13, cnt, out=out[:, :128], swiglu=True),
              lambda: ops.expert_ffn_fp8(a, sa, w13, s13, w2, s2, cnt, out=out),
              lambda: ops.grouped_linear(x, w, cnt, out=out),
              lambda: ops.grouped_linear_dgrad(x, w, cnt, out=out),
              lambda: ops.grouped_linear_wgrad(x, x, cnt, out=buf.view(256, 256))):
        with pytest.raises(ValueError, match="overlap"):
            f()
    assert int(cnt) == 0


def test_error_word_is_taken_in_one_step():
    """Read and cleared by one kernel: with a copy and then a memset, a bit that a
    product on another stream sets between the two would be lost."""
    from torch.profiler import ProfilerActivity, profile

    g = _gen(4)
    a, sa, _ = _fp8(g, 8, 128)
    b, sb, _ = _fp8_weights(g, 256, 128)
    ops.check_gemm()
    ops.grouped_fp8_gemm(a, sa, b, sb, torch.tensor([9], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        with pytest.raises(RuntimeError, match="counts"):
            ops.check_gemm()
    names = [e.name for e in p.events()]
    if not names:
        pytest.skip("no profiler events on this machine")
    assert any("take_error" in n for n in names) and not any("emset" in n for n in names), names
    ops.check_gemm()


def _ffn(seed):
    g = _gen(seed)
    w13, w2 = ((torch.randn(2 * 256, k, generator=g, device="cuda") * 0.02).bfloat16() for k in (256, 128))
    return ops.ExpertFFN(w13, w2, 2, 8, weight_format="fp8")


def test_each_ffn_reports_its_own_errors():
    a, b = _ffn(1), _ffn(2)
    good, bad = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in ([4, 4], [4, 5]))
    ops.check_gemm()
    a(bad), b(good)
    b.check()
    ops.check_gemm()  # an object's errors are its own
    with pytest.raises(RuntimeError, match="counts"):
        a.check()
    a.check()


@pytest.mark.parametrize("accumulate", [False, True])
def test_weight_gradient_into_fp32_rows_of_four(accumulate):
    g = _gen(5)
    x, dy = (torch.randn(70, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    cnt = torch.tensor([70], dtype=torch.int32, device="cuda")
    wide = torch.full((64, 68), 2.0, device="cuda")
    ops.grouped_linear_wgrad(dy, x, cnt, out=wide[:, :64], accumulate=accumulate)
    ref = dy.double().T @ x.double()
    bound = 70 * F32 * (dy.double().abs().T @ x.double().abs()) + 4 * F32 * (ref.abs() + 2)
    assert bool(((wide[:, :64].double() - ref - (2 if accumulate else 0)).abs() <= bound).all())
    assert bool((wide[:, 64:] == 2).all())


@pytest.mark.parametrize("counts", [[2 ** 32 + 4], [2 ** 31], [-2 ** 32 + 4]])
def test_counts_past_32_bits_are_reported(counts):
    g = _gen(4)
    a, sa, _ = _fp8(g, 8, 128)
    b, sb, _ = _fp8_weights(g, 256, 128)
    x, w = torch.zeros(8, 64, device="cuda").bfloat16(), torch.zeros(64, 64, device="cuda").bfloat16()
    cnt = torch.tensor(counts, device="cuda")
    ops.check_gemm()
    for f in (lambda: ops.grouped_fp8_gemm(a, sa, b, sb, cnt), lambda: ops.grouped_linear(x, w, cnt)):
        f()
        with pytest.raises(RuntimeError, match="counts"):
            ops.check_gemm()


@pytest.mark.parametrize("quant", ["none", "fp8", "nvfp4"])
def test_collective_layer_with_fp8_experts_and_few_or_no_tokens(quant):
    """Tokens are independent of one another but for the order of an fp32 sum,
    which the number of rows decides: a few tokens come out as they do among
    others, to a bf16 rounding of each expert's row and of their sum, and to the
    neighbouring e4m3 code (2^-3 of a value) of hidden values on a border, of
    which the norm sees few."""
    from kiwi_b200.models import moe
    from kiwi_b200.parallel.ep_collective import CollectiveMoE

    cfg = moe.MoEConfig(hidden=512, ffn=256, num_experts=4, topk=2, tokens_per_rank=600, quant=quant, name="t")
    layer = CollectiveMoE(cfg, weight_format="fp8")
    x, logits = moe.synthetic_inputs(cfg, 0, "cuda", tokens=600)
    full = layer(x, logits)
    for t in (0, 1, 37):
        out = layer(x[:t], logits[:t])
        assert tuple(out.shape) == (t, 512) and bool(torch.isfinite(out).all())
        assert (out.float() - full[:t].float()).norm() <= 2 * BF16 * full[:t].float().norm()
    layer.check()


def test_products_in_a_thread_of_their_own():
    """Tensor maps are built by the driver, which needs a context that a new
    thread may not have bound yet."""
    import threading

    g = _gen(8)
    a, sa, _ = _fp8(g, 40, 256)
    b, sb, _ = _fp8_weights(g, 256, 256)
    x, w = (torch.randn(r, 256, generator=g, device="cuda").bfloat16() for r in (40, 256))
    cnt = torch.tensor([40], dtype=torch.int32, device="cuda")
    out = torch.empty(40, 256, dtype=torch.bfloat16, device="cuda")
    calls = [lambda: ops.fp8_gemm(a, sa, b, sb, out=out).clone(), lambda: ops.grouped_linear(x, w, cnt, out=out).clone(),
             lambda: ops.GroupedGemm(x, w, 1)(cnt, out)[:40].clone()]
    for f in calls:
        want, got = f(), []
        t = threading.Thread(target=lambda: got.append(f()))
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert len(got) == 1 and torch.equal(got[0], want)


def test_a_check_lets_other_threads_run_while_it_waits():
    """A kernel ahead of it on the stream may be waiting for a callback in Python."""
    import threading
    import time

    ops.check_gemm()
    stop, ticks = threading.Event(), []

    def tick():
        while not stop.is_set():
            ticks.append(time.perf_counter())
            time.sleep(1e-3)

    t = threading.Thread(target=tick)
    t.start()
    try:
        torch.cuda._sleep(1_000_000_000)  # half a second of a busy GPU
        begin = time.perf_counter()
        ops.check_gemm()
        end = time.perf_counter()
    finally:
        stop.set()
        t.join()
    assert end - begin > 0.1
    assert sum(begin < x < end for x in ticks) > 10
