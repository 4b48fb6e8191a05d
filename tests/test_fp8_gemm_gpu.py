"""Block-scaled FP8 products on the GPU against 64-bit sums of the same codes
and scales.

Tolerance: the result is rounded once to bf16 (half a step, 2^-8 of the value);
the fp32 sum of K products is off by at most K steps of 2^-23 of the sum of
their magnitudes (one rounding or truncation a product, scaling included).
"""
import pytest
import torch

from kiwi_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -23


def _rows(g, rows, k):
    """Codes and scales of random rows; scales over a range of magnitudes."""
    codes = torch.randn(rows, k, generator=g, device="cuda").mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp(torch.randn(rows, -(-k // 128), generator=g, device="cuda"))
    return codes, scales


def _weights(g, groups, n, k):
    codes = torch.randn(groups * n, k, generator=g, device="cuda").mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.exp(torch.randn(groups * -(-n // 128), -(-k // 128), generator=g, device="cuda")) * 1e-4
    return codes, scales


def _f64(codes, scales, rows_per_scale=1):
    s = scales.double().repeat_interleave(rows_per_scale, 0)[:codes.shape[0]]
    return codes.double() * s.repeat_interleave(128, 1)[:, :codes.shape[1]]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _product(a, sa, b, sb):
    """(64-bit product, bound on the fp32 sum's error)."""
    x, w = _f64(a, sa), _f64(b, sb, 128)
    return x @ w.T, F32 * a.shape[1] * (x.abs() @ w.abs().T)


def _close(got, ref, slack):
    bad = ~((got.double() - ref).abs() <= BF16 * ref.abs() + slack)  # a NaN is bad
    assert not bool(bad.any()), (int(bad.sum()), got.double()[bad][:4], ref[bad][:4])


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 256, 128), (2, 7, 144), (33, 129, 112), (64, 1000, 256),
                                   (65, 384, 2064), (127, 255, 640), (129, 257, 384), (300, 640, 1040),
                                   (1, 4096, 2048), (16, 1152, 7168), (700, 2048, 272),
                                   (2000, 300, 272), (1500, 1003, 528), (3000, 512, 128), (200, 1111, 2064), (400, 4096, 512), (48, 2048, 256),
                                   (1000, 1111, 272)])
def test_dense_matches_64_bits(m, n, k):
    g = _gen(m * 7 + n)
    a, sa = _rows(g, m, k)
    b, sb = _weights(g, 1, n, k)
    out = ops.fp8_gemm(a, sa, b, sb)
    ops.check_gemm()
    assert out.dtype == torch.bfloat16 and tuple(out.shape) == (m, n)
    _close(out, *_product(a, sa, b, sb))
    assert torch.equal(out, ops.fp8_gemm(a, sa, b, sb))  # nothing depends on the order of execution


COUNTS = [[5], [0, 0, 130, 1], [256, 0, 77], [1] * 9, [0, 0], [64, 65, 128, 129], [1000, 3], [2000, 0, 1, 7000, 130], [48, 47, 96, 49] * 7]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("swiglu", [False, True])
def test_grouped_matches_64_bits(counts, swiglu):
    n, k, spare = 512, 400, 5
    rows = sum(counts) + spare
    g = _gen(len(counts))
    a, sa = _rows(g, rows, k)
    b, sb = _weights(g, len(counts), n, k)
    scale = torch.rand(rows, generator=g, device="cuda") + 0.5
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = ops.grouped_fp8_gemm(a, sa, b, sb, cnt, swiglu=swiglu, row_scale=scale)
    ops.check_gemm()
    off = 0
    for e, c in enumerate(counts):
        ref, slack = _product(a[off:off + c], sa[off:off + c], b[e * n:(e + 1) * n], sb[e * n // 128:(e + 1) * n // 128])
        if swiglu:
            ref, slack = _swiglu(ref, slack)
        s = scale[off:off + c, None].double()
        _close(out[off:off + c], ref * s, slack * s + F32 * (ref * s).abs())
        off += c
    assert bool((out[off:] == 0).all())


def _swiglu(y, err):
    """64-bit SwiGLU of interleaved columns and its bound: |silu'| <= 1.1, and the
    kernel's exponential, division and products are good to 16 + 2 |gate| steps."""
    t, e = (v.view(len(v), v.shape[1] // 256, 2, 128) for v in (y, err))
    gate, up = t[:, :, 0], t[:, :, 1]
    h = gate * torch.sigmoid(gate) * up
    d = 1.1 * e[:, :, 0] * up.abs() + (gate * torch.sigmoid(gate)).abs() * e[:, :, 1] + 1.1 * e[:, :, 0] * e[:, :, 1]
    return h.flatten(1), (d + h.abs() * (16 + 2 * gate.abs()) * F32).flatten(1)


@pytest.mark.parametrize("counts", [[5], [0, 130, 1], [3, 0, 260], [4000, 0, 3001]], ids=str)
def test_swiglu_rows_come_back_quantised(counts):
    n, k = 768, 272
    rows = sum(counts) + 3
    g = _gen(11)
    a, sa = _rows(g, rows, k)
    b, sb = _weights(g, len(counts), n, k)
    if counts[0]:
        b[:1] = 0  # a zero gate row: a zero hidden column
        a[0] = 0   # an all-zero row: scale 1, codes 0
    cnt = torch.tensor(counts, dtype=torch.int32, device="cuda")
    codes, scales = ops.grouped_fp8_swiglu(a, sa, b, sb, cnt)
    ops.check_gemm()
    assert codes.dtype == torch.float8_e4m3fn and tuple(codes.shape) == (rows, n // 2)
    assert tuple(scales.shape) == (rows, n // 256)
    off = 0
    for e, c in enumerate(counts):
        y, err = _product(a[off:off + c], sa[off:off + c], b[e * n:(e + 1) * n], sb[e * n // 128:(e + 1) * n // 128])
        h, d = _swiglu(y, err)
        s = scales[off:off + c].double().repeat_interleave(128, 1)
        got = codes[off:off + c].double() * s
        # e4m3: half a step is 2^-4 of a value, and 2^-10 of the scale below its
        # normal range; two fp32 roundings on the way there.
        ok = (got - h).abs() <= (2.0 ** -4 + 4 * F32) * h.abs() + 2.0 ** -10 * s + 1.1 * d
        assert bool(ok.all())
        hb, db = h.view(c, n // 256, 128).abs(), d.view(c, n // 256, 128)
        top = hb.amax(2)
        want = torch.where(top > 0, top / 448, torch.ones_like(top))
        assert bool(((scales[off:off + c].double() - want).abs() <= 2 * F32 * want + db.amax(2) / 448).all())
        off += c
    if counts[0]:
        assert bool((scales[0] == 1).all()) and bool((codes[0].float() == 0).all())
    assert bool((codes[off:].float() == 0).all()) and bool((scales[off:] == 1).all())


@pytest.mark.parametrize("groups", [1, 31, 33, 100, 1024])
def test_many_groups(groups):
    n, k = 128, 64
    g = _gen(groups)
    counts = torch.randint(0, 4, (groups,), generator=g, device="cuda", dtype=torch.int32)
    rows = int(counts.sum()) + 1
    a, sa = _rows(g, rows, k)
    b, sb = _weights(g, groups, n, k)
    out = ops.grouped_fp8_gemm(a, sa, b, sb, counts)
    ops.check_gemm()
    e = torch.repeat_interleave(torch.arange(groups, device="cuda"), counts.long())
    x, w = _f64(a, sa)[:rows - 1], _f64(b, sb, 128).view(groups, n, k)
    ref = torch.einsum("rk,rnk->rn", x, w[e])
    slack = F32 * k * torch.einsum("rk,rnk->rn", x.abs(), w[e].abs())
    _close(out[:rows - 1], ref, slack)


def test_ffn_is_its_two_products():
    g = _gen(5)
    counts = torch.tensor([40, 0, 131, 2], dtype=torch.int32, device="cuda")
    rows, h, f = 180, 256, 384
    x, sx = _rows(g, rows, h)
    w13, s13 = _weights(g, 4, 2 * f, h)
    w2, s2 = _weights(g, 4, h, f)
    scale = torch.rand(rows, generator=g, device="cuda")
    y = ops.expert_ffn_fp8(x, sx, w13, s13, w2, s2, counts, row_scale=scale)
    hc, hs = ops.grouped_fp8_swiglu(x, sx, w13, s13, counts)
    want = ops.grouped_fp8_gemm(hc, hs, w2, s2, counts, row_scale=scale)
    ops.check_gemm()
    assert torch.equal(y, want) and bool((y[173:] == 0).all())
    out = torch.full_like(y, 7.0)
    assert ops.expert_ffn_fp8(x, sx, w13, s13, w2, s2, counts, scale, out) is not None
    assert torch.equal(out[:173], y[:173]) and bool((out[173:] == 7).all())


def test_rows_of_other_groups_and_stale_rows_do_not_leak():
    g = _gen(9)
    a, sa = _rows(g, 200, 256)
    b, sb = _weights(g, 3, 256, 256)
    cnt = torch.tensor([60, 0, 70], dtype=torch.int32, device="cuda")
    want = ops.grouped_fp8_gemm(a, sa, b, sb, cnt)
    bad = a.clone()
    bad.view(torch.uint8)[130:] = 0x7F  # NaN codes behind the last group
    bad.view(torch.uint8)[59] = 0x7F    # and one NaN row inside the first
    sb2 = sb.clone()
    sb2[2:4] = float("inf")             # the empty group's scales
    sa2 = sa.clone()
    sa2[130:] = float("nan")
    got = ops.grouped_fp8_gemm(bad, sa2, b, sb2, cnt)
    ops.check_gemm()
    assert bool(got[59].isnan().all()) and bool((got[130:] == 0).all())
    keep = [i for i in range(130) if i != 59]
    assert torch.equal(got[keep], want[keep])


def test_strided_operands_and_outputs():
    g = _gen(3)
    big, sbig = _rows(g, 90, 320)
    wide, swide = _weights(g, 1, 200, 320)
    want = ops.fp8_gemm(big[:, 128:288].contiguous(), sbig[:, 1:3].contiguous(), wide[:, :160].contiguous(),
                        swide[:, :2].contiguous())
    assert torch.equal(ops.fp8_gemm(big[:, 128:288], sbig[:, 1:3], wide[:, :160], swide[:, :2]), want)
    odd = torch.empty(90 * 160 + 1, dtype=torch.uint8, device="cuda")[1:].view(90, 160).view(torch.float8_e4m3fn)
    odd.copy_(big[:, 128:288])  # rows that do not start on 16-byte boundaries
    assert torch.equal(ops.fp8_gemm(odd, sbig[:, 1:3], wide[:, :160], swide[:, :2]), want)
    every = big[::2]
    assert torch.equal(ops.fp8_gemm(every, sbig[::2], wide, swide),
                       ops.fp8_gemm(every.contiguous(), sbig[::2].contiguous(), wide, swide))
    out = torch.full((90, 211), 3.0, device="cuda", dtype=torch.bfloat16)
    ops.fp8_gemm(big[:, 128:288], sbig[:, 1:3], wide[:, :160], swide[:, :2], out=out[:, 5:205])
    assert torch.equal(out[:, 5:205], want)
    assert bool((out[:, :5] == 3).all()) and bool((out[:, 205:] == 3).all())


def test_bad_counts_are_reported_and_write_nothing_outside():
    g = _gen(4)
    a, sa = _rows(g, 100, 128)
    b, sb = _weights(g, 3, 256, 128)
    buf = torch.full((140, 256), 5.0, device="cuda", dtype=torch.bfloat16)
    ops.check_gemm()
    for counts in ([50, 60, 70], [2 ** 31 - 1, 2 ** 31 - 1, 5], [-5, 40, 20]):
        ops.grouped_fp8_gemm(a, sa, b, sb, torch.tensor(counts, dtype=torch.int32, device="cuda"), out=buf[20:120])
        with pytest.raises(RuntimeError, match="counts"):
            ops.check_gemm()
        ops.check_gemm()  # cleared
        assert bool((buf[:20] == 5).all()) and bool((buf[120:] == 5).all())


def test_captured_calls_follow_the_counts_and_share_nothing():
    g = _gen(6)
    a, sa = _rows(g, 150, 256)
    b, sb = _weights(g, 3, 512, 256)
    c1 = torch.tensor([50, 0, 60], dtype=torch.int32, device="cuda")
    c2 = torch.tensor([10, 100, 9], dtype=torch.int32, device="cuda")
    run = lambda c: ops.grouped_fp8_swiglu(a, sa, b, sb, c)  # noqa: E731
    run(c1), run(c2)
    torch.cuda.synchronize()
    graphs = []
    for c in (c1, c2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = run(c)
        graphs.append((gr, o))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (gr, _), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for (_, o), c in zip(graphs, (c1, c2)):
            want = run(c)
            assert torch.equal(o[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(o[1], want[1])
        c1.copy_(torch.tensor([0, 150, 0]))
        c2.copy_(torch.tensor([1, 1, 1]))
    ops.check_gemm()


@pytest.mark.parametrize("rows,groups,h,f", [(9, 4, 256, 128), (70, 3, 1024, 512), (3000, 4, 512, 384)])
def test_captured_ffn_and_calls_in_a_row(rows, groups, h, f):
    """The FFN's second product starts while its first one ends: in graphs, with
    other rows and counts from replay to replay, and with calls back to back that
    reuse each other's memory, each result is that of a call by itself."""
    g = _gen(rows)
    x, sx = _rows(g, rows, h)
    w13, s13 = _weights(g, groups, 2 * f, h)
    w2, s2 = _weights(g, groups, h, f)
    scale = torch.rand(rows, generator=g, device="cuda")
    cnt = torch.zeros(groups, dtype=torch.int32, device="cuda")
    inputs = []
    for i in range(3):
        c = torch.bincount(torch.randint(0, groups, (rows - i,), generator=g, device="cuda"), minlength=groups)
        inputs.append((_rows(g, rows, h), c.int()))
    alone = []
    for (a, sa), c in inputs:
        hc, hs = ops.grouped_fp8_swiglu(a, sa, w13, s13, c)
        torch.cuda.synchronize()
        alone.append(ops.grouped_fp8_gemm(hc, hs, w2, s2, c, row_scale=scale))
        torch.cuda.synchronize()
        del hc, hs
    for _ in range(5):
        got = [ops.expert_ffn_fp8(a, sa, w13, s13, w2, s2, c, row_scale=scale) for (a, sa), c in inputs]
        for y, want in zip(got, alone):
            assert torch.equal(y, want)
        del got, y
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        one = ops.expert_ffn_fp8(x, sx, w13, s13, w2, s2, cnt, row_scale=scale)
        two = ops.expert_ffn_fp8(x, sx, w13, s13, w2, s2, cnt, row_scale=scale)
    for ((a, sa), c), want in zip(inputs, alone):
        x.view(torch.uint8).copy_(a.view(torch.uint8)), sx.copy_(sa), cnt.copy_(c)
        for _ in range(3):
            gr.replay()
        assert torch.equal(one, want) and torch.equal(two, want)
    ops.check_gemm()


def test_runs_on_the_current_stream():
    g = _gen(8)
    a, sa = _rows(g, 64, 256)
    b, sb = _weights(g, 1, 256, 256)
    want = ops.fp8_gemm(a, sa, b, sb)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    late = torch.zeros_like(a.view(torch.uint8))
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        late.copy_(a.view(torch.uint8))
        out = ops.fp8_gemm(late.view(torch.float8_e4m3fn), sa, b, sb)
    s.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("r,k", [(128, 128), (1, 1), (130, 257), (700, 2064), (256, 1032)])
def test_weight_quantisation(r, k):
    g = _gen(r + k)
    w = (torch.randn(r, k, generator=g, device="cuda") * 0.02).bfloat16()
    w[:, :1] = 0
    if r >= 128 and k >= 128:
        w[:128, :128] = 0
    codes, scales = ops.quant_fp8_weights(w)
    ref_c, ref_s = ops.quant_fp8_weights(w.cpu())
    assert torch.equal(scales.cpu(), ref_s)
    # The GPU and the CPU divide and multiply alike in fp32; a value on the border
    # of two codes may still fall to either.
    near = (codes.float().cpu() - ref_c.float()).abs() <= 2.0 ** -3 * ref_c.float().abs() + 2.0 ** -9
    assert bool(near.all()) and (codes.float().cpu() != ref_c.float()).float().mean() < 1e-3
    back = ops.dequant_fp8(codes, scales, 128)
    s = scales.repeat_interleave(128, 0)[:r].repeat_interleave(128, 1)[:, :k]
    assert bool(((back - w.float()).abs() <= (2.0 ** -4 + 4 * F32) * w.float().abs() + 2.0 ** -10 * s).all())
    part = torch.zeros(r, k + 3, device="cuda", dtype=torch.bfloat16)
    part[:, 3:] = w
    c2, s2 = ops.quant_fp8_weights(part[:, 3:])
    assert torch.equal(c2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s2, scales)


def test_offsets_past_32_bits():
    """An output of more than 2^31 elements, and its last rows."""
    m, n, k = 66000, 32768, 16
    g = _gen(2)
    a, sa = _rows(g, m, k)
    b, sb = _weights(g, 1, n, k)
    out = ops.fp8_gemm(a, sa, b, sb)
    ops.check_gemm()
    assert out.numel() > 2 ** 31
    for r in (slice(0, 3), slice(32767, 32770), slice(m - 3, m)):
        _close(out[r], *_product(a[r], sa[r], b, sb))


def _codes(g, rows, k):
    """Random finite codes, made in place of a conversion's fp32 operand."""
    c = torch.randint(0, 100, (rows, k), generator=g, device="cuda", dtype=torch.uint8)
    return c.bitwise_or_(torch.randint(0, 2, (1, k), generator=g, device="cuda", dtype=torch.uint8) << 7).view(torch.float8_e4m3fn)


def test_operands_past_32_bits():
    """Rows of more than 2^31 bytes, and weights of more, of which the last group alone has rows."""
    m, n, k = 300_001, 16, 7168
    g = _gen(22)
    a = _codes(g, m, k)
    sa = torch.rand(m, k // 128, generator=g, device="cuda")
    b, sb = _weights(g, 1, n, k)
    out = ops.fp8_gemm(a, sa, b, sb)
    for r in (slice(0, 2), slice(299_592, 299_596), slice(m - 2, m)):
        _close(out[r], *_product(a[r], sa[r], b, sb))
    groups, n = 33, 9216
    w = _codes(g, groups * n, k)
    sw = torch.rand(groups * n // 128, k // 128, generator=g, device="cuda") * 1e-3
    cnt = torch.zeros(groups, dtype=torch.int32, device="cuda")
    for rows in (3, 600):
        cnt[-1] = rows
        out = ops.grouped_fp8_gemm(a[:rows], sa[:rows], w, sw, cnt)
        _close(out, *_product(a[:rows], sa[:rows], w[-n:], sw[-n // 128:]))
    ops.check_gemm()


def test_refusals():
    g = _gen(1)
    a, sa = _rows(g, 8, 256)
    b, sb = _weights(g, 2, 256, 256)
    cnt = torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    bad = [
        lambda: ops.fp8_gemm(a.float(), sa, b, sb),
        lambda: ops.fp8_gemm(a, sa[:, :1], b, sb),
        lambda: ops.fp8_gemm(a, sa.double(), b, sb),
        lambda: ops.fp8_gemm(a, sa.cpu(), b, sb),
        lambda: ops.fp8_gemm(a, sa, b.cpu(), sb.cpu()),
        lambda: ops.fp8_gemm(a, sa, b, sb[:1]),
        lambda: ops.fp8_gemm(a[:, :40], sa[:, :1], b[:, :40], sb[:, :1]),
        lambda: ops.fp8_gemm(a, sa, b[:, :128], sb[:, :1]),
        lambda: ops.fp8_gemm(a, sa, b, sb, out=torch.empty(8, 512, device="cuda")),
        lambda: ops.fp8_gemm(a, sa, b, sb, out=torch.empty(8, 511, device="cuda", dtype=torch.bfloat16)),
        lambda: ops.grouped_fp8_gemm(a, sa, b[:400], sb, cnt),
        lambda: ops.grouped_fp8_gemm(a, sa, b[:256], sb[:2], cnt, swiglu=True),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, cnt, row_scale=torch.ones(7, device="cuda")),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, torch.zeros(0, dtype=torch.int32, device="cuda")),
        lambda: ops.grouped_fp8_gemm(a, sa, b, sb, [1.5, 2.0]),
        lambda: ops.expert_ffn_fp8(a, sa, b, sb, b, sb, cnt),
        lambda: ops.quant_fp8_weights(a),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    assert tuple(ops.fp8_gemm(a[:0], sa[:0], b, sb).shape) == (0, 512)
    ops.check_gemm()


@pytest.mark.parametrize("quant", ["none", "fp8"])
def test_fp8_experts_in_the_collective_layer(quant):
    """The layer with FP8 experts equals its own pieces: dispatched rows, FP8
    weights, each expert's FFN and the routing-weighted sum."""
    from kiwi_b200.models import moe
    from kiwi_b200.parallel.ep_collective import CollectiveMoE

    cfg = moe.MoEConfig(hidden=512, ffn=256, num_experts=8, topk=2, tokens_per_rank=64, quant=quant, name="t")
    layer = CollectiveMoE(cfg, weight_format="fp8")
    for step in range(2):
        t = 64 - 20 * step
        x, logits = moe.synthetic_inputs(cfg, 0, "cuda", tokens=t, step=step)
        out = layer(x, logits)
        layer.check()
        idx, w = ops.route_topk(logits, cfg.topk)
        codes, scales = ops.quant_fp8(x)
        ref = torch.zeros(t, 512, device="cuda")
        for e in range(8):
            r, s = (idx == e).nonzero(as_tuple=True)
            a, b, c = moe.expert_weights(cfg, e, "cuda")
            w13, s13 = ops.quant_fp8_weights(moe.interleave_gate_up(a, b))
            w2, s2 = ops.quant_fp8_weights(c)
            y = ops.expert_ffn_fp8(codes[r], scales[r], w13, s13, w2, s2, [len(r)], row_scale=w[r, s].contiguous())
            ref.index_add_(0, r, y.float())
        # bf16 rows of this comparison may be rounded from sums in another order
        # (the kernels split K by the number of rows): one bf16 step each way.
        assert bool(((out.float() - ref).abs() <= 4 * BF16 * ref.abs() + 2 * BF16 * ref.abs().max()).all())
        assert (out.float() - ref).norm() <= 2 * BF16 * ref.norm()


def test_fp8_expert_ffn_object():
    from kiwi_b200.models import moe

    cfg = moe.MoEConfig(hidden=256, ffn=128, num_experts=3, topk=1, tokens_per_rank=8, quant="none", name="t")
    w13, w2 = moe.local_expert_weights(cfg, 0, 1, "cuda")
    ffn = ops.ExpertFFN(w13, w2, 3, 16, weight_format="fp8")
    x = torch.randn(10, 256, device="cuda").bfloat16()
    ffn.input_buffer()[:10].copy_(x)
    counts, scale = torch.tensor([4, 0, 6], device="cuda"), torch.rand(16, device="cuda")
    rows = ops.quant_fp8(x)
    want = ops.expert_ffn_fp8(*rows, ffn.w13, ffn.w13_scale, ffn.w2, ffn.w2_scale, counts, row_scale=scale[:10])
    y = ffn(counts, scale).clone()
    assert tuple(y.shape) == (16, 256) and (y[:10].float() - want.float()).norm() <= BF16 * want.float().norm()
    assert torch.equal(ffn(counts, scale, rows=rows), want)
    ffn.check()
    with pytest.raises(ValueError):
        ffn(counts, scale, rows=ops.quant_fp8(torch.zeros(17, 256, device="cuda").bfloat16()))
