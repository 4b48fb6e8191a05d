"""Edges of the experts' operators on CPU tensors: blocks too small for a finite
factor, counts past 32 bits, refusals."""
import pytest
import torch

from kiwi_b200 import ops
from kiwi_b200.models import moe

BF16, F32 = 2.0 ** -8, 2.0 ** -23
FLOOR = float.fromhex("0x1.c00002p-120")  # the smallest amax whose 448 / amax is finite in fp32


def _e4m3_close(codes, scale, x):
    """Quantised values against x (64 bits): half a step is 2^-4 of a value, and
    2^-10 of the scale below e4m3's normal range.  2^-20 of a value is for the
    factor's and the scale's own rounding: 2^-24 each, and 2^-22 where the scale
    is subnormal (2^-128 with steps of 2^-149)."""
    got = codes.double() * scale
    assert bool(((got - x).abs() <= (2.0 ** -4 + 2.0 ** -20) * x.abs() + 2.0 ** -10 * scale).all())


TINY = [2.0 ** -149, 1e-40, 1e-37, 1.3e-36, FLOOR * (1 - 2.0 ** -24), FLOOR, 2e-36, 1e-35, 1e-30]


@pytest.mark.parametrize("amax", TINY, ids=lambda a: f"{a:.3g}")
def test_rows_of_a_tiny_block(amax):
    x = torch.zeros(3, 256)
    x[0, 0], x[0, 5], x[0, 200] = amax, -amax / 3, 1.0
    x[1, 100] = -amax
    codes, scales = moe.quant_fp8_codes(x)
    assert bool((scales > 0).all()) and scales[2, 0] == 1 and bool((codes[x == 0].float() == 0).all())
    _e4m3_close(codes, scales.double().repeat_interleave(128, 1), x.double())
    x = x.bfloat16()
    codes, scales = ops.quant_fp8(x)
    _e4m3_close(codes, scales.double().repeat_interleave(128, 1), x.double())


@pytest.mark.parametrize("amax", TINY, ids=lambda a: f"{a:.3g}")
def test_weights_of_a_tiny_block(amax):
    w = torch.zeros(200, 256).bfloat16()
    w[3, 7], w[100, 100], w[0, 200] = amax, -amax / 3, 1.0
    codes, scales = ops.quant_fp8_weights(w)
    assert bool((codes[w == 0].float() == 0).all())
    s = scales.double().repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)
    _e4m3_close(codes, s, w.double())


def test_blocks_with_a_finite_factor_keep_their_codes():
    x = torch.randn(64, 256) * torch.exp2(torch.randint(-118, 60, (64, 1)).float())
    amax = x.view(64, 2, 128).abs().amax(2, keepdim=True)
    assert float(amax.min()) >= FLOOR
    codes, scales = moe.quant_fp8_codes(x)
    want = (x.view(64, 2, 128) * (torch.full_like(amax, 448.0) / amax)).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(scales, (amax / 448)[:, :, 0]) and torch.equal(codes.float(), want.view(64, 256).float())


@pytest.mark.parametrize("magnitude", [1e-18, 1e-19, 3e-20, 1e-20, 1e-21, 1e-22, 1e-23, 1e-37])
def test_ffn_of_tiny_rows(magnitude):
    """Against 64 bits of the same codes: gate and up are fp32 sums of K products
    (K steps of 2^-23 of their magnitudes), each hidden value loses at most 4
    steps of 2^-149 besides and is quantised once (as above, with a scale of at
    least 2^-128), the second product's scales round to a step of 2^-149, and the
    result to bf16 steps of 2^-133 at the least."""
    torch.manual_seed(1)
    h, f, rows = 256, 128, 6
    x = (torch.randn(rows, h) * magnitude).bfloat16()
    a, sa = ops.quant_fp8(x)
    w13, s13 = ops.quant_fp8_weights((torch.randn(2 * f, h) * 0.02).bfloat16())
    w2, s2 = ops.quant_fp8_weights((torch.randn(h, f) * 0.02).bfloat16())
    out = ops.expert_ffn_fp8(a, sa, w13, s13, w2, s2, [rows])
    xd = a.double() * sa.double().repeat_interleave(128, 1)
    wd = w13.double() * s13.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    y, e = xd @ wd.T, h * F32 * (xd.abs() @ wd.abs().T)
    gate, up = y[:, :f], y[:, f:]
    silu = gate * torch.sigmoid(gate)
    hid = silu * up
    d = 1.1 * e[:, :f] * (up.abs() + e[:, f:]) + silu.abs() * e[:, f:] + 16 * F32 * hid.abs() + 4 * 2.0 ** -149
    w = w2.double() * s2.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    ref = hid @ w.T
    s = ((hid.abs() + d).amax(1, keepdim=True) / 448).clamp(min=2.0 ** -128)
    each = (2.0 ** -4 + 2.0 ** -20) * (hid.abs() + d) + 2.0 ** -10 * s + d
    slack = each @ w.abs().T + f * F32 * (hid.abs() + each) @ w.abs().T + f * 448 * 448 * 2.0 ** -149 + 2.0 ** -134
    assert bool(((out.double() - ref).abs() <= BF16 * ref.abs() + slack).all())


def test_rows_too_long_for_32_bits():
    """Meta tensors: the check comes before any arithmetic."""
    k = 2 ** 31 - 16
    a = torch.empty(1, k, dtype=torch.float8_e4m3fn, device="meta")
    s = torch.empty(1, -(-k // 128), device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.fp8_gemm(a, s, a, s)
    x = torch.empty(64, 2 ** 31 - 64, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.grouped_linear(x, x, torch.tensor([64]))


@pytest.mark.parametrize("counts", [[2 ** 32 + 4], [2 ** 31], [-2 ** 32 + 4], [2 ** 32, 4], [2 ** 62 + 2, 2]])
def test_counts_past_32_bits(counts):
    """They were wrapped into 32 bits, 2^32 + 4 into 4."""
    e = len(counts)
    a, s = torch.zeros(8, 128).to(torch.float8_e4m3fn), torch.ones(8, 1)
    b, sb = torch.zeros(e * 128, 128).to(torch.float8_e4m3fn), torch.ones(e, 1)
    x, w = torch.zeros(8, 64).bfloat16(), torch.zeros(e * 64, 64).bfloat16()
    for c in (counts, torch.tensor(counts)):
        with pytest.raises(ValueError, match="counts"):
            ops.grouped_fp8_gemm(a, s, b, sb, c)
        with pytest.raises(ValueError, match="counts"):
            ops.grouped_linear(x, w, c)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8])
def test_counts_of_every_whole_type(dtype):
    x, w = torch.randn(8, 64).bfloat16(), torch.randn(128, 64).bfloat16()
    want = ops.grouped_linear(x, w, [3, 5])
    assert torch.equal(ops.grouped_linear(x, w, torch.tensor([3, 5], dtype=dtype)), want)


@pytest.mark.parametrize("quant", ["none", "fp8", "nvfp4"])
def test_collective_layer_gives_its_fp8_experts_the_rows_it_has(quant, monkeypatch):
    """The experts' buffer is sized for the worst case; a step works on the rows
    that arrived, not on all of it."""
    from kiwi_b200.parallel.ep_collective import CollectiveMoE

    cfg = moe.MoEConfig(hidden=256, ffn=128, num_experts=3, topk=2, tokens_per_rank=50, quant=quant, name="t")
    layer = CollectiveMoE(cfg, device="cpu", weight_format="fp8")
    seen = []
    call = ops.ExpertFFN.__call__
    monkeypatch.setattr(ops.ExpertFFN, "__call__", lambda self, counts, scale=None, rows=None: (
        seen.append((int(counts.sum()), self.max_rows if rows is None else len(rows[0]))), call(self, counts, scale, rows))[1])
    for tokens in (7, 0, 50):
        x, logits = moe.synthetic_inputs(cfg, 0, "cpu", tokens=tokens)
        out = layer(x, logits)
        assert tuple(out.shape) == (tokens, 256) and bool(torch.isfinite(out).all())
    assert seen == [(14, 14), (0, 0), (100, 100)]
