"""4-bit operands on the CPU: rules, layouts, refusals; the W4A4 formats of the quant techniques on both devices."""

import pytest
import torch

import economize_b200 as eco
from economize_b200 import ops
from economize_b200.errors import ConfigError
from economize_b200.ops import fp4
from economize_b200.ops.fp4 import FP4Weight
from economize_b200.ops.fp8 import FP8BlockWeight
from economize_b200.techniques.eagle3 import Eagle3Config
from economize_b200.techniques.quant import DraftQuantConfig, QuantConfig

from .helpers import gpu_tiny_model, prompts, reference_greedy, tiny_model


def test_known_values():
    x = torch.zeros(2, 32)
    x[0, :9] = torch.tensor([6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5, 0.2, -5.0])  # 5 is a tie between 4 and 6: 4
    x[1, :4] = torch.tensor([7.0, 1.0, 0.25, -0.75])  # mantissa 1.75: the unit is 2, so 0.25 and 0.5 are halves
    want = torch.tensor([6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5, 0.0, -4.0])
    q = ops.fp4_quantize(x, "mxfp4")
    assert torch.equal(q.dequantize()[0, :9].float(), want)
    assert torch.equal(q.dequantize()[1, :4].float(), torch.tensor([8.0, 1.0, 0.0, -1.0]))
    assert q.codes[0, :5].tolist() == [0x67, 0x45, 0x23, 0x01, 0x0E]  # column 2b in the low nibble
    assert int(q.scales[0, 0, 0]) == 127 and int(q.scales[0, 0, 16]) == 128  # 2^0 and 2^1
    q = ops.fp4_quantize(x, "nvfp4")
    # row 0: 6 / 2688 = 2^-8.8, so 2^-8; its first group's scale is 6 / 6 / 2^-8 = 256, exact
    assert float(q.row_scale[0]) == 2.0 ** -8
    assert torch.equal(q.dequantize()[0, :9].float(), want)


def test_scales_in_the_order_of_the_tensor_cores():
    g = torch.Generator().manual_seed(0)
    for fmt, group in fp4.GROUPS.items():
        rows, cols = 200, 288
        x = torch.randn(rows, cols, generator=g)
        q = ops.fp4_quantize(x, fmt)
        tiles = fp4._tiles(cols, fmt)
        assert q.scales.shape == (2, tiles, 512)
        for r, c in ((0, 0), (5, 64), (33, 100), (127, 287), (128, 31), (199, 256)):
            alone = ops.fp4_quantize(x[r:r + 1], fmt)
            k = c // group
            at = (r % 128 % 32) * 16 + (r % 128 // 32) * 4 + k % 4
            assert int(q.scales[r // 128, k // 4, at]) == int(alone.scales[0, k // 4, k % 4])
        flat = fp4._flat_scales(q.scales, rows, cols, fmt)
        assert torch.equal(fp4._tile_scales(flat, cols, fmt), q.scales)  # and zeros in the padding


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_error_and_product(fmt):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(3, 7, 256, generator=g), torch.randn(40, 256, generator=g) * 0.02
    q = ops.fp4_quantize(x, fmt)
    # a step is at most a third of the value above it, so an error a sixth of the group's largest value
    top = x.view(3, 7, -1, fp4.GROUPS[fmt]).abs().amax(-1, keepdim=True)
    err = (q.dequantize(torch.float32) - x).view(3, 7, -1, fp4.GROUPS[fmt]).abs()
    assert (err <= top / 3.5).all()
    weight = FP4Weight.from_weight(w, fmt)
    y = ops.linear(x, weight)
    assert y.shape == (3, 7, 40) and y.dtype == torch.float32
    torch.testing.assert_close(y, q.dequantize(torch.float32) @ weight.dequantize(torch.float32).t())
    assert torch.equal(ops.linear(q, weight), y.bfloat16())
    assert torch.equal(ops.linear(x, weight, torch.ones(40)), y + 1)
    assert q.nbytes() < x.numel() and repr(q) and repr(weight)


def test_not_finite():
    x = torch.ones(1, 64)
    x[0, 3], x[0, 40] = float("inf"), float("nan")
    for fmt, group in fp4.GROUPS.items():
        d = ops.fp4_quantize(x, fmt).dequantize()[0]
        bad = (~x.isfinite()).view(-1, group).any(-1, keepdim=True).expand(-1, group).reshape(-1)
        clean = ops.fp4_quantize(torch.ones(1, 64), fmt).dequantize()[0]  # (1 / 6 is no e4m3 value: 1.03 in nvfp4)
        assert d[bad].isnan().all() and torch.equal(d[~bad], clean[~bad])


def _plain():
    return FP8BlockWeight.from_weight(torch.ones(128, 128))


def test_refusals():
    x = torch.zeros(2, 64)
    w = FP4Weight.from_weight(torch.ones(8, 64))
    for bad in (lambda: ops.fp4_quantize(x, "fp4"), lambda: ops.fp4_quantize(x[:, :40]), lambda: ops.fp4_quantize(x[:, :0]),
                lambda: ops.fp4_quantize(x.long()), lambda: ops.fp4_quantize(torch.zeros(1, 65568)),
                lambda: ops.linear(x[:, :32], w), lambda: ops.linear(ops.fp4_quantize(x, "mxfp4"), w),
                lambda: ops.linear(ops.fp4_quantize(x), torch.ones(8, 64)),
                lambda: ops.linear(ops.fp4_quantize(x), _plain()), lambda: FP4Weight.from_weight(torch.ones(8)), lambda: FP4Weight(w.codes, w.scales[:, :1], w.row_scale, "nvfp4"),
                lambda: FP4Weight(w.codes, w.scales, w.row_scale, "mxfp4")):
        with pytest.raises(ConfigError):
            bad()
    for kw in (dict(method="gptq"), dict(method="awq"), dict(method="hqq"), dict(group_size=48)):
        with pytest.raises(ConfigError):
            QuantConfig(format="nvfp4_w4a4", **kw)


@pytest.mark.parametrize("fmt", ["nvfp4_w4a4", "mxfp4_w4a4"])
def test_technique_decodes_and_reloads(fmt, tmp_path):
    eff = eco.apply(tiny_model(), QuantConfig(format=fmt))
    tech = eff.techniques["quant"]
    assert isinstance(eff.model.layers[0].wqkv, FP4Weight) and "layers.0.w_down" in tech.skipped  # 688 = 21.5 x 32
    p = prompts((14,))[0]
    out = eff.decode(p, 6).tokens
    assert torch.equal(out, reference_greedy(eff.model, p, 6))
    eff.save_pretrained(tmp_path)
    again = eco.load(tiny_model(), tmp_path)
    assert torch.equal(again.decode(p, 6).tokens, out)
    a, b = eff.model.layers[1].wo, again.model.layers[1].wo
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.row_scale, b.row_scale)
    fake = eco.apply(tiny_model(), QuantConfig(format=fmt, backend="fake"))
    assert torch.equal(fake.model.layers[0].wqkv, eff.model.layers[0].wqkv.dequantize())
    cal = torch.randint(0, 1024, (2, 32), generator=torch.Generator().manual_seed(3))
    smooth = eco.apply(tiny_model(), QuantConfig(format=fmt, method="smoothquant"), calibration=cal)
    assert isinstance(smooth.model.layers[0].w_gate_up, FP4Weight)
    assert smooth.decode(p, 4).tokens.numel() == 4


@pytest.mark.parametrize("fmt", ["nvfp4_w4a4", "mxfp4_w4a4"])
def test_drafter_in_four_bits_stays_lossless(fmt):
    model = tiny_model()
    em = eco.apply(model, Eagle3Config(), DraftQuantConfig(format=fmt))
    assert any(isinstance(m, FP4Weight) for m in em.techniques["eagle3"].modules())
    p = prompts((14,))[0]
    assert torch.equal(em.decode(p, 8).tokens, reference_greedy(model, p, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["nvfp4_w4a4", "mxfp4_w4a4"])
def test_technique_on_the_kernels(cuda, fmt):
    """Logits near those of the dequantised weights, and tree decoding token for token equal to plain decoding."""
    eff = eco.apply(gpu_tiny_model(cuda), QuantConfig(format=fmt), Eagle3Config())
    fake = eco.apply(gpu_tiny_model(cuda), QuantConfig(format=fmt, backend="fake"))
    ids = torch.randint(0, 1024, (2, 40), generator=torch.Generator().manual_seed(0)).to(cuda)
    a, b = eff(ids).float(), fake(ids).float()
    # 4-bit activations add as much error as the 4-bit weights: some 10 % a projection
    assert a.isfinite().all() and float((a - b).norm() / b.norm()) < 0.6
    tree = eco.DecodeConfig(cycle_length=5, draft_policy="dynamic_tree", cuda_graphs=True,
                            draft_policy_options={"depth": 4, "topk": 4, "total_tokens": 20})
    ps = [p.to(cuda) for p in prompts((17, 40))]
    plain = eff.decode_batch(ps, 24, decoding=eco.DecodeConfig(cycle_length=1))
    spec = eff.decode_batch(ps, 24, decoding=tree)
    for x, y in zip(plain, spec):
        assert torch.equal(x.tokens, y.tokens)
    assert ops.require().status(0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["gemma2", "granite", "llama"])
def test_norms_hand_over_four_bits(cuda, family):
    """The executor's norms in front of 4-bit projections against the same model with the fusion turned off. One rounding
    fewer moves a 4-bit value here and there by a step, and such steps spread from layer to layer until two runs differ by
    as much as either does from the model with the same weights and bf16 activations: their distance says nothing. But
    either is as far from that model, where a wrong weight, scale or order would be far from both."""
    from economize_b200.models.config import ModelConfig, tiny_llama
    from economize_b200.models.llama import CausalLM, init_weights

    extra = {"gemma2": dict(sandwich_norm=True), "granite": dict(residual_multiplier=0.22), "llama": {}}[family]
    cfg = tiny_llama(hidden_size=512, head_dim=128, num_heads=4, num_kv_heads=2, intermediate_size=1024, **extra)
    assert isinstance(cfg, ModelConfig)

    def model(**kw):
        return eco.apply(init_weights(CausalLM(cfg, torch.bfloat16, cuda), seed=0, std=0.05),
                         QuantConfig(format="nvfp4_w4a4", **kw))

    em = model()
    ids = torch.randint(0, 1024, (1, 200), generator=torch.Generator().manual_seed(1)).to(cuda)
    fused = em(ids).float()
    em.model._takes_fp4 = lambda layer, weight: False
    apart, wide = em(ids).float(), model(backend="fake")(ids).float()
    assert not torch.equal(fused, apart)
    assert float((fused - wide).norm()) < 1.25 * float((apart - wide).norm()) < 0.75 * float(wide.norm())


def _casts(device):
    x = torch.randn(5, 96, generator=torch.Generator().manual_seed(8)).bfloat16().to(device)
    for fmt in ("nvfp4", "mxfp4"):
        w = torch.randn(40, 96, generator=torch.Generator().manual_seed(9)) * torch.exp2(torch.arange(40.0) - 30)[:, None]
        weight = FP4Weight.from_weight(w.to(device), fmt)
        want, y = weight.dequantize(torch.float32), ops.linear(x, weight)
        holder = torch.nn.ModuleDict({"w": weight})
        for cast in (torch.nn.Module.half, torch.nn.Module.bfloat16, torch.nn.Module.double, torch.nn.Module.float,
                     lambda m: m.to(device, torch.float16)):
            cast(holder)
            assert weight.row_scale.dtype == torch.float32 and weight.codes.dtype == weight.scales.dtype == torch.uint8
            assert torch.equal(weight.dequantize(torch.float32), want) and torch.equal(ops.linear(x, weight), y)
        if device != "cpu":
            assert torch.equal(holder.half().cpu()["w"].dequantize(torch.float32), want.cpu())


def test_casts_leave_the_scales_of_rows():
    _casts("cpu")
    # from meta to a device that has memory: the values are the caller's to fill, the type is not a cast's to change
    meta = FP4Weight.from_weight(torch.ones(8, 64)).to("meta").half()
    assert meta.to_empty(device="cpu").row_scale.dtype == torch.float32


@pytest.mark.gpu
def test_casts_leave_the_scales_of_rows_on_the_kernels(cuda):
    _casts(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 64, 65, 100, 128, 129])
def test_norms_hand_over_four_bits_at_any_row_count(cuda, rows):
    """In a partly quantised model a bf16 projection in front of a norm leaves split-K partials up to 64 rows and a plain
    tensor beyond. The norm is the same on either side: that of the unrounded stream, in 4 bits, bit for bit."""
    from economize_b200.models.config import tiny_llama
    from economize_b200.models.llama import CausalLM, init_weights

    cfg = tiny_llama(hidden_size=512, head_dim=128, num_heads=4, num_kv_heads=2, intermediate_size=1024,
                     residual_multiplier=0.22)
    em = eco.apply(init_weights(CausalLM(cfg, torch.bfloat16, cuda), seed=0, std=0.05),
                   QuantConfig(format="nvfp4_w4a4", exclude=("*o_proj", "*down_proj")))
    lm, g = em.model, torch.Generator(device=cuda).manual_seed(rows)
    layer = lm.layers[0]
    assert isinstance(layer.wo, torch.Tensor) and isinstance(layer.w_gate_up, FP4Weight)
    o, resid = (torch.randn(1, rows, 512, device=cuda, generator=g).bfloat16() for _ in range(2))
    h = ops.linear_parts(o, layer.wo)
    assert isinstance(h, ops.Partials) == (rows <= 64)
    plain = h.sum() if isinstance(h, ops.Partials) else h
    x, stream = lm._input_norm(layer, layer.mlp_norm, layer.w_gate_up, h, resid, True)
    with torch.no_grad():
        normed, want = ops.block_norm(plain, resid, layer.mlp_norm, scale=0.22, eps=cfg.rms_norm_eps)
    q = ops.fp4_quantize(normed, "nvfp4")
    assert isinstance(x, ops.FP4Tensor) and torch.equal(stream, want)
    assert all(torch.equal(a, b) for a, b in zip(x.parts(), q.parts()))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("family", ["gemma2", "granite", "llama"])
def test_norms_hand_over_four_bits_exactly(cuda, fmt, family):
    """The executor's fused norms against passes whose norms and quantisations are two operators, with the family's own
    multiplier and weights of the norms, at row counts of one token, of a tree and of a prompt: equal bits. A multiplier
    that is off by a percent is not equal."""
    from economize_b200.models.config import tiny_llama
    from economize_b200.models.llama import CausalLM, init_weights
    from economize_b200.runtime.cache import StepBatch

    extra = {"gemma2": dict(sandwich_norm=True), "granite": dict(residual_multiplier=0.22), "llama": {}}[family]
    cfg = tiny_llama(hidden_size=512, head_dim=128, num_heads=4, num_kv_heads=2, intermediate_size=1024, **extra)
    lm = eco.apply(init_weights(CausalLM(cfg, torch.bfloat16, cuda), seed=0, std=0.05),
                   QuantConfig(format=fmt + "_w4a4")).model
    g = torch.Generator(device=cuda).manual_seed(3)
    with torch.no_grad():
        for layer in lm.layers:  # norms that differ, so that one taken for another shows
            for name in ("attn_norm", "mlp_norm", "attn_post_norm", "mlp_post_norm"):
                p = getattr(layer, name, None)
                if p is not None:
                    p.copy_(1 + 0.3 * torch.randn(p.shape, device=cuda, generator=g))

    @torch.no_grad()
    def hidden(rows):
        ids = torch.randint(0, 1024, (1, rows), generator=torch.Generator().manual_seed(rows)).to(cuda)
        return lm.forward_step(ids, StepBatch.prefill(torch.tensor([rows], dtype=torch.int32, device=cuda), rows),
                               lm.new_cache(1, 256))[0]

    def input_norm(layer, norm, weight, h, resid, partial, multiplier=extra.get("residual_multiplier", 1.0)):
        assert isinstance(weight, FP4Weight)  # the embeddings enter as they are, branches times the multiplier
        n, s = ops.block_norm(h, resid, norm, scale=multiplier if resid is not None else 1.0, eps=cfg.rms_norm_eps)
        return ops.fp4_quantize(n, fmt), s

    def norm_fp4(weight, h, resid, norm, post_weight=None):
        layer = next(l for l in lm.layers if l.w_gate_up is weight)
        n, s = ops.block_norm(h, resid, layer.mlp_norm, post_weight=layer.attn_post_norm, eps=cfg.rms_norm_eps)
        return ops.fp4_quantize(n, fmt), s

    sizes = (1, 61, 200)
    fused = [hidden(n) for n in sizes]
    if family == "gemma2":
        lm._norm_fp4 = norm_fp4
    else:
        lm._input_norm = input_norm
    assert all(torch.equal(a, hidden(n)) for a, n in zip(fused, sizes))
    if family == "granite":
        lm._input_norm = lambda *args: input_norm(*args, multiplier=0.222)
        assert not any(torch.equal(a, hidden(n)) for a, n in zip(fused, sizes))


def test_row_scales_are_powers_of_two():
    q = ops.fp4_quantize(torch.randn(6, 64, generator=torch.Generator().manual_seed(5)))
    codes, scales, row = q.parts()
    for good in (2.0 ** -100, 1.0, 2.0 ** 120):
        assert torch.equal(FP4Weight(codes, scales, torch.full_like(row, good), "nvfp4").row_scale, torch.full((6,), good))
    for bad in (1.5, 0.0, -1.0, float("nan"), float("inf"), 2.0 ** -101, 2.0 ** 121):
        scale = row.clone()
        scale[3] = bad
        with pytest.raises(ConfigError, match="powers of two"):
            FP4Weight(codes, scales, scale, "nvfp4")
    tiny = FP4Weight.from_weight(torch.tensor([[1e-38] * 32, [3e38] * 32, [0.0] * 32]))  # what quantize makes is taken
    assert tiny.row_scale.tolist() == [2.0 ** -100, 2.0 ** 117, 1.0]
