"""The norms around a block on the CPU: the formulas, their gradients, refusals; scaled residuals in packed training."""

import copy

import pytest
import torch
import torch.nn.functional as F

import economize_b200 as eco
from economize_b200 import ops
from economize_b200.errors import ConfigError
from economize_b200.models.config import tiny_llama
from economize_b200.models.llama import CausalLM, init_weights
from economize_b200.runtime.cache import StepBatch
from economize_b200.techniques.width_prune import WidthPruneConfig
from economize_b200.train import PackedSource, fit, pack
from economize_b200.train.objective import OBJECTIVES


def _tensors(rows=5, hidden=12, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = [torch.randn(rows, hidden, generator=g, dtype=dtype) for _ in range(2)]
    t += [1 + 0.2 * torch.randn(hidden, generator=g, dtype=dtype) for _ in range(2)]
    return t + [torch.rand(rows, 1, generator=g, dtype=dtype), torch.rand(rows, hidden, generator=g, dtype=dtype)]


def _rms(v, eps):
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)


def test_formula_and_gradients():
    x, r, w, p, token, full = _tensors()
    for post, gate, res, scale in ((None, None, r, 1.0), (p, None, r, 0.22), (p, token, r, 2.0), (None, full, None, 0.5)):
        b = x if post is None else _rms(x, 1e-5) * post
        s = scale * (b if gate is None else b * gate) + (0 if res is None else res)
        normed, stream = ops.block_norm(x, res, w, post_weight=post, gate=gate, scale=scale, eps=1e-5)
        torch.testing.assert_close(stream, s)
        torch.testing.assert_close(normed, _rms(s, 1e-5) * w)
        leaves = [t.clone().requires_grad_() for t in (x, res, w, post, gate) if t is not None]

        def call(*t):
            it = iter(t)
            args = [next(it) if given is not None else None for given in (x, res, w, post, gate)]
            return ops.block_norm(args[0], args[1], args[2], post_weight=args[3], gate=args[4], scale=scale, eps=1e-5)

        assert torch.autograd.gradcheck(call, leaves)


def test_types_and_four_bits():
    x, r, w, *_ = _tensors(hidden=64, dtype=torch.float32)
    normed, stream = ops.block_norm(x.bfloat16(), r.bfloat16(), w.bfloat16())
    assert normed.dtype == stream.dtype == torch.bfloat16
    q, s = ops.block_norm(x.bfloat16(), r.bfloat16(), w.bfloat16(), quantize="mxfp4")
    assert torch.equal(s, stream) and torch.equal(q.codes, ops.fp4_quantize(normed, "mxfp4").codes)
    y = x.view(5, 2, 32)
    a, _ = ops.block_norm(y, None, w[:32])
    assert a.shape == y.shape


def test_refusals():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for args, kw in (((x, None, w[:4]), {}), ((x, x[:2], w), {}), ((x, None, w.double()), {}), ((x, None, w[None]), {}),
                     ((x, None, w), {"post_weight": w[:1]}), ((x, None, w), {"gate": x[:, :2]}),
                     ((x, None, w), {"scale": float("nan")}), ((x, None, w), {"eps": -1.0}),
                     ((x, None, w), {"quantize": "fp8"}), ((x.long(), None, w.long()), {})):
        with pytest.raises(ValueError):
            ops.block_norm(*args, **kw)


def _scaled(dtype=torch.float32, device="cpu", **kw):
    cfg = tiny_llama(residual_multiplier=0.3, attention_multiplier=0.09, logits_scaling=3.0, embedding_multiplier=4.0, **kw)
    model = init_weights(CausalLM(cfg, dtype, device), seed=0, std=0.06)
    data = torch.randint(0, 1024, (2, 48), generator=torch.Generator().manual_seed(3)).to(device)
    em = eco.apply(model, WidthPruneConfig(ratio=0.5, recovery_rank=8), calibration=data)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for lora in em.techniques["width_prune"].recovery.values():
            lora.b.copy_(0.05 * torch.randn(lora.b.shape, generator=g).to(lora.b))
    return em


def _documents(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, 1024, (n,), generator=g) for n in lens]


@torch.no_grad()
def _engine_loss(model, docs):
    """The mean next-token loss of every document by itself, by the engine's own forward pass."""
    total, count = 0.0, 0
    for doc in docs:
        if doc.numel() < 2:
            continue
        n = doc.numel()
        h, _ = model.forward_step(doc[None], StepBatch.prefill(torch.tensor([n], dtype=torch.int32), n),
                                  model.new_cache(1, 512))
        total += float(F.cross_entropy(model.logits(h)[0, :-1].double(), doc[1:], reduction="sum"))
        count += n - 1
    return total / count


def test_packed_training_of_scaled_residuals():
    em = _scaled()
    docs = _documents([17, 1, 30, 5])
    obj = OBJECTIVES.get("packed_recovery_ce")(em)
    loss, _ = obj.loss(pack(docs, length=60))
    assert float(loss.detach()) == pytest.approx(_engine_loss(em.model, docs), rel=1e-5)
    # gradients against differences of the engine's loss
    params = obj.parameters()
    grads = torch.autograd.grad(loss, params)
    g = torch.Generator().manual_seed(7)
    for p, grad in list(zip(params, grads))[:4]:
        v = torch.randn(p.shape, generator=g)
        v, step = v / v.norm(), 0.02
        with torch.no_grad():
            p.add_(step * v)
            up = _engine_loss(em.model, docs)
            p.sub_(2 * step * v)
            down = _engine_loss(em.model, docs)
            p.add_(step * v)
        assert (up - down) / (2 * step) == pytest.approx(float((grad * v).sum()), rel=0.05, abs=2e-5)
    fit(em, PackedSource(docs, 64, seed=2), objective="packed_recovery_ce", steps=3, warmup_steps=1, log_every=100)
    with pytest.raises(ConfigError, match="scaled attention or residuals"):
        OBJECTIVES.get("recovery_ce")(em).loss(docs[0][None])


@pytest.mark.gpu
def test_packed_training_of_scaled_residuals_on_the_kernels(cuda):
    em = _scaled(torch.bfloat16, cuda, hidden_size=256, num_heads=2, num_kv_heads=1, head_dim=128)
    from economize_b200.ops.lora import LoRAWeight

    wide = copy.deepcopy(em.model).float().cpu()
    for lora in (m for m in wide.modules() if isinstance(m, LoRAWeight)):
        lora._base[0] = lora._base[0].detach().float().cpu()
    docs = _documents([150, 1, 300, 33])
    obj = OBJECTIVES.get("packed_recovery_ce")(em)
    loss, _ = obj.loss(pack(docs, length=500))
    grads = torch.autograd.grad(loss, obj.parameters())
    assert all(g.isfinite().all() for g in grads)
    assert float(loss.detach()) == pytest.approx(_engine_loss(wide, docs), rel=1e-2)
    fit(em, PackedSource([d.to(cuda) for d in docs], 512, seed=2), objective="packed_recovery_ce", steps=3, warmup_steps=1,
        log_every=100)
    assert ops.require().status(0) == 0


def _stream_gradients(x, r, w, p, gate, dev="cpu"):
    """Of a 4-bit call and of the plain one: results and the stream's gradients."""
    out = []
    for kw in ({}, {"quantize": "mxfp4"}):
        leaves = [t.to(dev).bfloat16().requires_grad_() for t in (x, r, w, p, gate)]
        normed, stream = ops.block_norm(leaves[0], leaves[1], leaves[2], post_weight=leaves[3], gate=leaves[4], scale=0.5, **kw)
        up = torch.linspace(-1, 1, stream.numel(), device=dev).view_as(stream).bfloat16()
        grads = torch.autograd.grad(stream, [leaves[i] for i in (0, 1, 3, 4)], up)
        out.append((normed, stream, grads))
    (n, s, g), (q, s4, g4) = out
    assert torch.equal(s, s4) and torch.equal(ops.fp4_quantize(n.detach(), "mxfp4").codes, q.codes)
    assert all(torch.equal(a, b) for a, b in zip(g, g4))
    with torch.no_grad():
        q, s = ops.block_norm(*leaves[:3], post_weight=leaves[3], gate=leaves[4], scale=0.5, quantize="mxfp4")
    assert not s.requires_grad and torch.equal(s, s4) and torch.equal(q.codes, out[1][0].codes)


def test_the_stream_of_a_four_bit_call_keeps_its_gradient():
    x, r, w, p, token, full = _tensors(hidden=64)
    _stream_gradients(x, r, w, p, token)
    _stream_gradients(x, r, w, p, full)


@pytest.mark.gpu
def test_the_stream_of_a_four_bit_call_keeps_its_gradient_on_the_kernels(cuda):
    x, r, w, p, token, full = _tensors(rows=130, hidden=416)
    _stream_gradients(x, r, w, p, token, cuda)
    _stream_gradients(x, r, w, p, full, cuda)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: ops.block_norm(v, None, w.to(cuda).bfloat16(), quantize="nvfp4")[1],
                       (x.to(cuda).bfloat16(),), (x.to(cuda).bfloat16(),))
