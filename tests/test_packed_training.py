"""Packed documents: rows, the source, and the recovery objective against each document by itself."""

import copy

import pytest
import torch
import torch.nn.functional as F

import economize_b200 as eco
from economize_b200.errors import ConfigError
from economize_b200.ops.reference import rmsnorm
from economize_b200.techniques.width_prune import WidthPruneConfig
from economize_b200.train import PackedSource, fit, pack
from economize_b200.train.objective import OBJECTIVES, torch_block

from .helpers import tiny_model


def _documents(lens, vocab=1024, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, vocab, (n,), generator=g) for n in lens]


def _pruned(model=None):
    model = model or tiny_model()
    data = torch.randint(0, 1024, (2, 48), generator=torch.Generator().manual_seed(3)).to(model.device)
    em = eco.apply(model, WidthPruneConfig(ratio=0.5, recovery_rank=8), calibration=data)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():  # adapters that do something
        for lora in em.techniques["width_prune"].recovery.values():
            lora.b.copy_(0.05 * torch.randn(lora.b.shape, generator=g).to(lora.b))
    return em


def _by_document(target, docs):
    """Summed next-token losses of every document run alone in fp32, and how many tokens they cover."""
    c, total, count = target.config, 0.0, 0
    for doc in docs:
        if doc.numel() < 2:
            continue
        cos, sin = target.rope_tables(doc.numel())
        h = target.embed_tokens(doc[None]).float()
        for layer in target.layers:
            h = torch_block(layer, h, c, cos, sin)
        logits = F.linear(rmsnorm(h, target.norm.float(), c.rms_norm_eps)[0], target.head_weight.float())
        total = total + F.cross_entropy(logits[0, :-1], doc[1:], reduction="sum")
        count += doc.numel() - 1
    return total, count


def test_pack_counts_positions_and_targets_within_documents():
    docs = _documents([3, 0, 1, 4])
    b = pack(docs, length=11)
    assert b.cu_seqlens.tolist() == [0, 3, 3, 4, 8] and b.cu_seqlens.dtype == torch.int32
    assert b.positions.tolist() == [0, 1, 2, 0, 0, 1, 2, 3, 0, 0, 0]
    want = [int(docs[0][1]), int(docs[0][2]), -100, -100, *docs[3][1:].tolist(), -100, -100, -100, -100]
    assert b.targets.tolist() == want
    assert torch.equal(b.tokens[:8], torch.cat(docs)) and (b.tokens[8:] == 0).all()
    with pytest.raises(ConfigError, match="do not fit"):
        pack(docs, length=7)


def test_source_fills_rows_and_resumes():
    src = PackedSource(_documents([5, 9, 30, 2]), 64, seed=1)
    first = src.next()
    assert first.tokens.numel() == 64 and int(first.cu_seqlens[-1]) == 64
    state = src.state()
    second = src.next()
    src.restore(state)
    assert torch.equal(src.next().tokens, second.tokens)
    with pytest.raises(ConfigError, match="not empty"):
        PackedSource([torch.empty(0)], 8)
    with pytest.raises(ConfigError, match="positive"):
        PackedSource(_documents([3]), 0)


def _rows_of_rank(rank, port, queue):
    import datetime

    torch.distributed.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2,
                                         timeout=datetime.timedelta(seconds=60))
    try:
        src = PackedSource(_documents([5, 9, 30, 2]), 64, seed=1)
        queue.put((rank, [src.next().tokens.tolist() for _ in range(3)]))
        torch.distributed.barrier()
    finally:
        torch.distributed.destroy_process_group()


@pytest.mark.slow
def test_ranks_draw_rows_of_their_own():
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    procs = [ctx.Process(target=_rows_of_rank, args=(r, port, queue)) for r in range(2)]
    for p in procs:
        p.start()
    rows = dict(queue.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
    assert all(a != b for a, b in zip(rows[0], rows[1]))
    alone = PackedSource(_documents([5, 9, 30, 2]), 64, seed=1)
    assert [alone.next().tokens.tolist() for _ in range(3)] == rows[0]


def test_ranks_resume_from_one_checkpoint():
    """A run's checkpoint holds the position of one rank; another continues with the rows that it would have drawn."""
    docs = _documents([5, 9, 30, 2])
    a, b = (PackedSource(docs, 64, seed=1, rank=r) for r in (0, 1))
    for _ in range(3):
        a.next(), b.next()
    state = a.state()
    want = [s.next().tokens for s in (a, b)]
    for rank in (0, 1):
        src = PackedSource(docs, 64, seed=1, rank=rank)
        src.next()
        src.restore(state)
        assert src.drawn == 3 and torch.equal(src.next().tokens, want[rank])


def test_objective_is_the_mean_over_documents_by_themselves():
    em = _pruned()
    docs = _documents([17, 1, 30, 5])
    obj = OBJECTIVES.get("packed_recovery_ce")(em)
    loss, metrics = obj.loss(pack(docs, length=60))
    total, count = _by_document(em.model, docs)
    torch.testing.assert_close(loss, total / count, rtol=1e-5, atol=1e-5)
    assert metrics["loss"] == pytest.approx(float(loss.detach()))
    params = obj.parameters()
    got = torch.autograd.grad(loss, params)
    want = torch.autograd.grad(total / count, params)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-6)


def test_fit_trains_the_adapters():
    em = _pruned()
    docs = _documents([20, 33, 8, 40], seed=5)
    obj = OBJECTIVES.get("packed_recovery_ce")
    before, _ = obj(em).loss(pack(docs))
    fit(em, PackedSource(docs, 96, seed=2), objective="packed_recovery_ce", steps=30, lr=3e-3, warmup_steps=2,
        log_every=100)
    after, _ = obj(em).loss(pack(docs))
    assert float(after.detach()) < float(before.detach())


def test_rows_longer_than_the_models_positions():
    """The rotary tables cover the longest document, not the row: they are replaced only where a document needs it."""
    em = _pruned(tiny_model(max_position_embeddings=128))
    tables = em.model.rope_tables()
    assert tables[0].shape[0] == 128
    batch = pack(_documents([90, 1, 60, 5]), length=180)
    obj = OBJECTIVES.get("packed_recovery_ce")(em)
    loss, _ = obj.loss(batch)
    assert em.model.rope_tables()[0] is tables[0]
    assert batch.longest == 90 and batch.to("cpu").longest == 90 and pack([]).longest == 0
    batch.longest = None
    assert torch.equal(obj.loss(batch)[0], loss)
    obj.loss(pack(_documents([130])))
    assert em.model.rope_tables()[0].shape[0] == 130


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 2, 1), (64, 6, 2)])
def test_objective_on_the_kernels(cuda, head_dim, heads, kv_heads):
    """bf16 on the kernels against an fp32 copy on the CPU by document: losses to 1 % and gradients in direction and
    size."""
    from economize_b200 import ops
    from economize_b200.models.config import tiny_llama
    from economize_b200.models.llama import CausalLM, init_weights
    from economize_b200.ops.lora import LoRAWeight

    cfg = tiny_llama(hidden_size=256, num_heads=heads, num_kv_heads=kv_heads, head_dim=head_dim)
    em = _pruned(init_weights(CausalLM(cfg, torch.bfloat16, "cuda"), seed=0))
    wide = copy.deepcopy(em.model).float().cpu()
    adapters = [m for m in wide.modules() if isinstance(m, LoRAWeight)]
    for lora in adapters:
        lora._base[0] = lora._base[0].detach().float().cpu()
    docs = _documents([150, 1, 300, 33])
    obj = OBJECTIVES.get("packed_recovery_ce")(em)
    loss, _ = obj.loss(pack(docs, length=500))
    names = {id(p): n for n, p in em.model.named_parameters()}
    params = {names[id(p)]: p for p in obj.parameters()}
    got = torch.cat([t.flatten().cpu() for t in torch.autograd.grad(loss, list(params.values()))])
    total, count = _by_document(wide, docs)
    same = dict(wide.named_parameters())
    want = torch.cat([t.flatten() for t in torch.autograd.grad(total / count, [same[n] for n in params])])
    assert float(loss.detach()) == pytest.approx(float(total.detach()) / count, rel=1e-2)
    assert F.cosine_similarity(got, want, dim=0) > 0.99
    assert float(got.norm()) == pytest.approx(float(want.norm()), rel=5e-2)
    before = float(loss.detach())
    fit(em, PackedSource([d.to(cuda) for d in docs], 512, seed=2), objective="packed_recovery_ce", steps=30, lr=3e-3,
        warmup_steps=2, log_every=100)
    assert float(obj.loss(pack(docs, length=500))[0].detach()) < before
    assert ops.require().status(0) == 0
