"""Training on packed documents: rows of whole documents one after another, without padding between them, and the
recovery objective on such rows (the packed form of ``recovery_ce``).

A packed step attends each document by itself (:func:`~economize_b200.ops.packed_attention`), counts rotary positions
from each document's first token, and takes its loss from :func:`~economize_b200.ops.linear_cross_entropy`, which
never holds the ``[tokens, vocabulary]`` logits. It runs in the model's own dtype on CUDA (fp32 on CPU)::

    source = PackedSource(documents, tokens_per_batch=8192)
    fit(model, source, objective="packed_recovery_ce", steps=200)
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch

from .. import ops
from ..errors import ConfigError
from .objective import OBJECTIVES, RecoveryCE, packed_block, torch_block

__all__ = ["PackedBatch", "PackedRecoveryCE", "PackedSource", "pack"]

IGNORE = -100


@dataclass
class PackedBatch:
    """Documents one after another: ``tokens [T]``; document ``i`` is tokens ``cu_seqlens[i]`` to ``cu_seqlens[i + 1]``
    (int32 ``[B + 1]``), what follows the last one is padding. ``positions [T]`` count within a document; ``targets
    [T]`` are each position's next token in its document, ``-100`` at a document's last token and in the padding.
    ``longest``: the longest document's tokens (known on the host; None: read from ``positions``)."""

    tokens: torch.Tensor
    cu_seqlens: torch.Tensor
    positions: torch.Tensor
    targets: torch.Tensor
    longest: int | None = None

    def to(self, device) -> PackedBatch:
        return PackedBatch(*(t.to(device) for t in (self.tokens, self.cu_seqlens, self.positions, self.targets)),
                           self.longest)


def pack(documents: Sequence[torch.Tensor], length: int | None = None) -> PackedBatch:
    """The documents (1-D token tensors) as one packed row, padded with token 0 up to ``length``."""
    lens = [int(d.numel()) for d in documents]
    total = sum(lens)
    if length is not None and total > length:
        raise ConfigError(f"{total} tokens do not fit a row of {length}")
    pad = 0 if length is None else length - total
    device = documents[0].device if lens else torch.device("cpu")
    tokens = torch.cat([*(d.reshape(-1).long() for d in documents), torch.zeros(pad, dtype=torch.long, device=device)])
    edges = torch.tensor([0, *lens]).cumsum(0)
    positions = torch.cat([*(torch.arange(n) for n in lens), torch.zeros(pad, dtype=torch.long)])
    targets = torch.cat([tokens[1:], tokens[:1]])
    targets[(edges[1:] - 1)[torch.tensor(lens, dtype=torch.long) > 0].to(device)] = IGNORE
    targets[total:] = IGNORE
    return PackedBatch(tokens, edges.to(torch.int32).to(device), positions.to(device), targets, max(lens, default=0))


class PackedSource:
    """Packed rows of random documents, reproducible from ``seed`` and resumable. Documents are drawn until the row of
    ``tokens_per_batch`` is full; the last one is cut to fit. Every data-parallel rank draws rows of its own: ``rank`` is
    the process's in the default group (0 without one); equal ranks draw equal rows, for a stream that is sharded
    otherwise (:class:`~economize_b200.train.data.ShardedSource`)."""

    def __init__(self, documents: Sequence[torch.Tensor], tokens_per_batch: int, seed: int = 0,
                 rank: int | None = None) -> None:
        self.documents = [d.reshape(-1) for d in documents if d.numel() > 0]
        if not self.documents:
            raise ConfigError("PackedSource needs at least one document that is not empty")
        if tokens_per_batch < 1:
            raise ConfigError(f"tokens_per_batch must be positive, got {tokens_per_batch}")
        self.tokens_per_batch = tokens_per_batch
        if rank is None:
            on = torch.distributed.is_available() and torch.distributed.is_initialized()
            rank = torch.distributed.get_rank() if on else 0
        self.rank = rank
        self.seed = seed + 1000003 * rank  # as fit seeds the ranks' batches of a token tensor
        self.gen = torch.Generator().manual_seed(self.seed)
        self.drawn = 0

    def _draw(self) -> list[torch.Tensor]:
        picked, left = [], self.tokens_per_batch
        while left > 0:
            doc = self.documents[int(torch.randint(0, len(self.documents), (1,), generator=self.gen))]
            picked.append(doc[:left])
            left -= picked[-1].numel()
        self.drawn += 1
        return picked

    def next(self) -> PackedBatch:
        return pack(self._draw())

    def state(self) -> dict:
        return {"drawn": self.drawn, "gen": self.gen.get_state(), "rank": self.rank}

    def restore(self, state: dict) -> None:
        """Continue behind ``state``; a checkpoint holds one rank's, from which the others draw as many rows again."""
        if state.get("rank", self.rank) == self.rank:
            self.drawn = state["drawn"]
            self.gen.set_state(state["gen"])
            return
        self.drawn = 0
        self.gen.manual_seed(self.seed)
        while self.drawn < state["drawn"]:
            self._draw()


@OBJECTIVES.register("packed_recovery_ce")
class PackedRecoveryCE(RecoveryCE):
    """Next-token cross-entropy of a pruned target through its recovery adapters over packed documents
    (:class:`PackedBatch`). Targets with scaled residuals, attention or logits (Granite) are trained too."""

    name = "packed_recovery_ce"

    def __init__(self, model) -> None:
        super().__init__(model)
        if model.model.config.final_softcap:
            raise ConfigError("packed_recovery_ce does not model a soft-cap on the final logits")

    def loss(self, batch: PackedBatch) -> tuple[torch.Tensor, dict[str, float]]:
        from ..ops.reference import rmsnorm

        target = self.model.model
        c = target.config
        head = target.head_weight.detach()
        # positions count within documents: a row of many does not need the tables of a sequence as long
        longest = int(batch.positions.max()) + 1 if batch.longest is None else batch.longest
        batch = batch.to(head.device)
        dtype = head.dtype if head.is_cuda else torch.float32
        cos, sin = target.rope_tables(longest)
        cos, sin = cos[batch.positions], sin[batch.positions]
        h = target.embed_tokens(batch.tokens[None]).to(dtype)
        if c.residual_multiplier == 1.0 and c.attention_multiplier is None:
            for layer in target.layers:
                h = torch_block(layer, h, c, cos, sin, cu_seqlens=batch.cu_seqlens)
            h = rmsnorm(h, target.norm.to(dtype), c.rms_norm_eps)[0][0]
        else:
            branch = None
            for layer in target.layers:
                branch, h = packed_block(layer, branch, h, c, cos, sin, batch.cu_seqlens)
            h = ops.block_norm(branch, h, target.norm.to(dtype), scale=c.residual_multiplier, eps=c.rms_norm_eps)[0][0]
        loss = ops.linear_cross_entropy(h, head.to(dtype), batch.targets, ignore_index=IGNORE,
                                        logit_scale=1.0 / c.logits_scaling)
        return loss, {"loss": float(loss.detach())}
