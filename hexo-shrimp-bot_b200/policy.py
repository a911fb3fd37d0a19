"""A cell-token move policy that is fitted with the library's fit operators.

Tokens are the cells near a position's stones (``hexgraph.cell_tokens``:
empty, the mover's or the opponent's). Blocks are pre-norm: attention with a
learned bias by displacement orbit (``bucket_attention``), then a ReLU FFN,
each added to the fp32 residual stream through dropout (``dropout_add``). A
linear head gives one logit per empty cell, and ``loss`` is the negative log
probability of the played cell less an entropy bonus (``log_probs``). The
projections run through torch. ``forward`` in training goes through the
autograd ops of ``torch_ops.define_fit``; in evaluation it calls the serving
form, which keeps nothing for a backward pass.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import numpy as np
import torch
import torch.nn.functional as F
from torch import nn

from . import hexgraph, ops, torch_ops

EMPTY, OWN, OPPONENT = 0, 1, 2


@dataclass(frozen=True)
class PolicyConfig:
    h: int = 128
    blocks: int = 2
    heads: int = 4
    kv_heads: int = 4
    ffn_factor: int = 2
    dropout: float = 0.0

    def __post_init__(self) -> None:
        if self.h % self.heads or self.heads % self.kv_heads:
            raise ValueError("h must divide into heads, and heads into kv_heads groups")


class TokenBatch(NamedTuple):
    """Padded cell tokens of a batch of positions."""
    kind: torch.Tensor     # (P, L) int64: EMPTY, OWN, OPPONENT (pads EMPTY)
    coords: torch.Tensor   # (P, L, 2) int32 axial coordinates
    valid: torch.Tensor    # (P,) int32 tokens per position
    offsets: torch.Tensor  # (P + 1,) int64: each position's L logits


def token_batch(positions, radius: int = 2, device="cuda") -> TokenBatch:
    """Tokens of ``engine.Position`` objects (stone_qr, stone_owner, mover)."""
    cells = [hexgraph.cell_tokens(np.asarray(s.stone_qr), radius) for s in positions]
    p, length = len(cells), max((len(c) for c in cells), default=0)
    kind = np.zeros((p, length), dtype=np.int64)
    coords = np.zeros((p, length, 2), dtype=np.int32)
    for i, (s, c) in enumerate(zip(positions, cells)):
        coords[i, :len(c)] = c
        at = {tuple(x): j for j, x in enumerate(c.tolist())}
        for qr, owner in zip(np.asarray(s.stone_qr).tolist(), np.asarray(s.stone_owner).tolist()):
            kind[i, at[tuple(qr)]] = OWN if owner == s.mover else OPPONENT
    valid = np.array([len(c) for c in cells], dtype=np.int32)
    offsets = np.arange(p + 1, dtype=np.int64) * length
    return TokenBatch(*(torch.from_numpy(a).to(device) for a in (kind, coords, valid, offsets)))


class _Block(nn.Module):
    def __init__(self, cfg: PolicyConfig, n_buckets: int) -> None:
        super().__init__()
        d = cfg.h // cfg.heads
        self.ln_attn = nn.LayerNorm(cfg.h)
        self.qkv = nn.Linear(cfg.h, (cfg.heads + 2 * cfg.kv_heads) * d, bias=False)
        # spread, so that tokens of one kind differ by where they stand from the start
        self.bias = nn.Parameter(torch.randn(n_buckets, cfg.heads))
        self.out = nn.Linear(cfg.h, cfg.h)
        self.ln_ffn = nn.LayerNorm(cfg.h)
        self.up = nn.Linear(cfg.h, cfg.ffn_factor * cfg.h)
        self.down = nn.Linear(cfg.ffn_factor * cfg.h, cfg.h)


class CellPolicy(nn.Module):
    def __init__(self, cfg: PolicyConfig | None = None, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.cfg = cfg or PolicyConfig()
        self.dtype = dtype
        torch_ops.define_fit()
        buckets = torch.from_numpy(hexgraph.displacement_buckets())
        self.register_buffer("bucket_map", buckets, persistent=False)
        self.embed = nn.Embedding(3, self.cfg.h)
        self.blocks = nn.ModuleList(_Block(self.cfg, int(buckets.max()) + 1) for _ in range(self.cfg.blocks))
        self.ln_out = nn.LayerNorm(self.cfg.h)
        self.head = nn.Linear(self.cfg.h, 1)

    def _linear(self, layer: nn.Linear, x: torch.Tensor) -> torch.Tensor:
        b = None if layer.bias is None else layer.bias.to(self.dtype)
        return F.linear(x.to(self.dtype), layer.weight.to(self.dtype), b)

    def forward(self, batch: TokenBatch, seed: int = 0) -> torch.Tensor:
        """(P * L,) fp32 logits of the tokens, -inf for stones and pads.
        ``seed`` draws the dropout masks in training: one a step."""
        cfg = self.cfg
        p, length = batch.kind.shape
        drop = cfg.dropout if self.training else 0.0
        x = self.embed(batch.kind)
        for i, block in enumerate(self.blocks):
            qkv = self._linear(block.qkv, block.ln_attn(x)).view(p, length, cfg.heads + 2 * cfg.kv_heads,
                                                                 cfg.h // cfg.heads)
            q, k, v = qkv.permute(0, 2, 1, 3).split([cfg.heads, cfg.kv_heads, cfg.kv_heads], 1)
            where = (self.bucket_map, batch.coords, batch.valid)
            if torch.is_grad_enabled():
                att = torch.ops.mantis_b200.bucket_attention(q, k, v, block.bias, *where)[0]
            else:
                att = ops.bucket_attention(q, k, v, block.bias, *where)
            y = self._linear(block.out, att.transpose(1, 2).reshape(p, length, cfg.h))
            x = self._add(x, y, drop, seed, 2 * i)
            y = self._linear(block.down, F.relu(self._linear(block.up, block.ln_ffn(x))))
            x = self._add(x, y, drop, seed, 2 * i + 1)
        logits = self._linear(self.head, self.ln_out(x)).float()[..., 0]
        live = torch.arange(length, device=x.device) < batch.valid[:, None]
        return logits.masked_fill((batch.kind != EMPTY) | ~live, float("-inf")).reshape(-1)

    @staticmethod
    def _add(x, y, drop, seed, offset):
        return torch.ops.mantis_b200.dropout_add(x, y, drop, seed, offset) if drop > 0 else x + y

    def loss(self, batch: TokenBatch, played: torch.Tensor, entropy_bonus: float = 0.01, seed: int = 0):
        """Mean negative log probability of ``played`` (P,) int64 token ranks,
        less ``entropy_bonus`` times the mean entropy."""
        logp, entropy, *_ = torch.ops.mantis_b200.log_probs(self.forward(batch, seed), batch.offsets, played)
        return -logp.mean() - entropy_bonus * entropy.mean()

    @torch.no_grad()
    def report(self, batch: TokenBatch, top: int = 5):
        """``ops.LogProbs`` of a batch: entropies and the ``top`` likeliest cells."""
        return ops.log_probs(self.forward(batch), batch.offsets, None, top=top)
