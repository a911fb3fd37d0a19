"""Cell-token graphs of the isolated-op workloads: the hex message-passing op
(neighbour table over cell tokens) and the axial-bias attention op (token
coordinates and valid lengths). Bucket maps of relative offsets for the
bucketed-bias attention.

A position's cell tokens are its occupied cells plus the empty cells within
hex distance ``radius`` of a stone, in ascending (q, r) order. Neighbour slot
order follows the reference adjacency walk (builder.py:458-471): for each
engine axis Q, R, QR (builder.py:32) the step -1 then the step +1, so slot
2 * axis + (sign > 0). A slot holds the global token row of that neighbour,
or -1 when the neighbour cell is not a token. Rows past a position's token
count (padding) have every slot -1.
"""

from __future__ import annotations

import numpy as np

from .engine import random_positions
from .vocab import AXES, ORBIT48_CLASSES, ORBIT48_TABLE, ORBIT_SPAN

SLOTS = 6
# (6, 2) unit steps in slot order: axis 0 (-, +), axis 1 (-, +), axis 2 (-, +)
SLOT_STEPS = np.stack([s * AXES[a] for a in range(3) for s in (-1, 1)]).astype(np.int64)


def _pack(qr: np.ndarray) -> np.ndarray:
    """Order-preserving int64 key of (q, r) pairs (|q|, |r| < 2**20)."""
    return (qr[..., 0] + (1 << 20)) * (1 << 21) + (qr[..., 1] + (1 << 20))


def cell_tokens(stone_qr: np.ndarray, radius: int = 2) -> np.ndarray:
    """(n, 2) int64 token coordinates in ascending (q, r): the stones and
    every cell within hex distance ``radius`` of one."""
    offs = np.array([(dq, dr) for dq in range(-radius, radius + 1) for dr in range(-radius, radius + 1)
                     if max(abs(dq), abs(dr), abs(dq + dr)) <= radius], dtype=np.int64)
    cells = (stone_qr[:, None, :] + offs[None, :, :]).reshape(-1, 2)
    keys = np.unique(_pack(cells))  # sorted, unique
    q = keys // (1 << 21) - (1 << 20)
    r = keys % (1 << 21) - (1 << 20)
    return np.stack([q, r], 1)


def neighbour_table(tokens: np.ndarray, length: int, row0: int = 0) -> np.ndarray:
    """(length, 6) int32 neighbour rows for the first ``length`` tokens (the
    rest padding), offset by ``row0``."""
    n = min(len(tokens), length)
    kept = tokens[:n]
    keys = _pack(kept)  # ascending because the tokens are
    out = np.full((length, SLOTS), -1, dtype=np.int32)
    if n:
        nb = _pack(kept[:, None, :] + SLOT_STEPS[None, :, :])  # (n, 6)
        pos = np.searchsorted(keys, nb)
        hit = (pos < n) & (keys[np.minimum(pos, n - 1)] == nb)
        out[:n] = np.where(hit, pos + row0, -1).astype(np.int32)
    return out


def message_graph(n_pos: int, length: int = 256, lo: int = 40, hi: int = 200, seed: int = 0):
    """The message-passing workload's table: ``n_pos`` seeded random-play
    positions (``lo``-``hi`` stones), ``length`` token rows each (tokens at
    hex distance <= 2, truncated or padded). Returns (nbr (n_pos*length, 6)
    int32, tokens per position)."""
    specs = random_positions(n_pos, lo, hi, seed=seed)
    tables, counts = [], []
    for i, s in enumerate(specs):
        tok = cell_tokens(s.stone_qr, 2)
        counts.append(min(len(tok), length))
        tables.append(neighbour_table(tok, length, i * length))
    return np.concatenate(tables), np.asarray(counts)


def attention_layout(n_pos: int, length: int = 256, lo: int = 10, hi: int = 40, seed: int = 0,
                     min_valid: int = 32):
    """The axial-attention workload's token coordinates and valid lengths:
    per position the first ``length`` tokens in ascending (q, r) of a seeded
    random-play position of ``lo``-``hi`` stones (token radius grown from 2
    until there are ``length`` of them), and a valid length uniform in
    [``min_valid``, ``length``]. Returns (coords (n_pos, length, 2) int32,
    valid (n_pos,) int32)."""
    specs = random_positions(n_pos, lo, hi, seed=seed)
    rng = np.random.default_rng(seed + 1)
    coords = np.zeros((n_pos, length, 2), dtype=np.int32)
    for i, s in enumerate(specs):
        radius = 2
        tok = cell_tokens(s.stone_qr, radius)
        while len(tok) < length:
            radius += 1
            tok = cell_tokens(s.stone_qr, radius)
        coords[i] = tok[:length]
    valid = rng.integers(min_valid, length + 1, size=n_pos).astype(np.int32)
    return coords, valid


def displacement_buckets() -> np.ndarray:
    """(27, 27) int32 bucket map of axial offsets for the bucketed-bias
    attention: the 48 displacement orbits within distance 12, 48 for the token
    itself, 49 for every farther offset (the map's rim)."""
    out = np.full((2 * ORBIT_SPAN + 3,) * 2, ORBIT48_CLASSES + 1, dtype=np.int32)
    inner = np.where(ORBIT48_TABLE >= 0, ORBIT48_TABLE, ORBIT48_CLASSES + 1)
    inner[ORBIT_SPAN, ORBIT_SPAN] = ORBIT48_CLASSES
    out[1:-1, 1:-1] = inner
    return out


def line_buckets(n_buckets: int = 32, max_distance: int = 128, causal: bool = False) -> np.ndarray:
    """(2 max_distance + 1, 1) int32 bucket map of signed distances along a
    line of tokens (coordinates (t, 0)) for the bucketed-bias attention: on
    each side half the buckets for exact distances, then log-spaced ones up to
    ``max_distance``. ``causal`` excludes later keys (-1) and gives the earlier
    ones every bucket. The log-spaced scheme is that of Raffel et al. (2020,
    relative position buckets)."""
    side = n_buckets if causal else n_buckets // 2
    exact = side // 2
    if exact < 1 or max_distance <= exact or (not causal and n_buckets % 2):
        raise ValueError(f"need an even n_buckets >= 4 and max_distance > {exact}, got ({n_buckets}, {max_distance})")
    d = np.arange(-max_distance, max_distance + 1)
    a = np.abs(d)
    far = exact + np.floor(np.log(np.maximum(a, 1) / exact) / np.log(max_distance / exact) * (side - exact))
    b = np.where(a < exact, a, np.minimum(far, side - 1)).astype(np.int32)
    b = np.where(d > 0, -1 if causal else b + side, b)
    return np.ascontiguousarray(b[:, None], dtype=np.int32)
