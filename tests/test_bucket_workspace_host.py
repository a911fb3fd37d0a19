"""The workspace of bucketed attention's backward pass, without a GPU: what it
asks for over the sharing's thresholds, and the limit on dQ's parts."""

from __future__ import annotations

import ctypes

import pytest

from golden_io import mb

_lib = mb._lib
pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")
BF16, F32 = 1, 0
GIB = 1 << 30


def _bytes(dtype, n_pos, heads, kv_heads, dim, length, buckets):
    need = ctypes.c_int64(0)
    _lib.call("mb_bucket_attention_workspace", dtype, n_pos, heads, kv_heads, dim, length, buckets, ctypes.byref(need))
    return need.value


def _part(n_pos, heads, length, dim):
    """Bytes of one part of dQ: fp32, of q's size."""
    return 4 * n_pos * heads * length * dim


@pytest.fixture
def limit():
    yield mb.ops.bucket_attention_limit_parts
    mb.ops.bucket_attention_limit_parts(0)


def test_parts_on_both_sides_of_whole_items():
    """148 positions of 4 key / value heads are shared by whole items (one sum);
    one position fewer keeps parts of key tiles and their running sum, within
    16 GiB, not 23."""
    size = 16, 4, 128, 4096, 32
    whole, tiles = _bytes(BF16, 148, *size), _bytes(BF16, 147, *size)
    assert _part(148, 16, 4096, 128) <= whole <= 1.05 * _part(148, 16, 4096, 128)
    assert 2 * _part(147, 16, 4096, 128) <= tiles <= 16.5 * GIB
    # sizes whose four parts fit keep four and the sum; 80 items x 4 tiles are
    # fewer than 592 CTAs, so two share a tile's queries, each with parts of dK and dV
    small, own = _bytes(BF16, 20, *size), 5 * _part(20, 16, 4096, 128) + 2 * 2 * _part(20, 4, 4096, 128)
    assert own <= small <= 1.05 * own
    # and where the running sum and one part pass 16 GiB, these two (588 items: two share a tile's queries)
    most, own = _bytes(BF16, 147, 64, 4, 128, 4096, 32), 2 * _part(147, 64, 4096, 128) + 4 * _part(147, 4, 4096, 128)
    assert own <= most <= 1.05 * own


def test_limit_on_parts(limit):
    """The limit counts parts (the sum beside them is kept in any case), is at
    least one, and 0 restores the default; the wrapper's sizes follow it."""
    size = BF16, 2, 4, 4, 64, 1300, 32  # eleven key tiles
    part = _part(2, 4, 1300, 64)
    wrapped = lambda: mb.ops._bucket_workspace(*size)  # noqa: E731
    default = _bytes(*size)
    assert wrapped() == default and default >= 11 * part
    rest = default - 11 * part  # no running sum: one launch takes every tile
    for parts in (1, 2, 5, 10):
        limit(parts * part)
        assert parts + 1 <= _bytes(*size) / part
        assert wrapped() == _bytes(*size)
    limit(1)
    assert _bytes(*size) >= 2 * part
    limit(11 * part)
    assert _bytes(*size) == 11 * part + rest
    limit(0)
    assert wrapped() == default
    with pytest.raises(ValueError, match="negative"):
        limit(-1)


def test_bias_sums_of_the_path_that_runs():
    """The tensor cores keep bias sums for 296 CTAs, not one for each of 70,000
    query tiles; the CUDA cores, which keep no parts, have theirs in the same place."""
    size = 10_000, 16, 16, 32, 400
    parts, delta = _part(10_000, 16, 400, 32), 4 * 10_000 * 16 * 400
    assert _bytes(BF16, *size, 128) == parts + delta + 4 * 296 * 16 * 128
    sums = 4 * 10_000 * 7 * 16 * 128
    assert _bytes(F32, *size, 128) == delta + sums
    # one key tile of a bf16 batch has no parts: the CUDA cores' sums decide
    assert _bytes(BF16, 10_000, 16, 16, 32, 40, 128) == 4 * 10_000 * 16 * (40 + 128)
