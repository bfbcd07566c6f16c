"""The streamed tiles of the gradient's causal items (attn_bwd.cuh, Items::next), on the CPU.

dK/dV streams the query tiles from t0 = max(0, 128 tile - offset) // 128 on, dQ the first
n = min(nkv, ceil(max(end + offset, 0) / 128)) key tiles, where offset = seq_kv - seq_q aligns the
sequences at their ends.  Both have to cover exactly the pairs of tiles that hold a visible pair."""

from __future__ import annotations

import pytest

TILE = 128


def tiles(rows):
    return -(-rows // TILE)


@pytest.mark.parametrize("seq_q,seq_kv", [(1, 1), (1, 700), (5, 1), (127, 128), (128, 129), (129, 257), (300, 170),
                                          (257, 128), (1000, 1000), (700, 129), (129, 1001), (640, 1)])
def test_items_stream_the_tiles_that_hold_visible_pairs(seq_q, seq_kv):
    offset = seq_kv - seq_q
    nq, nkv = tiles(seq_q), tiles(seq_kv)
    seen = set()
    for i in range(seq_q):
        last = min(i + offset, seq_kv - 1)
        seen |= {(i // TILE, j) for j in range(last // TILE + 1)} if last >= 0 else set()
    kv_pass = set()
    for tile in range(nkv):
        t0 = max(0, tile * TILE - offset) >> 7
        assert t0 < nq  # the last query sees every key: no key tile is without a query tile
        kv_pass |= {(t, tile) for t in range(t0, nq)}
    q_pass = set()
    for tile in range(nq):
        end = min(tile * TILE + TILE, seq_q) + offset
        q_pass |= {(tile, j) for j in range(min(nkv, (max(end, 0) + TILE - 1) >> 7))}
    assert kv_pass == q_pass == seen
