"""The plan that the grouped forward runs for its sizes, asked on the CPU.

Causal work takes the plan of the candidate's own forward (lists over groups of heads, mode 2,
from two items per multiprocessor on) although it is given no workspace; unmasked work and single
queries are folded to one head per key/value head and split where a workspace is given.
"""

from __future__ import annotations

import pytest

WAVES, TAIL, TABLE = 0, 1, 2


@pytest.mark.parametrize("batch,heads,kv_heads,seq", [(2, 16, 4, 4096), (2, 16, 16, 8192), (8, 16, 16, 2048),
                                                      (4, 32, 8, 4001), (148, 2, 1, 256)])
def test_causal_work_takes_the_lists_without_a_workspace(b200, batch, heads, kv_heads, seq):
    for split in (False, True):
        got = b200.grouped_plan(batch, heads, kv_heads, seq, seq, True, split=split)
        assert got[0] == TABLE
        assert got == b200.schedule_units(batch * heads, seq, seq, True, split=True, max_units=4096)[:4]


def test_causal_lengths_are_aligned_at_their_ends(b200):
    for seq_q, seq_kv in ((2048, 5000), (5000, 2048)):
        got = b200.grouped_plan(2, 64, 8, seq_q, seq_kv, True, split=False)
        want = b200.schedule_units(128, seq_q, seq_kv, True, q_pos0=seq_kv - seq_q, max_units=4096)
        assert got[0] == TABLE and got == want[:4]


def test_few_or_many_causal_items_stay_in_waves(b200):
    assert b200.grouped_plan(1, 16, 4, 2048, 2048, True)[0] == WAVES          # 128 items
    assert b200.grouped_plan(8, 128, 8, 4096, 4096, True)[0] == WAVES         # 16384 items, past the lists' room


def test_unmasked_work_is_folded_and_split_only_with_a_workspace(b200):
    for causal, seq_q, seq_kv in ((False, 1001, 9003), (True, 1, 30000)):
        want = b200.schedule_units(2, 12 * seq_q, seq_kv, False, max_units=4096)
        assert b200.grouped_plan(1, 24, 2, seq_q, seq_kv, causal, split=True) == want[:4]
        assert want[0] == TAIL
        assert b200.grouped_plan(1, 24, 2, seq_q, seq_kv, causal, split=False)[0] == WAVES


def test_refusals(b200):
    for sizes in ((1, 3, 2, 8, 8), (1, 2, 0, 8, 8), (-1, 2, 1, 8, 8), (1, 2, 1, -8, 8), (1, 2, 1, 8, -8),
                  (2**30, 4, 4, 8, 8), (1, 1, 1, 2**31 - 1, 2**31 - 1)):
        with pytest.raises(b200.B200AttentionError):
            b200.grouped_plan(*sizes, True)
    with pytest.raises(b200.B200AttentionError):
        b200.grouped_plan(1, 2, 1, 8, 8, True, sm_count=0)
    for empty in ((0, 2, 1, 8, 8), (1, 2, 1, 0, 8), (1, 2, 1, 8, 0)):
        assert b200.grouped_plan(*empty, True)[0] == WAVES
