"""CPU: when tree attention leaves a (sequence, kv head) pair whole, seen by the workspace (partial states only where it does not)."""
import ctypes as C

import pytest

from mi355q import _lib as L


def size(past, batch, heads, kv_heads, draft, kv=L.BF16):
    p = L.TreeAttentionParams()
    p.batch, p.num_heads, p.num_kv_heads, p.head_size = batch, heads, kv_heads, 128
    p.num_tokens, p.max_draft_length, p.max_past_length, p.mask_words = batch * draft, draft, past, (draft + 31) // 32
    p.max_blocks_per_seq, p.tokens_per_block, p.act_type, p.kv_type = 128, 64, L.BF16, kv
    n = L.lib().mi355q_tree_attention_workspace_size(C.byref(p))
    assert n > 0
    return n


@pytest.mark.parametrize("batch,heads,kv_heads,draft,limit", [(16, 64, 8, 64, 4096), (8, 32, 32, 16, 2048), (4, 32, 32, 16, 1024), (128, 32, 8, 4, 4096)])
def test_the_history_decides(batch, heads, kv_heads, draft, limit):
    # the nodes on top of a history of the limit do not cut it, one token more does
    least = size(64, batch, heads, kv_heads, draft)
    assert size(limit, batch, heads, kv_heads, draft) == least
    assert size(limit + 1, batch, heads, kv_heads, draft) > least


def test_few_workgroups_split_from_512_keys_on():
    least = size(64, 1, 32, 8, 8)
    assert size(504, 1, 32, 8, 8) == least and size(505, 1, 32, 8, 8) > least
