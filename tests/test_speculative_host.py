"""CPU tests of the speculative-decoding entry points: what they refuse (before anything is launched), with which status and
words, the workspace sizes, and the host side of the block manager."""
import ctypes as C

import pytest
import torch

from mi355q import _lib as L
from mi355q import functional as F
from mi355q.kv_cache_manager import DeviceBlocksManager

FAKE = 4096  # an address that is never read: every call here is refused first
INVALID, UNSUPPORTED = -1, -2


def tree_params(**kw):
    p = L.TreeAttentionParams()
    for name in ("qkv", "out", "past_lengths", "draft_offsets", "tree_mask", "block_pointers", "workspace"):
        setattr(p, name, FAKE)
    p.workspace_bytes = 1 << 40
    p.batch, p.num_heads, p.num_kv_heads, p.head_size = 2, 8, 2, 128
    p.num_tokens, p.max_draft_length, p.max_past_length, p.mask_words = 32, 16, 1000, 1
    p.max_blocks_per_seq, p.tokens_per_block = 32, 64
    p.act_type = p.kv_type = L.BF16
    p.rotary_embedding_base, p.q_scaling = 10000.0, 1.0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def refused(fn, params, status, words):
    rc = getattr(L.lib(), fn)(C.byref(params), None)
    text = L.lib().mi355q_last_error().decode()
    assert rc == status and words in text, (rc, text)


ROPE = dict(position_embedding_type=2, rotary_embedding_dim=128)


@pytest.mark.parametrize("kw,status,words", [
    (dict(act_type=L.FLOAT), INVALID, "act_type"), (dict(kv_type=L.HALF), INVALID, "kv cache type"),
    (dict(kv_type=L.FLOAT), INVALID, "kv cache type"), (dict(batch=-1), INVALID, "batch"), (dict(batch=70000), INVALID, "batch"),
    (dict(num_kv_heads=3), INVALID, "heads"), (dict(num_kv_heads=0), INVALID, "heads"), (dict(head_size=100), INVALID, "head_size"),
    (dict(head_size=264), INVALID, "head_size"), (dict(head_size=72, kv_type=L.INT8), INVALID, "head_size"),
    (dict(max_draft_length=1025), INVALID, "max_draft_length"), (dict(num_tokens=-1), INVALID, "num_tokens"),
    (dict(tokens_per_block=48), INVALID, "power of 2"), (dict(tokens_per_block=0), INVALID, "power of 2"),
    (dict(tokens_per_block=8), UNSUPPORTED, "not built"), (dict(max_blocks_per_seq=0), INVALID, "max_blocks_per_seq"),
    (dict(max_past_length=-1), INVALID, "max_past_length"), (dict(max_past_length=2049), INVALID, "exceeds the block table"),
    (dict(mask_words=0), INVALID, "tree_mask"), (dict(max_draft_length=33), INVALID, "tree_mask"),
    (dict(qkv=None), INVALID, "null"), (dict(tree_mask=None), INVALID, "null"), (dict(block_pointers=None), INVALID, "null"),
    (dict(qkv=FAKE + 8), INVALID, "16-byte"), (dict(out=FAKE + 2), INVALID, "16-byte"), (dict(workspace=FAKE + 4), INVALID, "16-byte"),
    (dict(qkv_stride=1528), INVALID, "qkv_stride"), (dict(qkv_stride=1540), INVALID, "qkv_stride"),
    (dict(kv_type=L.INT8), INVALID, "kv_scale"), (dict(kv_type=L.FP8, kv_scale_quant_orig=FAKE), INVALID, "kv_scale"),
    (dict(position_embedding_type=3), UNSUPPORTED, "position_embedding_type"), (dict(position_embedding_type=-1), UNSUPPORTED, "position"),
    (dict(position_embedding_type=2), INVALID, "rotary_embedding_dim"), (dict(ROPE, rotary_embedding_dim=130), INVALID, "rotary"),
    (dict(ROPE, rotary_embedding_dim=63), INVALID, "rotary"), (dict(ROPE, rotary_embedding_base=0.0), INVALID, "base"),
    (dict(ROPE, rotary_embedding_scale_type=3), INVALID, "scale_type"), (dict(ROPE, rotary_embedding_scale_type=1), INVALID, "scale"),
    (dict(ROPE, rotary_embedding_scale_type=2, rotary_embedding_scale=2.0), INVALID, "dynamic"),
    (dict(multi_block_mode=-1), INVALID, "multi_block_mode"), (dict(workspace=None), INVALID, "workspace too small"),
    (dict(workspace_bytes=1000), INVALID, "workspace too small"),
    # more than the grids hold
    (dict(batch=65535, num_heads=1024, num_kv_heads=512, num_tokens=65535), INVALID, "row tiles"),
    (dict(batch=65535, multi_block_mode=4), INVALID, "pairs in parts"),
    (dict(batch=65535, num_heads=2048, num_kv_heads=1024, max_past_length=2048), INVALID, "kv heads")])
def test_tree_attention_refusals(kw, status, words):
    refused("mi355q_tree_attention", tree_params(**kw), status, words)


def test_tree_attention_workspace():
    size = lambda **kw: L.lib().mi355q_tree_attention_workspace_size(C.byref(tree_params(**kw)))
    q = 32 * 8 * 128 * 2
    # short histories: the queries (two parts) and the sequences' records; long ones: the partial states too
    assert 2 * q <= size(max_past_length=100) < 2 * q + 4096
    assert size(max_past_length=2048) > size(max_past_length=100)
    # fp16 products for a bf16 result over an 8-bit cache: one part
    assert size(max_past_length=100, kv_type=L.INT8) < 2 * q
    assert size(batch=0, num_tokens=0, max_past_length=100) < 4096
    assert size(head_size=100) == 0 and b"head_size" in L.lib().mi355q_last_error()
    assert L.lib().mi355q_tree_attention_workspace_size(None) == 0


def test_empty_calls_do_nothing():
    for kw in (dict(batch=0), dict(num_tokens=0), dict(max_draft_length=0)):
        assert L.lib().mi355q_tree_attention(C.byref(tree_params(qkv=None, **kw)), None) == 0
    assert L.lib().mi355q_kv_block_tables(C.byref(table_params(batch=0, past_lengths=None)), None) == 0
    assert L.lib().mi355q_draft_tree_accept(C.byref(L.DraftTreeAcceptParams(batch=0, max_path=1)), None) == 0
    assert L.lib().mi355q_kv_commit_path(C.byref(commit_params(batch=0, new_lengths=None)), None) == 0


def table_params(**kw):
    p = L.KvBlockTablesParams()
    for i, name in enumerate(("past_lengths", "new_lengths", "block_table", "block_counts", "block_counts_out", "free_blocks", "free_state",
                              "free_state_out", "pool_bases", "block_pointers", "token_offsets", "slot_map", "status", "workspace")):
        setattr(p, name, FAKE * (i + 1))
    p.workspace_bytes, p.block_bytes = 1 << 20, 4096
    p.batch, p.max_blocks_per_seq, p.num_blocks, p.num_pools, p.num_tokens, p.tokens_per_block = 4, 8, 16, 2, 10, 64
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,words", [
    (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(max_blocks_per_seq=0), "max_blocks_per_seq"), (dict(num_blocks=0), "num_blocks"),
    (dict(num_pools=-1), "num_pools"), (dict(num_tokens=-1), "num_tokens"), (dict(block_bytes=0), "block_bytes"),
    (dict(tokens_per_block=3), "power of 2"), (dict(past_lengths=None), "null"), (dict(free_state=None), "null"), (dict(status=None), "null"),
    (dict(pool_bases=None), "null"), (dict(block_pointers=None), "null"), (dict(slot_map=None), "null"), (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=63), "workspace"), (dict(workspace=FAKE + 8), "workspace"), (dict(block_counts_out=FAKE + 4), "overlaps"),
    (dict(token_offsets=FAKE + 8), "overlaps"), (dict(block_counts_out=4 * FAKE + 4), "overlaps")])
def test_block_tables_refusals(kw, words):
    refused("mi355q_kv_block_tables", table_params(**kw), INVALID, words)


@pytest.mark.parametrize("kw,words", [(dict(batch=-1), "batch"), (dict(max_path=0), "max_path"), (dict(num_tokens=-5), "num_tokens"),
                                      (dict(parents=None), "null"), (dict(accept_path=None), "null"), (dict(draft_offsets=None), "null")])
def test_accept_refusals(kw, words):
    p = L.DraftTreeAcceptParams(*[FAKE] * 7, 2, 8, 4)
    for k, v in kw.items():
        setattr(p, k, v)
    refused("mi355q_draft_tree_accept", p, INVALID, words)


def commit_params(**kw):
    p = L.KvCommitPathParams(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, 2, 3, 8, 64, 2, 128, 4, L.BF16)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,words", [
    (dict(batch=-1), "batch"), (dict(num_pools=0), "num_pools"), (dict(max_path=0), "max_path"), (dict(num_kv_heads=0), "num_kv_heads"),
    (dict(max_blocks_per_seq=0), "max_blocks_per_seq"), (dict(kv_type=L.FLOAT), "kv cache type"), (dict(head_size=12), "head_size"),
    (dict(tokens_per_block=24), "power of 2"), (dict(block_pointers=None), "null"), (dict(accept_counts=None), "null"),
    (dict(new_lengths=2 * FAKE), "overlaps"), (dict(new_lengths=3 * FAKE + 16), "overlaps"), (dict(new_lengths=4 * FAKE + 4), "overlaps")])
def test_commit_refusals(kw, words):
    refused("mi355q_kv_commit_path", commit_params(**kw), INVALID, words)


def test_null_params():
    for fn in ("mi355q_tree_attention", "mi355q_kv_block_tables", "mi355q_draft_tree_accept", "mi355q_kv_commit_path"):
        assert getattr(L.lib(), fn)(None, None) == INVALID and b"null" in L.lib().mi355q_last_error()


def test_python_refusals():
    with pytest.raises(ValueError, match="dtype"):
        F.TreeAttention(num_heads=4, num_kv_heads=4, head_size=64, dtype=torch.float32)
    with pytest.raises(ValueError, match="kv_dtype"):
        F.TreeAttention(num_heads=4, num_kv_heads=4, head_size=64, dtype=torch.float16, kv_dtype=torch.bfloat16)
    op = F.TreeAttention(num_heads=4, num_kv_heads=4, head_size=100, dtype=torch.float16)
    with pytest.raises(L.Mi355qError, match="head_size"):
        op.workspace_size(1, 4, 4, 100, 8)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        op(torch.zeros(2, 1200, dtype=torch.float16), i, i, i[None], i.long()[None, None], max_draft_length=1, max_past_length=1)
    with pytest.raises(ValueError, match="on the GPU"):
        F.draft_tree_accept(i, i, i, i, 3)
    with pytest.raises(ValueError, match="on the GPU"):
        F.kv_commit_path(torch.zeros(1, 2, 2, 4, dtype=torch.int64), i, i[None], i, num_kv_heads=1, head_size=8, tokens_per_block=4,
                         kv_dtype=torch.float16)
    pools = [torch.zeros(2 * 6 * 64, dtype=torch.float16) for _ in range(2)]
    mgr = DeviceBlocksManager(pools, 6, 4, 3, batch_size=2)
    assert mgr.block_bytes == 128 and mgr.pool_bases.tolist() == [p.data_ptr() for p in pools] and mgr.free_blocks() == 6
    with pytest.raises(ValueError, match="on the GPU"):
        mgr.step(i, i, 2)
    with pytest.raises(ValueError, match="one block size"):
        DeviceBlocksManager([pools[0], pools[1][:-64]], 6, 4, 3, batch_size=2)
