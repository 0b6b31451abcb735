"""The speculative-decoding operators on a batch without requests."""
import pytest
import torch

from mi355q import functional as F

pytestmark = pytest.mark.gpu
I32 = torch.int32


def test_tables_of_no_requests(cuda):
    # offsets, slots and the ring's state as for any other batch in which nobody asks for anything
    t = lambda *shape: torch.full(shape, 77, dtype=I32, device=cuda)
    for tokens in (0, 5):
        state, out = torch.tensor([3, 9], dtype=I32, device=cuda), t(2)
        ptr, offsets, slots, status = F.kv_block_tables(t(0), t(0), t(0, 4), t(0), t(16), state, torch.zeros(2, dtype=torch.int64, device=cuda),
                                                        block_bytes=64, tokens_per_block=16, num_tokens=tokens, free_state_out=out)
        assert ptr.shape == (2, 0, 2, 4) and status.shape == (0,)
        assert offsets.tolist() == [0] and slots.tolist() == [-1] * tokens and out.tolist() == [3, 9] == state.tolist()
        F.kv_block_tables(t(0), t(0), t(0, 4), t(0), t(16), state, torch.zeros(2, dtype=torch.int64, device=cuda), block_bytes=64,
                          tokens_per_block=16, num_tokens=tokens)
        assert state.tolist() == [3, 9]


def test_path_and_commit_of_no_requests(cuda):
    e = torch.zeros(0, dtype=I32, device=cuda)
    path, counts, said = F.draft_tree_accept(e, e, e, torch.zeros(1, dtype=I32, device=cuda), 4)
    assert path.shape == (0, 4) == said.shape and counts.shape == (0,)
    ptr = torch.zeros(3, 0, 2, 4, dtype=torch.int64, device=cuda)
    assert F.kv_commit_path(ptr, e, path, counts, num_kv_heads=2, head_size=64, tokens_per_block=16, kv_dtype=torch.float16).shape == (0,)
