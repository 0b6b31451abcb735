"""Block tables, accepted paths and the cache commit on the device against their definitions (whole numbers: equal), and the
speculative step as a whole: tables -> tree attention in every layer -> accepted path -> commit -> the next step."""
import numpy as np
import pytest
import torch

from mi355q import functional as F
from mi355q.kv_cache_manager import BlocksManager, DeviceBlocksManager, GenerationSequence
import speculative_reference as R
from speculative_reference import TreeCase, random_tree

pytestmark = pytest.mark.gpu
I32 = torch.int32


def dev_t(a, dev, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).to(dev)


# ------------------------------------------------------------------------------------------------ block tables
def table_case(B, max_blocks, tpb, seed, admit=0.2, release=0.2, spare=1.0, new_hi=None):
    rs = np.random.RandomState(seed)
    past = rs.randint(0, max_blocks * tpb + 1, B)
    new = rs.randint(0, (new_hi or 2 * tpb) + 1, B)
    u = rs.random_sample(B)
    past[u < admit] = 0
    new[u < admit] = rs.randint(0, max_blocks * tpb + 1, int((u < admit).sum()))
    new[u > 1 - release] = -1 - rs.randint(0, 3)
    held = np.minimum(-(-past // tpb) + rs.randint(0, 2, B), max_blocks)  # sometimes a block ahead of the tokens
    want = np.maximum(np.minimum(-(-(past + np.maximum(new, 0)) // tpb), max_blocks) - held, 0)
    N = int(held.sum() + spare * want.sum()) + 1
    order, at = rs.permutation(N), 0
    table = rs.randint(-5, N + 5, (B, max_blocks))  # behind the held blocks: anything
    for b in range(B):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    head, ring = int(rs.randint(0, N)), np.full(N, -1)
    ring[(head + np.arange(N - at)) % N] = order[at:]
    return past, new, table, held, ring, head, N - at


def run_tables(dev, past, new, table, held, ring, head, avail, pools, block_bytes, tpb, num_tokens, in_place=False):
    bases = (1 << 44) + np.arange(pools, dtype=np.int64) * (len(ring) * 2 * block_bytes + 4096)
    d = dict(past=dev_t(past, dev), new=dev_t(new, dev), table=dev_t(table, dev), counts=dev_t(held, dev), ring=dev_t(ring, dev),
             state=dev_t([head, avail], dev), bases=dev_t(bases, dev, np.int64))
    out = {} if in_place else dict(block_counts_out=torch.full_like(d["counts"], 99), free_state_out=torch.full_like(d["state"], 99))
    got = F.kv_block_tables(d["past"], d["new"], d["table"], d["counts"], d["ring"], d["state"], d["bases"], block_bytes=block_bytes,
                            tokens_per_block=tpb, num_tokens=num_tokens, **out)
    torch.cuda.synchronize()
    counts, state = (d["counts"], d["state"]) if in_place else (out["block_counts_out"], out["free_state_out"])
    t2, r2 = np.array(table), np.array(ring)
    want = R.block_tables(list(past), list(new), t2, list(held), r2, head, avail, bases, block_bytes, tpb, num_tokens)
    names = ("block_pointers", "token_offsets", "slot_map", "status", "block_counts", "free_state")
    for name, g, w in zip(names, list(got) + [counts, state], want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w).reshape(g.shape)), name
    assert np.array_equal(d["table"].cpu().numpy(), t2) and np.array_equal(d["ring"].cpu().numpy(), r2)
    if not in_place:
        assert np.array_equal(d["counts"].cpu().numpy(), held) and d["state"].tolist() == [head, avail]
    return d, want


@pytest.mark.parametrize("B,max_blocks,pools,tpb", [(1, 1, 1, 64), (3, 7, 2, 16), (17, 64, 5, 1), (64, 33, 32, 64), (300, 12, 3, 8),
                                                    (1025, 6, 2, 32), (2100, 5, 1, 16), (2, 1500, 4, 64), (40, 514, 64, 128)])
@pytest.mark.parametrize("spare", [1.0, 0.5, 0.0])
def test_tables(cuda, B, max_blocks, pools, tpb, spare):
    c = table_case(B, max_blocks, tpb, seed=B + max_blocks, spare=spare)
    total = int(np.maximum(c[1], 0).sum())
    run_tables(cuda, *c, pools, 4096, tpb, total)
    run_tables(cuda, *c, pools, 1 << 21, tpb, total + 300, in_place=True)
    run_tables(cuda, *c, pools, 4096, tpb, total // 2)
    run_tables(cuda, *c, 0, 4096, tpb, 0, in_place=True)


def test_tables_out_of_range_lengths_and_entries(cuda):
    # negative histories, counts beyond the table, more blocks than a row holds, table and ring entries outside the pool
    past, new = [-1, 5, 10, 60, 0, 3], [4, 4, 4, 10, 2, -1]
    held = [1, 9, -2, 8, 0, 1]
    table = np.arange(48).reshape(6, 8) % 20
    table[3, 2], table[5, 0] = -7, 1 << 20
    ring = np.array([19, 500, 3] + [-1] * 17)
    run_tables(cuda, past, new, table, held, ring, 0, 3, 2, 256, 8, 24)


def test_tables_hand_blocks_out_like_the_host_manager(cuda):
    # the host manager's pointer tensor, one admission after another, with a request that ends in between
    blocks, tpb, max_blocks = 12, 4, 5
    pools = [torch.zeros(2 * blocks * 2 * tpb * 8, dtype=torch.float16, device=cuda) for _ in range(3)]
    host = BlocksManager(pools, blocks, max_blocks_per_seq=max_blocks)
    dev = DeviceBlocksManager(pools, blocks, tpb, max_blocks, batch_size=3)
    seqs = [GenerationSequence(i, i) for i in range(3)]
    lengths = [0, 0, 0]

    def both(new):
        for b, add in enumerate(new):
            if add < 0:
                host.free(seqs[b])
                lengths[b] = 0
        for b, add in enumerate(new):
            if add > 0:
                have = host.get_number_blocks(seqs[b]) if seqs[b] in host._slot_of else 0
                for _ in range(-(-(lengths[b] + add) // tpb) - have):
                    host.allocate(seqs[b])
        past = torch.tensor([max(x, 0) for x in lengths], dtype=I32, device=cuda)
        ptr, _, slots, status = dev.step(past, torch.tensor(new, dtype=I32, device=cuda), num_tokens=32)
        for b, add in enumerate(new):
            lengths[b] += max(add, 0)
        assert status.tolist() == [0, 0, 0]
        want = torch.zeros(3, 3, 2, max_blocks, dtype=torch.int64)
        for p in range(3):
            rows = [s.get_batch_idx() for s in host._slot_of]
            want[p, sorted(rows)] = host.get_pointer_array(p, 1)[sorted(rows), 0] if len(rows) == 3 else want[p, sorted(rows)]
        return ptr.cpu(), want

    for new in ([5, 1, 9], [3, 4, 1], [1, 0, 4]):
        got, want = both(new)
        assert torch.equal(got, want)
    assert dev.free_blocks() == len(host.free_blocks)
    both([0, -1, 0])
    assert dev.free_blocks() == len(host.free_blocks)
    got, want = both([0, 9, 0])
    assert torch.equal(got, want)


def test_tables_in_a_graph(cuda):
    # a captured step whose state is updated in place: every replay goes on from the last
    B, max_blocks, tpb, N = 6, 16, 4, 64
    d = dict(past=torch.zeros(B, dtype=I32, device=cuda), new=torch.zeros(B, dtype=I32, device=cuda),
             table=torch.full((B, max_blocks), -1, dtype=I32, device=cuda), counts=torch.zeros(B, dtype=I32, device=cuda),
             ring=torch.arange(N, dtype=I32, device=cuda), state=torch.tensor([60, N], dtype=I32, device=cuda),
             bases=torch.tensor([1 << 40, 1 << 41], device=cuda))
    call = lambda: F.kv_block_tables(*d.values(), block_bytes=512, tokens_per_block=tpb, num_tokens=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()  # nothing asked, nothing changes
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call()
    torch.cuda.synchronize()
    table, counts, ring, head, avail = np.full((B, max_blocks), -1), [0] * B, np.arange(N), 60, N
    past = np.zeros(B, int)
    for new in ([5, 0, 3, 8, 1, 1], [1, 4, 1, 1, 1, 9], [-1, 2, 0, -1, 7, 1], [12, 1, 1, 30, 2, 2], [1] * B):
        for b in range(B):
            past[b] = 0 if new[b] < 0 else past[b]
        d["past"].copy_(torch.from_numpy(past.astype(np.int32)))
        d["new"].copy_(torch.tensor(new, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        want = R.block_tables(list(past), new, table, counts, ring, head, avail, [1 << 40, 1 << 41], 512, tpb, 64)
        for g, w in zip(list(got) + [d["counts"], d["state"]], want):
            assert np.array_equal(g.cpu().numpy(), np.asarray(w).reshape(g.shape))
        counts, (head, avail) = want[4], want[5]
        past = past + np.where(np.array(want[3]) == 0, np.maximum(new, 0), 0)


# ------------------------------------------------------------------------------------------------ accepted path
@pytest.mark.parametrize("ns,max_path", [([1], 1), ([0, 3, 0], 4), ([64], 8), ([65, 63, 1], 5), ([256], 300), ([257, 700], 20),
                                         (list(range(0, 40)), 6), ([27] * 130, 3)])
def test_accept(cuda, ns, max_path):
    rs = np.random.RandomState(len(ns) + max_path)
    parents = np.concatenate([random_tree(rs, n, wide=0.3 if n > 200 else 1.5) if n else [] for n in ns] + [[0] * 5]).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)
    # few different tokens: several children agree (the lowest counts), paths are long
    tokens, target = rs.randint(0, 2, len(parents)), rs.randint(0, 2, len(parents))
    got = F.draft_tree_accept(dev_t(tokens, cuda), dev_t(parents, cuda), dev_t(target, cuda), dev_t(offsets, cuda), max_path)
    want = R.accept(tokens, parents, target, offsets, max_path)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)


def test_accept_ignores_children_before_their_parents(cuda):
    # 2 -> 1 and a loop 3 <-> 4 are not followed; offsets outside the rows give an empty path
    parents, tokens = [-1, 2, 0, 4, 3, 2], [9, 5, 5, 5, 5, 5]
    args = [dev_t(x, cuda) for x in (tokens, parents, [5] * 6, [0, 6, 7, 3, -2])]
    path, counts, said = F.draft_tree_accept(*args, 4)
    assert path[0].tolist() == [0, 2, 5, -1] and counts.tolist() == [3, 0, 0, 0] and said[0].tolist() == [5, 5, 5, -1]
    assert (path[1:] == -1).all() and (said[1:] == -1).all()


# ------------------------------------------------------------------------------------------------ commit
@pytest.mark.parametrize("kv,D", [(torch.bfloat16, 128), (torch.float16, 72), (torch.int8, 64), (torch.float8_e4m3fn, 40), (torch.int8, 8)])
@pytest.mark.parametrize("tpb", [1, 16, 64])
def test_commit(cuda, kv, D, tpb):
    layers, Hkv, rs = 3, 3, np.random.RandomState(D + tpb)
    paths = [[0], [0, 1, 2, 3], [0, 2, 5], [0, 1, 2, 4, 5, 7, 8, 9, 10, 12, 20], [], list(range(18)), [1, 2, 3], [0, 19, 20]]
    # refused: not rising, negative, beyond the blocks, a missing block
    paths += [[0, 3, 3], [0, -1], [0, 5, 4], [0, 90]]
    B, P, room = len(paths) + 1, 20, 64
    paths.append([0, 30])
    past = rs.randint(0, room - 25, B)
    max_blocks = room // tpb
    blocks = B * max_blocks
    pool = torch.from_numpy(rs.randint(0, 100, (layers, 2, blocks, Hkv, tpb, D))).to(kv)
    table = rs.permutation(blocks).reshape(B, max_blocks)
    bb = Hkv * tpb * D * R.ESZ[kv]
    on = pool.to(cuda)
    idx = torch.from_numpy(table.astype(np.int64))
    ptr = torch.stack([idx, idx + blocks], 1)[None] * bb + (on.data_ptr() + torch.arange(layers) * (2 * blocks * bb))[:, None, None, None]
    past[-1] = 10
    ptr[:, -1, 1, 40 // tpb] = 0
    refused = set(range(B - 5, B))
    path = np.full((B, P), 77)
    for b, x in enumerate(paths):
        path[b, :len(x)] = x
    counts = np.array([len(x) for x in paths])
    lengths = F.kv_commit_path(ptr.contiguous().to(cuda), dev_t(past, cuda), dev_t(path, cuda), dev_t(counts, cuda), num_kv_heads=Hkv,
                               head_size=D, tokens_per_block=tpb, kv_dtype=kv)
    torch.cuda.synchronize()
    want, before = pool.view(torch.uint8).clone(), pool.view(torch.uint8)
    for b in range(B):
        if b in refused:
            continue
        for i, node in enumerate(paths[b]):
            s, t = past[b] + node, past[b] + i
            want[:, :, table[b, t // tpb], :, t % tpb] = before[:, :, table[b, s // tpb], :, s % tpb]
    assert torch.equal(on.view(torch.uint8).cpu(), want)
    assert lengths.tolist() == [int(past[b]) + (0 if b in refused else len(paths[b])) for b in range(B)]


def test_commit_long_paths(cuda):
    # more entries than one pass finds (64): every third node of 400, a chain that is accepted whole, and one refused at its end
    kv, D, tpb, Hkv, layers, max_blocks = torch.float16, 64, 32, 2, 2, 16
    paths = [list(range(0, 400, 3)), list(range(150)), list(range(0, 260, 2)) + [257], list(range(1, 66))]
    B, P = len(paths), max(map(len, paths))
    past, blocks = np.array([7, 0, 11, 100]), B * max_blocks
    rs = np.random.RandomState(0)
    pool = torch.from_numpy(rs.randint(0, 1000, (layers, 2, blocks, Hkv, tpb, D))).to(kv)
    table, bb = rs.permutation(blocks).reshape(B, max_blocks), Hkv * tpb * D * 2
    on, idx = pool.to(cuda), torch.from_numpy(table.astype(np.int64))
    ptr = torch.stack([idx, idx + blocks], 1)[None] * bb + (on.data_ptr() + torch.arange(layers) * (2 * blocks * bb))[:, None, None, None]
    path = np.full((B, P), -1)
    for b, x in enumerate(paths):
        path[b, :len(x)] = x
    lengths = F.kv_commit_path(ptr.contiguous().to(cuda), dev_t(past, cuda), dev_t(path, cuda), dev_t([len(x) for x in paths], cuda),
                               num_kv_heads=Hkv, head_size=D, tokens_per_block=tpb, kv_dtype=kv)
    torch.cuda.synchronize()
    want = pool.clone()
    for b, x in enumerate(paths):
        if b != 2:
            for i, node in enumerate(x):
                s, t = past[b] + node, past[b] + i
                want[:, :, table[b, t // tpb], :, t % tpb] = pool[:, :, table[b, s // tpb], :, s % tpb]
    assert torch.equal(on.cpu(), want)
    assert lengths.tolist() == [int(p) + (0 if b == 2 else len(x)) for b, (p, x) in enumerate(zip(past, paths))]


# ------------------------------------------------------------------------------------------------ the whole step
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.int8])
def test_speculative_steps(cuda, kv):
    """Four steps of three sequences over two layers.  After every step the cache must hold, in order, exactly what the
    definition stores for the committed tokens, and every layer's attention must match the definition over it."""
    layers, B, Hq, Hkv, D, tpb, max_blocks, blocks, P = 2, 3, 4, 2, 64, 16, 8, 20, 6
    rs, scale = np.random.RandomState(3), 1 / 32 if kv == torch.int8 else 1.0
    pool = [R.quantise(torch.randn(2, blocks, Hkv, tpb, D), kv, 1 / scale).to(cuda) for _ in range(layers)]
    mgr = DeviceBlocksManager(pool, blocks, tpb, max_blocks, batch_size=B)
    past = torch.tensor([0, 21, 40], dtype=I32, device=cuda)
    mgr.step(torch.zeros_like(past), past, num_tokens=61)  # the prompts' blocks (their K / V: what the pool holds)
    mirror = [p.cpu().clone() for p in pool]
    op = F.TreeAttention(num_heads=Hq, num_kv_heads=Hkv, head_size=D, dtype=torch.bfloat16, kv_dtype=kv, tokens_per_block=tpb,
                         position_embedding_type=2, rotary_embedding_dim=D)
    quant = {}
    if kv == torch.int8:
        quant = dict(kv_scale_orig_quant=torch.tensor([1 / scale], device=cuda), kv_scale_quant_orig=torch.tensor([scale], device=cuda))
    for step in range(4):
        host_past = past.tolist()
        ns = [int(n) for n in rs.randint(1, 14, B)]
        parents = [random_tree(rs, n) for n in ns]
        ptr, offsets, slots, status = mgr.step(past, torch.tensor(ns, dtype=I32, device=cuda), num_tokens=sum(ns))
        assert status.tolist() == [0] * B
        table = mgr.block_table.cpu().numpy().astype(np.int64)
        assert slots.tolist() == [int(table[b, (host_past[b] + i) // tpb]) * tpb + (host_past[b] + i) % tpb
                                  for b in range(B) for i in range(ns[b])]
        for layer in range(layers):
            c = TreeCase(host_past, parents, Hq, Hkv, D, torch.bfloat16, kv, tpb=tpb, rope=2, kv_scale=scale, seed=10 * step + layer)
            c.pool, c.table, c.blocks = mirror[layer], table, blocks
            assert offsets.tolist() == c.offsets.tolist()
            out = op(c.qkv.to(cuda), past, offsets, dev_t(c.mask.view(np.int32), cuda), ptr[layer], max_draft_length=max(ns),
                     max_past_length=max(host_past), position_offsets=dev_t(c.depth, cuda), **quant)
            ref, bound, mirror[layer] = c.reference()
            assert ((out.double().cpu() - ref).abs() <= bound).all()
        flat = np.concatenate(parents)
        tokens, target = rs.randint(0, 2, len(flat)), rs.randint(0, 2, len(flat))
        path, counts, _ = F.draft_tree_accept(dev_t(tokens, cuda), dev_t(flat, cuda), dev_t(target, cuda), offsets, P)
        past = F.kv_commit_path(ptr, past, path, counts, num_kv_heads=Hkv, head_size=D, tokens_per_block=tpb, kv_dtype=kv)
        want_path, want_counts, _ = R.accept(tokens, flat, target, offsets.tolist(), P)
        assert past.tolist() == [h + int(n) for h, n in zip(host_past, want_counts)]
        for layer in range(layers):
            before = mirror[layer].clone()
            for b in range(B):
                for i in range(want_counts[b]):
                    s, t = host_past[b] + want_path[b, i], host_past[b] + i
                    mirror[layer][:, table[b, t // tpb], :, t % tpb] = before[:, table[b, s // tpb], :, s % tpb]
            assert torch.equal(pool[layer].cpu().view(torch.uint8), mirror[layer].view(torch.uint8))


def test_captured_steps_on_two_streams(cuda):
    """A whole step captured once per batch, state updated in place, replayed on two streams at once with eager work in
    between: results and caches equal those of the same steps run eagerly, bit for bit."""
    layers, B, Hq, Hkv, D, tpb, max_blocks, blocks, P, n = 2, 4, 8, 2, 64, 16, 12, 60, 5, 9
    op = F.TreeAttention(num_heads=Hq, num_kv_heads=Hkv, head_size=D, dtype=torch.bfloat16, tokens_per_block=tpb,
                         position_embedding_type=2, rotary_embedding_dim=D)

    class State:
        def __init__(self, seed):
            g = torch.Generator().manual_seed(seed)
            self.pool = [torch.randn(2, blocks, Hkv, tpb, D, generator=g).to(torch.bfloat16).to(cuda) for _ in range(layers)]
            self.mgr = DeviceBlocksManager(self.pool, blocks, tpb, max_blocks, batch_size=B)
            self.past = torch.tensor([0, 21, 40, 64], dtype=I32, device=cuda)
            self.mgr.step(torch.zeros_like(self.past), self.past, num_tokens=1)
            rs = np.random.RandomState(seed)
            self.new = dev_t([n, n, 0, n], cuda)  # a row of a padded batch that drafts nothing
            trees = [R.tree_rows(random_tree(rs, n)) for _ in range(3)]
            self.mask = dev_t(np.concatenate([R.pack_rows(rows, 1) for rows, _ in trees]).view(np.int32), cuda)
            self.depth = dev_t(np.concatenate([depth for _, depth in trees]), cuda)
            self.qkv = torch.zeros(layers, 3 * n, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=cuda)
            self.tokens, self.target = (torch.zeros(3 * n, dtype=I32, device=cuda) for _ in range(2))
            self.parents = dev_t(np.concatenate([random_tree(rs, n) for _ in range(3)]), cuda)

        def inputs(self, step):
            g = torch.Generator().manual_seed(100 + step)
            self.qkv.copy_(torch.randn(self.qkv.shape, generator=g))
            for t in (self.tokens, self.target):
                t.copy_(torch.randint(0, 2, t.shape, generator=g))

        def step(self):
            ptr, offsets, _, _ = self.mgr.step(self.past, self.new, num_tokens=3 * n)
            outs = [op(self.qkv[i], self.past, offsets, self.mask, ptr[i], max_draft_length=n, max_past_length=150,
                       position_offsets=self.depth) for i in range(layers)]
            path, counts, said = F.draft_tree_accept(self.tokens, self.parents, self.target, offsets, P)
            self.past.copy_(F.kv_commit_path(ptr, self.past, path, counts, num_kv_heads=Hkv, head_size=D, tokens_per_block=tpb,
                                             kv_dtype=torch.bfloat16))
            return outs + [path, counts, said, ptr - self.mgr.pool_bases.view(-1, 1, 1, 1) * (ptr != 0)]

        def all(self):
            return self.pool + [self.past, self.mgr.block_table, self.mgr.block_counts, self.mgr.free_ring, self.mgr.free_state]

    graphs, eager = [State(1), State(2)], [State(1), State(2)]
    streams, captured = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s, stream in zip(graphs, streams):
        stream.wait_stream(torch.cuda.current_stream())
        before = [t.clone() for t in s.all()]
        with torch.cuda.stream(stream):
            s.step()  # outside the capture once
            for t, b in zip(s.all(), before):
                t.copy_(b)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = s.step()
        captured.append((graph, got))
    torch.cuda.synchronize()
    for step in range(4):
        for s in graphs + eager:
            s.inputs(step)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(captured, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, e, (_, got) in zip(graphs, eager, captured):
            for x, y in zip(got + s.all(), e.step() + e.all()):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), step
