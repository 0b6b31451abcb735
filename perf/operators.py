"""Cases of the operators behind speculative decoding over the paged cache: block tables and slot maps built on the
device, attention of a tree of drafted tokens, the choice of the accepted path, and the move of its keys and values.

Every case runs in two forms on the same inputs: `own = False` computes the operator from elementary torch operations,
`own = True` calls the framework's entry points.  `exact` is the operator's definition in 64 bits, written apart from
the plain form."""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_ESZ = {"bf16": 2, "fp16": 2, "int8": 1, "fp8": 1}


_F = None


def _functional():
    global _F
    if _F is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "tensorrt-llm_amd"))
        from mi355q import functional as _F
    return _F


def listed():
    return [
        # one conversation, eight drafted tokens on a short history: the latency of one layer's call
        dict(name="tree_one_small", op="tree", batch=1, heads=32, kv_heads=8, head=128, draft=8, past_lo=200, past_hi=200,
             tpb=64, act="bf16", kv="bf16", rope=2, ragged=False),
        # a batch of full 64-node trees, one kv head per query head, ragged histories: bound by the cache's bytes
        dict(name="tree_mha_ragged", op="tree", batch=16, heads=32, kv_heads=32, head=128, draft=64, past_lo=300, past_hi=2048,
             tpb=64, act="bf16", kv="bf16", rope=2, ragged=True),
        # trees of an odd size, grouped heads, small cache blocks
        dict(name="tree_gqa_odd", op="tree", batch=32, heads=32, kv_heads=8, head=128, draft=27, past_lo=257, past_hi=4099,
             tpb=32, act="fp16", kv="fp16", rope=2, ragged=True),
        # 8 query heads per kv head on an fp8 cache: 512 query rows share every key, the matrix cores decide
        dict(name="tree_gqa_fp8", op="tree", batch=16, heads=64, kv_heads=8, head=128, draft=64, past_lo=4096, past_hi=4096,
             tpb=64, act="bf16", kv="fp8", rope=2, ragged=False),
        # one very long history: the key axis has to be split over the chip
        dict(name="tree_one_long", op="tree", batch=1, heads=64, kv_heads=8, head=128, draft=60, past_lo=120001, past_hi=120001,
             tpb=64, act="bf16", kv="bf16", rope=2, ragged=False),
        # narrow heads, an int8 cache in blocks of 16, interleaved rotation
        dict(name="tree_narrow_int8", op="tree", batch=8, heads=16, kv_heads=16, head=64, draft=13, past_lo=65, past_hi=1500,
             tpb=16, act="fp16", kv="int8", rope=1, ragged=True),
        # a decode step of a small batch: most rows need no block
        dict(name="tables_decode", op="tables", batch=8, pools=32, max_blocks=64, tpb=64, new_lo=1, new_hi=64, admit=0.0,
             release=0.0, spare=1.0),
        # a full scheduler step: rows that decode, prompts that are admitted, requests that end
        dict(name="tables_mixed", op="tables", batch=256, pools=64, max_blocks=512, tpb=64, new_lo=1, new_hi=64, admit=0.1,
             release=0.1, spare=1.0),
        # the walk along one tree
        dict(name="accept_one", op="accept", batch=1, draft=27, path=6, vocab=32000),
        # a full batch of trees
        dict(name="accept_batch", op="accept", batch=512, draft=64, path=8, vocab=32000),
        # the accepted keys and values of one conversation, all layers
        dict(name="commit_one", op="commit", batch=1, layers=32, kv_heads=8, head=128, draft=27, path=5, tpb=64, kv="bf16"),
        # and of a batch
        dict(name="commit_batch", op="commit", batch=32, layers=32, kv_heads=8, head=128, draft=64, path=8, tpb=64, kv="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "tables", "accept", "commit"])
    if op == "tree":
        kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
        group = rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if kv_heads * g <= 64])
        head = rng.choice([64, 80, 128, 128, 128, 256])
        act = rng.choice(["bf16", "fp16"])
        kv = rng.choice([act, act, "fp8", "int8"])
        past = _log_int(rng, 1, 16000)
        # at most about 50 million values in the cache
        limit = max(1, int(5e7 / (2 * kv_heads * head * (past + 256))))
        batch = min(_log_int(rng, 1, 64), limit)
        return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head=head, draft=_log_int(rng, 1, 130),
                    past_lo=rng.randint(0, past), past_hi=past, tpb=rng.choice([16, 32, 64, 128]), act=act, kv=kv,
                    rope=rng.choice([0, 1, 2, 2]), ragged=rng.random() < 0.7)
    if op == "tables":
        return dict(op=op, batch=_log_int(rng, 1, 256), pools=rng.randint(1, 64), max_blocks=_log_int(rng, 8, 512),
                    tpb=rng.choice([16, 32, 64, 128]), new_lo=1, new_hi=rng.randint(1, 64), admit=rng.choice([0.0, 0.1, 0.5]),
                    release=rng.choice([0.0, 0.1, 0.5]), spare=rng.choice([1.0, 1.0, 0.6]))
    if op == "accept":
        return dict(op=op, batch=_log_int(rng, 1, 512), draft=_log_int(rng, 1, 130), path=rng.randint(1, 12), vocab=32000)
    return dict(op=op, batch=_log_int(rng, 1, 32), layers=rng.randint(1, 32), kv_heads=rng.choice([1, 2, 4, 8]),
                head=rng.choice([64, 80, 128]), draft=rng.randint(20, 64), path=rng.randint(1, 8), tpb=rng.choice([16, 32, 64]),
                kv=rng.choice(["bf16", "fp16", "fp8"]))


# ------------------------------------------------------------------------------------------------ inputs
def _tree(rs, n):
    """Parents of n nodes, the root first, a parent before its children; wide near the root like drafted trees are."""
    parents = [-1]
    for i in range(1, n):
        parents.append(int(i * rs.random() ** 1.5))
    return parents


def _lengths(case):
    """Histories and tree sizes belong to the case: every seed's outputs have the same shapes."""
    B, rs = case["batch"], np.random.RandomState(1000 * case["batch"] + case["draft"])
    past = rs.randint(case["past_lo"], case["past_hi"] + 1, B)
    past[0] = case["past_hi"]
    draft = rs.randint(max(1, case["draft"] // 3), case["draft"] + 1, B) if case["ragged"] else np.full(B, case["draft"])
    draft[0] = case["draft"]
    return past.astype(np.int32), draft.astype(np.int32)


def _prepare_tree(case, seed):
    dev = torch.device("cuda")
    rs, gen = np.random.RandomState(seed), torch.Generator(device=dev).manual_seed(seed)
    B, Hq, Hkv, D, tpb = (case[k] for k in ("batch", "heads", "kv_heads", "head", "tpb"))
    past, draft = _lengths(case)
    act, kv = _DT[case["act"]], _DT[case["kv"]]
    offsets = np.concatenate([[0], np.cumsum(draft)]).astype(np.int32)
    tokens, words = int(offsets[-1]), (int(draft.max()) + 31) // 32
    mask, depth = np.zeros((tokens, words), np.uint32), np.zeros(tokens, np.int32)
    for b in range(B):
        rows = []
        for i, parent in enumerate(_tree(rs, int(draft[b]))):
            rows.append((rows[parent] if parent >= 0 else 0) | (1 << i))
            depth[offsets[b] + i] = 0 if parent < 0 else depth[offsets[b] + parent] + 1
        if case["ragged"] and draft[b] > 4:
            rows[-1] = 0  # a padded node: it sees none of the tree, not itself either
        for i, r in enumerate(rows):
            for w in range(words):
                mask[offsets[b] + i, w] = (r >> (32 * w)) & 0xffffffff
    per_seq = (past.astype(np.int64) + draft + tpb - 1) // tpb
    blocks, max_blocks = int(per_seq.sum()) + 3, int(per_seq.max())
    # cached and new keys and values: unit variance; for the int8 cache, whose scale is 1 here, they fill its range and
    # the queries are small to match
    spread = 25.0 if case["kv"] == "int8" else 1.0
    pool = torch.empty(2, blocks, Hkv, tpb, D, dtype=kv, device=dev)
    for half in range(2):
        for lo in range(0, blocks, 1024):
            x = torch.randn(min(1024, blocks - lo), Hkv, tpb, D, generator=gen, device=dev) * spread
            pool[half, lo:lo + 1024] = (x.round().clamp(-128, 127) if kv == torch.int8 else x).to(kv)
    order, table, at = rs.permutation(blocks), np.full((B, max_blocks), -1, np.int32), 0
    for b in range(B):
        table[b, :per_seq[b]] = order[at:at + per_seq[b]]
        at += int(per_seq[b])
    block_bytes = Hkv * tpb * D * _ESZ[case["kv"]]
    idx = torch.from_numpy(table.astype(np.int64)).to(dev)
    ptr = torch.stack([idx, idx + blocks], 1) * block_bytes + pool.data_ptr()
    ptr = torch.where((idx >= 0)[:, None, :].expand_as(ptr), ptr, torch.zeros_like(ptr)).contiguous()
    qkv = torch.randn(tokens, (Hq + 2 * Hkv) * D, generator=gen, device=dev)
    qkv[:, :Hq * D] /= spread
    qkv[:, Hq * D:] *= spread
    one = torch.ones(1, dtype=torch.float32, device=dev)
    st = dict(case=case, qkv=qkv.to(act), pool=pool, past_host=past, draft_host=draft, offsets_host=offsets, table=idx,
              block_pointers=ptr, past=torch.from_numpy(past).to(dev), offsets=torch.from_numpy(offsets).to(dev),
              depth=torch.from_numpy(depth).to(dev), mask=torch.from_numpy(mask.view(np.int32)).to(dev), one=one,
              max_draft=int(draft.max()), max_past=int(past.max()))
    if own:
        st["attn"] = _functional().TreeAttention(
            num_heads=Hq, num_kv_heads=Hkv, head_size=D, dtype=act, kv_dtype=kv, tokens_per_block=tpb,
            position_embedding_type=case["rope"], rotary_embedding_dim=D if case["rope"] else 0)
    return st


def _prepare_tables(case, seed):
    dev, rs = torch.device("cuda"), np.random.RandomState(seed)
    B, pools, max_blocks, tpb = (case[k] for k in ("batch", "pools", "max_blocks", "tpb"))
    # the lengths belong to the case (every seed's outputs have the same shapes), the blocks to the seed
    ls = np.random.RandomState(1000 * B + max_blocks)
    past = ls.randint(1, max_blocks * tpb * 3 // 4 + 1, B)
    new = ls.randint(case["new_lo"], case["new_hi"] + 1, B)
    u = ls.random_sample(B)
    admitted = u < case["admit"]
    past[admitted] = 0
    new[admitted] = ls.randint(1, max_blocks * tpb + 1, int(admitted.sum()))
    new[u > 1 - case["release"]] = -1
    counts = (past + tpb - 1) // tpb
    demand = np.maximum((past + np.maximum(new, 0) + tpb - 1) // tpb, counts)
    # spare < 1: the pool runs dry, and the last rows that ask for blocks are refused
    blocks = int(counts.sum() + case["spare"] * (demand - counts).sum()) + 17
    order, table, at = rs.permutation(blocks), np.full((B, max_blocks), -1, np.int32), 0
    for b in range(B):
        table[b, :counts[b]] = order[at:at + counts[b]]
        at += int(counts[b])
    free = blocks - at
    head = rs.randint(0, blocks)
    ring = np.full(blocks, -1, np.int32)
    ring[(head + np.arange(free)) % blocks] = order[at:]
    t = lambda a, d=np.int32: torch.from_numpy(np.ascontiguousarray(a, d)).to(dev)
    block_bytes = 8 * tpb * 128 * 2
    bases = (1 << 40) + np.arange(pools, dtype=np.int64) * (2 * blocks * block_bytes)
    return dict(case=case, past=t(past), new=t(new), table=t(table), counts=t(counts), ring=t(ring), state=t([head, free]),
                counts_out=t(np.zeros(B)), state_out=t([0, 0]), bases=t(bases, np.int64), blocks=blocks, block_bytes=block_bytes,
                tokens=int(np.maximum(new, 0).sum()))


def _prepare_accept(case, seed):
    dev, rs = torch.device("cuda"), np.random.RandomState(seed)
    B, n, V = case["batch"], case["draft"], case["vocab"]
    draft = rs.randint(max(1, n // 2), n + 1, B)
    offsets = np.concatenate([[0], np.cumsum(draft)]).astype(np.int32)
    parents = np.concatenate([_tree(rs, int(d)) for d in draft]).astype(np.int32)
    tokens = rs.randint(0, V, len(parents)).astype(np.int32)
    target = rs.randint(0, V, len(parents)).astype(np.int32)
    for b in range(B):  # the model agrees with the drafts along one random path of the tree
        par, at, step = parents[offsets[b]:offsets[b + 1]], int(offsets[b]), int(rs.randint(0, draft[b]))
        while step > 0:
            target[at + par[step]] = tokens[at + step]
            step = int(par[step])
    t = lambda a: torch.from_numpy(a).to(dev)
    return dict(case=case, tokens=t(tokens), parents=t(parents), target=t(target), offsets=t(offsets), batch=B, offsets_host=offsets)


def _prepare_commit(case, seed):
    dev = torch.device("cuda")
    rs, gen = np.random.RandomState(seed), torch.Generator(device=dev).manual_seed(seed)
    B, L, Hkv, D, tpb, P = (case[k] for k in ("batch", "layers", "kv_heads", "head", "tpb", "path"))
    past = rs.randint(1, 129 - case["draft"], B).astype(np.int32)
    max_blocks = (128 + tpb - 1) // tpb
    blocks = B * max_blocks
    pool = torch.empty(L, 2, blocks, Hkv, tpb, D, dtype=_DT[case["kv"]], device=dev)
    for layer in range(L):
        pool[layer] = torch.randn(2, blocks, Hkv, tpb, D, generator=gen, device=dev).to(pool.dtype)
    table = rs.permutation(blocks).reshape(B, max_blocks)
    counts = rs.randint(1, P + 1, B).astype(np.int32)
    path = np.full((B, P), -1, np.int32)
    for b in range(B):  # the root, then nodes of a wide tree: sources and destinations lie apart, so a pass can be repeated
        path[b, :counts[b]] = [0] + sorted(rs.choice(np.arange(P, case["draft"]), counts[b] - 1, replace=False))
    block_bytes = Hkv * tpb * D * _ESZ[case["kv"]]
    idx = torch.from_numpy(table.astype(np.int64)).to(dev)
    half = torch.stack([idx, idx + blocks], 1) * block_bytes
    ptr = half[None] + (pool.data_ptr() + torch.arange(L, device=dev) * (2 * blocks * block_bytes))[:, None, None, None]
    t = lambda a: torch.from_numpy(a).to(dev)
    return dict(case=case, pool=pool, block_pointers=ptr.contiguous(), table=idx, past=t(past), path=t(path), counts=t(counts))


def prepare(case, seed):
    return {"tree": _prepare_tree, "tables": _prepare_tables, "accept": _prepare_accept, "commit": _prepare_commit}[case["op"]](
        case, seed)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"tree": _own_tree, "tables": _own_tables, "accept": _own_accept, "commit": _own_commit}[op](state)
    return {"tree": _plain_tree, "tables": _plain_tables, "accept": _plain_accept, "commit": _plain_commit}[op](state)


def _own_tree(s):
    quant = dict(kv_scale_orig_quant=s["one"], kv_scale_quant_orig=s["one"]) if s["case"]["kv"] in ("int8", "fp8") else {}
    out = s["attn"](s["qkv"], s["past"], s["offsets"], s["mask"], s["block_pointers"], position_offsets=s["depth"],
                    max_draft_length=s["max_draft"], max_past_length=s["max_past"], **quant)
    return out, s["pool"]


def _own_tables(s):
    pointers, offsets, slots, status = _functional().kv_block_tables(
        s["past"], s["new"], s["table"], s["counts"], s["ring"], s["state"], s["bases"], block_bytes=s["block_bytes"],
        tokens_per_block=s["case"]["tpb"], num_tokens=s["tokens"], block_counts_out=s["counts_out"], free_state_out=s["state_out"])
    return pointers, offsets, slots, status, s["table"], s["counts_out"], s["ring"], s["state_out"]


def _own_accept(s):
    return _functional().draft_tree_accept(s["tokens"], s["parents"], s["target"], s["offsets"], s["case"]["path"])


def _own_commit(s):
    c = s["case"]
    lengths = _functional().kv_commit_path(s["block_pointers"], s["past"], s["path"], s["counts"], num_kv_heads=c["kv_heads"],
                                           head_size=c["head"], tokens_per_block=c["tpb"], kv_dtype=_DT[c["kv"]])
    return s["pool"], lengths


def _rotate(x, positions, kind):
    """Rotary embedding of [tokens, heads, D] in 64 bits (angles of far positions, values next to a rounding border)."""
    D = x.shape[-1]
    freq = 10000.0 ** (-torch.arange(0, D, 2, device=x.device, dtype=torch.float64) / D)
    ang = positions.double()[:, None] * freq
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    if kind == 2:
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def _to_cache(x, dtype):
    if dtype == torch.int8:
        return x.round().clamp(-128, 127).to(dtype)
    if dtype == torch.float8_e4m3fn:
        return x.clamp(-448, 448).to(dtype)
    return x.to(dtype)


def _plain_tree(s):
    c, pool = s["case"], s["pool"]
    Hq, Hkv, D, tpb = (c[k] for k in ("heads", "kv_heads", "head", "tpb"))
    qkv = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
    seq = torch.repeat_interleave(torch.arange(c["batch"], device=qkv.device), s["offsets"][1:] - s["offsets"][:-1],
                                  output_size=qkv.shape[0])
    if c["rope"]:
        qk = _rotate(qkv[:, :Hq + Hkv], s["past"][seq] + s["depth"], c["rope"])
    else:
        qk = qkv[:, :Hq + Hkv]
    q = qk[:, :Hq].float()
    slot = s["past"][seq] + torch.arange(qkv.shape[0], device=qkv.device) - s["offsets"][seq]
    block, at = s["table"][seq, slot // tpb], slot % tpb
    bytes_view = pool.view(torch.int8) if c["kv"] == "fp8" else pool
    for half, x in ((0, qk[:, Hq:]), (1, qkv[:, Hq + Hkv:])):
        x = _to_cache(x, pool.dtype)
        bytes_view[half, block, :, at] = x.view(torch.int8) if c["kv"] == "fp8" else x
    out = torch.empty(qkv.shape[0], Hq * D, dtype=s["qkv"].dtype, device=qkv.device)
    for b in range(c["batch"]):
        lo, hi, past = int(s["offsets_host"][b]), int(s["offsets_host"][b + 1]), int(s["past_host"][b])
        n, total = hi - lo, past + hi - lo
        blocks = s["table"][b, :(total + tpb - 1) // tpb]
        k, v = (bytes_view[h, blocks].view(pool.dtype).float().transpose(1, 2).reshape(-1, Hkv, D)[:total].transpose(0, 1)
                for h in range(2))
        rows = q[lo:hi].view(n, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
        scores = torch.matmul(rows, k.transpose(1, 2).contiguous()) / math.sqrt(D)
        bit = torch.arange(n, device=out.device)
        seen = torch.ones(n, total, dtype=torch.bool, device=out.device)
        seen[:, past:] = (s["mask"][lo:hi][:, bit // 32] >> (bit % 32)) & 1 == 1
        seen = seen.repeat(Hq // Hkv, 1)
        scores = scores.masked_fill(~seen, float("-inf"))
        top = scores.amax(-1, keepdim=True)
        p = (scores - torch.where(top.isinf(), torch.zeros_like(top), top)).exp()
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
        o = torch.matmul(p, v.contiguous()).view(Hkv, Hq // Hkv, n, D).permute(2, 0, 1, 3)
        out[lo:hi] = o.reshape(n, Hq * D).to(out.dtype)
    return out, pool


def _plain_tables(s):
    c, dev = s["case"], s["past"].device
    B, max_blocks, tpb, N = c["batch"], c["max_blocks"], c["tpb"], s["blocks"]
    past, new, counts, table, ring = s["past"].long(), s["new"].long(), s["counts"].long(), s["table"], s["ring"]
    head, avail = s["state"][0].long(), s["state"][1].long()
    release, fresh = new < 0, new.clamp_min(0)
    total = (past + fresh + tpb - 1) // tpb
    broken = (past < 0) | (counts < 0) | (counts > max_blocks)
    too_long = ~broken & ~release & (total > max_blocks)
    need = torch.where(broken | too_long | release, torch.zeros_like(total), (total - counts).clamp_min(0))
    upto = need.cumsum(0)
    short = (need > 0) & (upto > avail)
    grant = torch.where(short, torch.zeros_like(need), need)
    status = broken.int() * 3 + too_long.int() * 2 + short.int()
    back = torch.where(release & ~broken, counts, torch.zeros_like(counts))
    back_from = back.cumsum(0) - back
    j = torch.arange(max_blocks, device=dev)
    given = (j >= counts[:, None]) & (j < (counts + grant)[:, None])
    at = (head + (upto - need)[:, None] + j - counts[:, None]) % N
    table.copy_(torch.where(given, ring[at], table))
    returned = j < back[:, None]
    where = (head + avail + back_from[:, None] + j) % N
    ring[where[returned]] = table[returned]
    counts_out = torch.where(release & ~broken, torch.zeros_like(counts), counts + grant)
    s["counts_out"].copy_(counts_out)
    s["state_out"].copy_(torch.stack([(head + grant.sum()) % N, avail - grant.sum() + back.sum()]))
    live = j < counts_out[:, None]
    idx = torch.stack([table.long(), table.long() + N], 1)
    pointers = s["bases"][:, None, None, None] + idx * s["block_bytes"]
    pointers = torch.where(live[:, None, :].expand(B, 2, max_blocks), pointers, torch.zeros_like(pointers))
    offsets = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)]).int()
    row = torch.repeat_interleave(torch.arange(B, device=dev), fresh, output_size=s["tokens"])
    pos = past[row] + torch.arange(s["tokens"], device=dev) - offsets[row].long()
    slots = table[row, (pos // tpb).clamp_max(max_blocks - 1)].long() * tpb + pos % tpb
    slots = torch.where(status[row] == 0, slots, torch.full_like(slots, -1))
    return pointers, offsets, slots, status, table, s["counts_out"], ring, s["state_out"]


def _plain_accept(s):
    c, dev = s["case"], s["tokens"].device
    B, P = c["batch"], c["path"]
    lo, n = s["offsets"][:-1].long(), (s["offsets"][1:] - s["offsets"][:-1]).long()
    j = torch.arange(c["draft"], device=dev)
    inside = j < n[:, None]
    at = (lo[:, None] + j).clamp_max(s["tokens"].numel() - 1)
    tokens, parents, target = s["tokens"][at], s["parents"][at], s["target"][at]
    path = torch.full((B, P), -1, dtype=torch.int32, device=dev)
    emitted, counts = path.clone(), torch.zeros(B, dtype=torch.int32, device=dev)
    cur, alive = torch.zeros(B, dtype=torch.long, device=dev), n > 0
    for i in range(P):
        path[:, i] = torch.where(alive, cur, torch.full_like(cur, -1)).int()
        said = target.gather(1, cur[:, None])
        emitted[:, i] = torch.where(alive, said[:, 0], torch.full_like(said[:, 0], -1))
        counts += alive.int()
        match = inside & (j > cur[:, None]) & (parents == cur[:, None]) & (tokens == said)
        alive = alive & match.any(1)
        cur = torch.where(alive, match.int().argmax(1), cur)
    return path, counts, emitted


def _plain_commit(s):
    c, pool = s["case"], s["pool"]
    src_pos = s["past"].long()[:, None] + s["path"].long()
    dst_pos = s["past"].long()[:, None] + torch.arange(c["path"], device=pool.device)
    live = torch.arange(c["path"], device=pool.device) < s["counts"][:, None]
    row = torch.arange(c["batch"], device=pool.device)[:, None].expand_as(live)[live]
    src, dst = src_pos[live], dst_pos[live]
    flat = pool.view(torch.int8) if c["kv"] == "fp8" else pool
    moved = flat[:, :, s["table"][row, src // c["tpb"]], :, src % c["tpb"]]
    flat[:, :, s["table"][row, dst // c["tpb"]], :, dst % c["tpb"]] = moved
    return pool, s["past"] + s["counts"]


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case["op"] == "tree":
        past, draft = _lengths(case)
        Hq, Hkv, D = case["heads"], case["kv_heads"], case["head"]
        tokens, keys = int(draft.sum()), int(past.astype(np.int64).sum() + draft.sum())
        pairs = int(((past.astype(np.int64) + draft) * draft).sum())
        moved = tokens * (2 * Hq + 2 * Hkv) * D * 2 + keys * 2 * Hkv * D * _ESZ[case["kv"]]
        return dict(bytes=moved, flops=4 * Hq * D * pairs)
    if case["op"] == "tables":
        B, table = case["batch"], case["batch"] * case["max_blocks"]
        return dict(bytes=case["pools"] * table * 16 + table * 4 + B * 28, flops=case["pools"] * table * 4)
    if case["op"] == "accept":
        nodes = case["batch"] * case["draft"] * 3 // 4
        return dict(bytes=nodes * 12 + case["batch"] * (case["path"] * 8 + 8), flops=nodes * case["path"] * 2)
    rows = case["batch"] * max(1, (case["path"] - 1) // 2)
    moved = rows * 2 * case["layers"] * case["kv_heads"] * case["head"] * _ESZ[case["kv"]]
    return dict(bytes=2 * moved + case["batch"] * (case["path"] * 4 + 12), flops=moved // 2)


# ------------------------------------------------------------------------------------------------ definitions, 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"tree": _exact_tree, "tables": _exact_tables, "accept": _exact_accept, "commit": _exact_commit}[case["op"]](s)


def _exact_tree(s):
    c = s["case"]
    Hq, Hkv, D, tpb, G = c["heads"], c["kv_heads"], c["head"], c["tpb"], c["heads"] // c["kv_heads"]
    pool = s["pool"].to(torch.float64)
    dev = pool.device
    rows = s["qkv"].to(torch.float64)
    out = torch.zeros(rows.shape[0], Hq, D, dtype=torch.float64, device=dev)
    depth, mask = s["depth"].cpu().numpy(), s["mask"].cpu().numpy().view(np.uint32)
    table = s["table"].cpu().numpy()
    for b in range(c["batch"]):
        lo, n, past = int(s["offsets_host"][b]), int(s["draft_host"][b]), int(s["past_host"][b])
        x = rows[lo:lo + n].reshape(n, Hq + 2 * Hkv, D).clone()
        if c["rope"]:
            # a pair of components as one complex number, turned by its angle
            angle = np.outer(past + depth[lo:lo + n].astype(np.float64), np.exp(-math.log(10000.0) * np.arange(D // 2) / (D // 2)))
            turn = torch.from_numpy(np.exp(1j * angle)).to(dev)[:, None]
            y = x[:, :Hq + Hkv]
            first, second = (y[..., :D // 2], y[..., D // 2:]) if c["rope"] == 2 else (y[..., 0::2], y[..., 1::2])
            z = torch.complex(first.contiguous(), second.contiguous()) * turn
            if c["rope"] == 2:
                x[:, :Hq + Hkv] = torch.cat([z.real, z.imag], -1)
            else:
                x[:, :Hq + Hkv] = torch.view_as_real(z).reshape(n, Hq + Hkv, D)
        for i in range(n):
            blk, t = int(table[b, (past + i) // tpb]), (past + i) % tpb
            for half in range(2):
                new = x[i, Hq + half * Hkv:Hq + (half + 1) * Hkv]
                if c["kv"] == "int8":
                    new = torch.clamp(torch.round(new), -128, 127)
                elif c["kv"] == "fp8":
                    new = torch.clamp(new, -448, 448).to(torch.float8_e4m3fn).double()
                else:
                    new = new.to(_DT[c["kv"]]).double()
                pool[half, blk, :, t] = new
        sees = np.ones((n, past + n), bool)
        for j in range(n):
            sees[:, past + j] = (mask[lo:lo + n, j // 32] >> np.uint32(j % 32)) & np.uint32(1)
        hidden = torch.from_numpy(~sees).to(dev)
        used = torch.from_numpy(table[b, :(past + n + tpb - 1) // tpb].astype(np.int64)).to(dev)
        for h in range(Hkv):
            k = pool[0, used, h].reshape(-1, D)[:past + n]
            v = pool[1, used, h].reshape(-1, D)[:past + n]
            for g in range(G):
                e = x[:, h * G + g] @ k.t().contiguous() * (D ** -0.5)
                e[hidden] = -math.inf
                w = torch.nan_to_num(torch.softmax(e, -1), nan=0.0)
                out[lo:lo + n, h * G + g] = w @ v
    return out.reshape(-1, Hq * D), pool


def _exact_tables(s):
    c = s["case"]
    get = lambda k: s[k].cpu().numpy().astype(np.int64)
    past, new, table, counts, ring, (head, avail), bases = (get(k) for k in ("past", "new", "table", "counts", "ring", "state", "bases"))
    B, N, tpb, max_blocks = c["batch"], s["blocks"], c["tpb"], c["max_blocks"]
    taken = demand = 0
    tail = head + avail
    status, counts_out, offsets, slots = np.zeros(B, np.int64), counts.copy(), np.zeros(B + 1, np.int64), []
    pointers = np.zeros((c["pools"], B, 2, max_blocks), np.int64)
    for b in range(B):
        offsets[b + 1] = offsets[b] + max(new[b], 0)
        if past[b] < 0 or not 0 <= counts[b] <= max_blocks:
            status[b] = 3
        elif new[b] < 0:
            for i in range(counts[b]):
                ring[tail % N] = table[b, i]
                tail += 1
            counts_out[b] = 0
        elif past[b] + new[b] > max_blocks * tpb:
            status[b] = 2
        else:
            lack = max(0, -(-(past[b] + new[b]) // tpb) - counts[b])
            demand += lack
            if lack and demand > avail:
                status[b] = 1
            else:
                for i in range(lack):
                    table[b, counts[b] + i] = ring[(head + demand - lack + i) % N]
                taken += lack
                counts_out[b] += lack
        for t in range(past[b], past[b] + max(new[b], 0)):
            slots.append(table[b, t // tpb] * tpb + t % tpb if status[b] == 0 else -1)
        held = table[b, :counts_out[b]]
        for half in range(2):
            pointers[:, b, half, :counts_out[b]] = bases[:, None] + (held + half * N) * s["block_bytes"]
    state = np.array([(head + taken) % N, tail - head - taken])
    return tuple(torch.from_numpy(np.asarray(a)) for a in (pointers, offsets, np.array(slots, np.int64), status, table, counts_out,
                                                           ring, state))


def _exact_accept(s):
    c = s["case"]
    tokens, parents, target = (s[k].cpu().numpy() for k in ("tokens", "parents", "target"))
    B, P = c["batch"], c["path"]
    path, emitted, counts = np.full((B, P), -1, np.int64), np.full((B, P), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        lo, n = int(s["offsets_host"][b]), int(s["offsets_host"][b + 1] - s["offsets_host"][b])
        node = 0 if n else None
        while node is not None and counts[b] < P:
            said = target[lo + node]
            path[b, counts[b]], emitted[b, counts[b]] = node, said
            counts[b] += 1
            node = next((i for i in range(node + 1, n) if parents[lo + i] == node and tokens[lo + i] == said), None)
    return torch.from_numpy(path), torch.from_numpy(counts), torch.from_numpy(emitted)


def _exact_commit(s):
    c = s["case"]
    pool = s["pool"].to(torch.float64)
    before, past, path, counts, table = (s["pool"], *(s[k].cpu().numpy() for k in ("past", "path", "counts", "table")))
    for b in range(c["batch"]):
        for i in range(counts[b]):
            a, z = past[b] + path[b, i], past[b] + i
            pool[:, :, table[b, z // c["tpb"]], :, z % c["tpb"]] = before[:, :, table[b, a // c["tpb"]], :, a % c["tpb"]].double()
    return pool, torch.from_numpy((past + counts).astype(np.int64))
