"""Plain 64-bit CPU definitions of the speculative-decoding operators, and the cases their tests share."""
import math

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
ESZ = {torch.bfloat16: 2, torch.float16: 2, torch.int8: 1, torch.float8_e4m3fn: 1}


def random_tree(rs, n, wide=1.5):
    parents = [-1]
    for i in range(1, n):
        parents.append(int(i * rs.random_sample() ** wide))
    return parents


def tree_rows(parents):
    """(visible sets as Python integers, depths): every node sees its ancestors and itself."""
    rows, depth = [], []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << i))
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return rows, depth


def pack_rows(rows, words):
    return np.array([[(r >> (32 * w)) & 0xffffffff for w in range(words)] for r in rows], np.uint32).reshape(len(rows), words)


def quantise(x, kv_dtype, scale_orig_quant=1.0):
    x = x.double() * float(scale_orig_quant)
    if kv_dtype == torch.int8:
        return x.round().clamp(-128, 127).to(torch.int8)
    if kv_dtype == torch.float8_e4m3fn:
        return torch.nan_to_num(x, nan=-448.0).clamp(-448, 448).to(kv_dtype) if x.isnan().any() else x.clamp(-448, 448).to(kv_dtype)
    return x.to(kv_dtype)


def angles(pos, rot_dim, base=10000.0, scale_type=0, scale=1.0, max_positions=1024):
    """[tokens, rot_dim / 2] rotary angles; a node's own position decides the dynamic base."""
    out = np.zeros((len(pos), rot_dim // 2))
    for i, t in enumerate(pos):
        b, s = float(base), 1.0
        if scale_type == 1:
            s = 1.0 / scale
        elif scale_type == 2 and t > max_positions:
            b *= (t * (scale / max_positions) - (scale - 1.0)) ** (rot_dim / (rot_dim - 2))
        out[i] = t * s * b ** (-np.arange(0, rot_dim, 2) / rot_dim)
    return torch.from_numpy(out)


def rotate(x, ang, kind, rot_dim):
    """x [tokens, heads, D] double; kind 1 pairs (2 j, 2 j + 1), 2 pairs (j, j + rot_dim / 2)."""
    c, s, y = ang.cos()[:, None], ang.sin()[:, None], x.clone()
    a, b = (x[..., 0:rot_dim:2], x[..., 1:rot_dim:2]) if kind == 1 else (x[..., :rot_dim // 2], x[..., rot_dim // 2:rot_dim])
    u, v = a * c - b * s, b * c + a * s
    if kind == 1:
        y[..., 0:rot_dim:2], y[..., 1:rot_dim:2] = u, v
    else:
        y[..., :rot_dim // 2], y[..., rot_dim // 2:rot_dim] = u, v
    return y


class TreeCase:
    """Host tensors of a tree-attention call over sequences with the given histories and parents."""

    def __init__(self, past, parents, Hq, Hkv, D, dtype, kv_dtype=None, tpb=64, rope=0, rot_dim=None, seed=0, kv_scale=1.0,
                 spread=1.0, bias=False, lead=0, behind=0, extra_words=0, max_blocks=None, rope_args=None):
        rs, g = np.random.RandomState(seed), torch.Generator().manual_seed(seed)
        self.past, self.parents, self.n = list(past), parents, [len(p) for p in parents]
        self.Hq, self.Hkv, self.D, self.dtype, self.tpb, self.rope = Hq, Hkv, D, dtype, tpb, rope
        self.kv_dtype, self.kv_scale, self.rot_dim = kv_dtype or dtype, kv_scale, (rot_dim or D) if rope else 0
        self.rope_args = rope_args or {}
        B = len(self.past)
        self.offsets = np.concatenate([[lead], lead + np.cumsum(self.n)]).astype(np.int32)
        self.tokens = int(self.offsets[-1]) + behind
        self.words = (max(self.n + [1]) + 31) // 32 + extra_words
        self.mask = np.full((self.tokens, self.words), 0xffffffff, np.uint32)  # rows outside the sequences: anything
        self.depth = np.zeros(self.tokens, np.int32)
        for b in range(B):
            rows, depth = tree_rows(parents[b])
            lo = int(self.offsets[b])
            self.mask[lo:lo + self.n[b]] = pack_rows(rows, self.words)
            self.depth[lo:lo + self.n[b]] = depth
        need = [-(-(p + n) // tpb) for p, n in zip(self.past, self.n)]
        self.max_blocks = max_blocks or max(need + [1])
        self.blocks = sum(need) + 2
        self.pool = quantise(torch.randn(2, self.blocks, Hkv, tpb, D, generator=g) * spread, self.kv_dtype, 1.0 / kv_scale)
        order, at = rs.permutation(self.blocks), 0
        self.table = np.full((B, self.max_blocks), -1, np.int64)
        for b in range(B):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        x = torch.randn(self.tokens, (Hq + 2 * Hkv) * D, generator=g)
        x[:, Hq * D:] *= spread
        self.qkv = x.to(dtype)
        self.bias = (torch.randn((Hq + 2 * Hkv) * D, generator=g) * 0.3).to(dtype) if bias else None

    def pointers(self, pool):
        """[B, 2, max_blocks] addresses into a device copy of the pool."""
        bb = self.Hkv * self.tpb * self.D * ESZ[self.kv_dtype]
        idx = torch.from_numpy(self.table)
        ptr = torch.stack([idx, idx + self.blocks], 1) * bb + pool.data_ptr()
        return torch.where((idx >= 0)[:, None].expand_as(ptr), ptr, torch.zeros_like(ptr)).contiguous()

    def seen(self, b):
        lo, n, past = int(self.offsets[b]), self.n[b], self.past[b]
        see = np.ones((n, past + n), bool)
        for j in range(n):
            see[:, past + j] = (self.mask[lo:lo + n, j // 32] >> np.uint32(j % 32)) & 1
        return torch.from_numpy(see)

    def reference(self, q_scaling=1.0, skip=()):
        """(out [tokens, Hq * D] double (NaN outside the sequences), bound per element, pool after the call).
        The bound: q and p are each rounded to the activation type once (half a step u, relative) and so is the result.  q's
        rounding moves a score by at most u A, A = max over the visible keys of sum_d |q_d k_d| / sqrt(D), the softmax weights by
        the factor exp(2 u A); the fp32 sums add less than 2^-16."""
        Hq, Hkv, D, G, tpb = self.Hq, self.Hkv, self.D, self.Hq // self.Hkv, self.tpb
        u = UNIT[self.dtype]
        out = torch.full((self.tokens, Hq * D), float("nan"), dtype=torch.float64)
        bound = out.clone()
        pool = self.pool.clone()
        raw = pool.view(torch.int8) if self.kv_dtype == torch.float8_e4m3fn else pool
        for b, (past, n) in enumerate(zip(self.past, self.n)):
            if n == 0 or b in skip:
                continue
            lo = int(self.offsets[b])
            x = self.qkv[lo:lo + n].double()
            if self.bias is not None:
                x = x + self.bias.double()
            x = x.view(n, Hq + 2 * Hkv, D)
            if self.rope:
                ang = angles(past + self.depth[lo:lo + n], self.rot_dim, **self.rope_args)
                x = torch.cat([rotate(x[:, :Hq + Hkv], ang, self.rope, self.rot_dim), x[:, Hq + Hkv:]], 1)
            for half in range(2):
                new = quantise(x[:, Hq + half * Hkv:Hq + (half + 1) * Hkv], self.kv_dtype, 1.0 / self.kv_scale)
                new = new.view(torch.int8) if self.kv_dtype == torch.float8_e4m3fn else new
                for i in range(n):
                    raw[half, self.table[b, (past + i) // tpb], :, (past + i) % tpb] = new[i]
            blocks = torch.from_numpy(self.table[b, :-(-(past + n) // tpb)])
            hidden = ~self.seen(b)
            for h in range(Hkv):
                k, v = (raw[half, blocks, h].reshape(-1, D)[:past + n].view(pool.dtype).double() * self.kv_scale for half in range(2))
                for g in range(G):
                    q = x[:, h * G + g] / (math.sqrt(D) * q_scaling)
                    s = q @ k.t()
                    s[hidden] = -math.inf
                    empty = hidden.all(1)
                    s[empty] = 0.0
                    w = torch.softmax(s, -1)
                    w[hidden] = 0.0
                    # 0 * inf of a key that is not seen is not part of the sum
                    strange = ~torch.isfinite(v).all(1)
                    o = w[:, ~strange] @ v[~strange]
                    ab = w[:, ~strange] @ v[~strange].abs()
                    for t in torch.nonzero(strange).flatten().tolist():
                        o[~hidden[:, t]] += w[~hidden[:, t], t][:, None] * v[t]
                    # (a key whose weight is 0 in 64 bits adds nothing, however its score is rounded)
                    amax = (q.abs() @ torch.nan_to_num(k).abs().t()).masked_fill(hidden | (w == 0), 0.0).amax(1, keepdim=True)
                    cols = slice((h * G + g) * D, (h * G + g + 1) * D)
                    out[lo:lo + n, cols] = o
                    bound[lo:lo + n, cols] = (torch.expm1(2 * u * amax) + 2 * u + 2.0 ** -16) * ab + 1e-7
        return out, bound, pool


# ------------------------------------------------------------------------------------------------ integer operators
def block_tables(past, new, table, counts, ring, head, avail, bases, block_bytes, tpb, num_tokens):
    """The definition, one request after another.  table / ring are changed in place."""
    B, max_blocks, N, pools = len(past), table.shape[1], len(ring), len(bases)
    taken = demand = 0
    tail = head + avail
    status, counts_out = [0] * B, list(counts)
    offsets, slots = [0], []
    pointers = np.zeros((pools, B, 2, max_blocks), np.int64)
    for b in range(B):
        fresh = max(new[b], 0)
        offsets.append(offsets[-1] + fresh)
        if past[b] < 0 or not 0 <= counts[b] <= max_blocks:
            status[b] = 3
        elif new[b] < 0:
            for i in range(counts[b]):
                ring[tail % N] = table[b, i]
                tail += 1
            counts_out[b] = 0
        elif -(-(past[b] + new[b]) // tpb) > max_blocks:
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
        for t in range(past[b], past[b] + fresh):
            ok = status[b] == 0 and 0 <= table[b, t // tpb] < N
            slots.append(int(table[b, t // tpb]) * tpb + t % tpb if ok else -1)
        if 0 <= counts_out[b] <= max_blocks:  # a refused request keeps what it has
            for j in range(counts_out[b]):
                if 0 <= table[b, j] < N:
                    for half in range(2):
                        pointers[:, b, half, j] = np.asarray(bases) + (int(table[b, j]) + half * N) * block_bytes
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    return pointers, offsets, slots, status, counts_out, [(head + taken) % N, tail - head - taken]


def accept(tokens, parents, target, offsets, max_path):
    B = len(offsets) - 1
    path, said, counts = np.full((B, max_path), -1), np.full((B, max_path), -1), np.zeros(B, int)
    for b in range(B):
        lo, n = offsets[b], offsets[b + 1] - offsets[b]
        node = 0 if n > 0 else None
        while node is not None and counts[b] < max_path:
            want = target[lo + node]
            path[b, counts[b]], said[b, counts[b]] = node, want
            counts[b] += 1
            node = next((i for i in range(node + 1, n) if parents[lo + i] == node and tokens[lo + i] == want), None)
    return path, counts, said
