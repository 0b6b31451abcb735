"""Attention of a tree of drafted tokens over the paged cache, through the C ABI, against the 64-bit definition.  The bound per
element is derived in TreeCase.reference; the cache rows the call stores are rounded once from 64 bits, so they are equal."""
import numpy as np
import pytest
import torch

from mi355q import _lib as L
from mi355q import functional as F
from speculative_reference import TreeCase, UNIT, pack_rows, random_tree

pytestmark = pytest.mark.gpu
BF, HF, I8, F8 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def trees(ns, seed=0):
    rs = np.random.RandomState(seed)
    return [random_tree(rs, n) if n else [] for n in ns]


def make_op(c, **kw):
    return F.TreeAttention(num_heads=c.Hq, num_kv_heads=c.Hkv, head_size=c.D, dtype=c.dtype, kv_dtype=c.kv_dtype,
                           tokens_per_block=c.tpb, position_embedding_type=c.rope, rotary_embedding_dim=c.rot_dim, **kw)


def device_args(c, dev, pool, depth=True):
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    args = [c.qkv.to(dev), t(np.array(c.past, np.int32)), t(c.offsets), t(c.mask.view(np.int32)), c.pointers(pool).to(dev)]
    kw = dict(max_draft_length=max(c.n), max_past_length=max(c.past), position_offsets=t(c.depth) if depth else None)
    if c.kv_dtype in (I8, F8):
        kw.update(kv_scale_orig_quant=torch.tensor([1.0 / c.kv_scale], dtype=torch.float32, device=dev),
                  kv_scale_quant_orig=torch.tensor([c.kv_scale], dtype=torch.float32, device=dev))
    if c.bias is not None:
        kw["qkv_bias"] = c.bias.to(dev)
    return args, kw


def bits(t):
    return t.contiguous().view(torch.uint8)


def compare(c, out, pool, ref, bound, ref_pool, rms=True):
    """Rows of sequences against the definition, the rest of `out` (given filled with a mark) untouched, the pool equal."""
    live = ~ref.isnan().all(1)
    o, r, t = out.double().cpu()[live], ref[live], bound[live]
    special = ~torch.isfinite(r)
    assert torch.equal(torch.isnan(o), torch.isnan(r)) and torch.equal(o[special & ~r.isnan()], r[special & ~r.isnan()])
    err = (o - r).abs()[~special]
    assert (err <= t[~special]).all(), f"error {err.max().item()} over its bound, worst ratio {(err / t[~special]).max().item()}"
    if rms and err.numel() > 64:
        # independent roundings (unit-variance inputs): each contributes at most u / sqrt(3), in all 1.15 u of sum p |v|
        assert err.square().mean().sqrt() <= 2 * UNIT[c.dtype] * r[~special].abs().max().clamp_min(1.0)
    mark = out.cpu()[~live]
    assert (mark == 7.0).all(), "rows outside the sequences were written"
    got = pool.cpu()
    if got.dtype in (BF, HF):  # a NaN is a NaN, whatever its payload bits (IEEE 754 leaves them to the conversion)
        got, ref_pool = (torch.where(x.isnan(), torch.full_like(x, float("nan")), x) for x in (got, ref_pool))
    assert torch.equal(bits(got), bits(ref_pool)), "cache rows differ"


def check(c, dev, depth=True, rms=True, skip=(), ref_kw=None, op_kw=None, **call):
    pool = c.pool.to(dev)
    args, kw = device_args(c, dev, pool, depth)
    kw.update(call)
    out = torch.full((c.tokens, c.Hq * c.D), 7.0, dtype=c.dtype, device=dev)
    make_op(c, **(op_kw or {}))(*args, out=out, **kw)
    torch.cuda.synchronize()
    compare(c, out, pool, *c.reference(skip=skip, **(ref_kw or {})), rms=rms)
    return out


@pytest.mark.parametrize("dtype,kv", [(BF, BF), (HF, HF), (BF, I8), (HF, I8), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (8, 1, 128), (6, 2, 64), (2, 1, 256), (3, 1, 80), (4, 2, 48)])
def test_types_and_head_layouts(cuda, dtype, kv, Hq, Hkv, D):
    scale = 4.0 / 127 if kv == I8 else 0.5 if kv == F8 else 1.0
    check(TreeCase([70, 130], trees([9, 21]), Hq, Hkv, D, dtype, kv, rope=2, kv_scale=scale, seed=D), cuda)


# lengths either side of a tile (64 keys), of a block, of the workgroup row counts (16, 32, 64, 128)
@pytest.mark.parametrize("past,n", [(0, 1), (1, 1), (0, 2), (63, 1), (64, 1), (65, 1), (0, 64), (1, 63), (64, 64), (127, 2), (300, 15),
                                    (200, 16), (200, 17), (129, 32), (190, 33), (255, 65), (100, 128), (31, 129), (5, 200)])
@pytest.mark.parametrize("kv", [BF, F8])
def test_lengths(cuda, past, n, kv):
    check(TreeCase([past, 17], trees([n, 3], n), 2, 2, 64, BF, kv, tpb=32, rope=1, seed=past + n), cuda)


@pytest.mark.parametrize("tpb", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("kv", [HF, I8])
def test_block_sizes(cuda, tpb, kv):
    check(TreeCase([150, 3], trees([20, 5]), 4, 2, 64, HF, kv, tpb=tpb, kv_scale=1 / 32 if kv == I8 else 1.0), cuda)


@pytest.mark.parametrize("rope,rot_dim,args", [(1, 32, {}), (2, 32, {}), (2, 20, {}), (1, 6, {}), (2, 64, dict(scale_type=1, scale=4.0)),
                                               (2, 64, dict(scale_type=2, scale=2.0, max_positions=100)), (2, 64, dict(base=500000.0))])
def test_rotary_forms_and_bias(cuda, rope, rot_dim, args):
    c = TreeCase([130, 80], trees([11, 30]), 4, 2, 64, BF, rope=rope, rot_dim=rot_dim, bias=True, rope_args=args)
    names = dict(scale_type="rotary_embedding_scale_type", scale="rotary_embedding_scale", base="rotary_embedding_base",
                 max_positions="rotary_embedding_max_positions")
    check(c, cuda, op_kw={names[k]: v for k, v in args.items()})


def test_positions_default_to_the_node_index(cuda):
    c = TreeCase([50], trees([12]), 2, 1, 64, HF, rope=2)
    c.depth = np.arange(c.tokens, dtype=np.int32)
    check(c, cuda, depth=False)


@pytest.mark.parametrize("kv", [BF, I8])
def test_far_positions(cuda, kv):
    # angles near 2^17: their fraction of a turn has to survive
    check(TreeCase([131000], trees([6]), 2, 1, 64, BF, kv, rope=2, kv_scale=1 / 32 if kv == I8 else 1.0), cuda)


@pytest.mark.parametrize("splits", [1, 2, 5, 64])
@pytest.mark.parametrize("Hq,n", [(1, 7), (8, 4), (8, 40)])
def test_key_splits(cuda, splits, Hq, n):
    c = TreeCase([1500, 64, 700, 0], trees([n, 1, n, 2]), Hq, 1, 128, BF, rope=2)
    check(c, cuda, op_kw=dict(multi_block_mode=splits))


@pytest.mark.parametrize("B,splits,bound", [(70, 0, 700), (200, 0, 2600), (256, 4, 700), (257, 4, 700), (300, 0, 2600), (300, 3, 700)])
def test_many_sequences(cuda, B, splits, bound):
    # lengths in any order, empty sequences and trees among them; bound: what the host says of the histories
    rs = np.random.RandomState(B + splits)
    past = [int(x) for x in rs.choice([0, 5, 63, 64, 130, 400, 600], B, p=[0.1, 0.3, 0.1, 0.1, 0.2, 0.1, 0.1])]
    c = TreeCase(past, trees([int(n) for n in rs.randint(0, 6, B)]), 2, 1, 64, BF, max_blocks=48, behind=3)
    check(c, cuda, op_kw=dict(multi_block_mode=splits), max_past_length=bound)


def test_masks(cuda):
    # nodes that see nothing (a zero row where there is no history), not themselves, everything, later nodes; bits beyond the
    # tree and rows beyond the sequences are set and must not count
    n = 40
    c = TreeCase([0, 90], [random_tree(np.random.RandomState(1), n)] * 2, 4, 2, 64, HF, lead=3, behind=5, extra_words=2)
    rows = [0, (1 << n) - 1, 1 << 39, 1 << 5] + [((1 << i) - 1) for i in range(4, n)]
    rows = [r | (1 << 63) | (1 << 100) | (1 << 41) for r in rows]
    for b in range(2):
        c.mask[c.offsets[b]:c.offsets[b + 1]] = pack_rows(rows, c.words)
    out = check(c, cuda)
    assert (out[3] == 0).all() and not (out[3 + n] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinities_and_nan_where_they_are_not_seen(cuda, dtype):
    c = TreeCase([30, 64, 0], trees([10, 50, 3], 3), 4, 2, 64, dtype)
    Hq, Hkv, D = 4, 2, 64
    k, v = Hq * D, (Hq + Hkv) * D
    # values of single nodes: they reach the rows that see the node, as infinities and NaN, and no other
    c.qkv[4, v + 5] = float("inf")
    c.qkv[6, v + 70] = float("nan")
    c.qkv[20, v + 1] = float("-inf")
    c.qkv[41, v + 127] = float("nan")
    for i in (4, 6, 20, 41):  # only the node itself sees it
        lo = 0 if i < 10 else 10
        c.mask[lo:lo + 60, (i - lo) // 32] &= np.uint32(~(1 << ((i - lo) % 32)) & 0xffffffff)
        c.mask[i, (i - lo) // 32] |= np.uint32(1 << ((i - lo) % 32))
    # a key that nobody sees, a query of its own
    c.qkv[60:63, :D] = 0.5
    c.qkv[62, k:k + D] = float("nan")
    c.mask[60:63, 0] = 3
    c.mask[62, 0] = 1
    # what lies in slots that no token uses
    used = set()
    for b, (p, n) in enumerate(zip(c.past, c.n)):
        used |= {(c.table[b, t // c.tpb], t % c.tpb) for t in range(p + n)}
    for blk in range(c.blocks):
        for t in range(c.tpb):
            if (blk, t) not in used:
                c.pool[:, blk, :, t] = float("nan")
    check(c, cuda, rms=False)


def test_large_scores(cuda):
    # scores of several hundred, positive and negative, maxima that keep growing along the keys
    c = TreeCase([400, 10], trees([13, 4]), 2, 1, 64, BF)
    ramp = torch.linspace(0.1, 12.0, c.blocks * c.tpb).view(1, c.blocks, 1, c.tpb, 1)
    c.pool = (c.pool.float() * ramp).to(BF)
    check(c, cuda, rms=False)
    c.qkv[:, :2 * 64] = -c.qkv[:, :2 * 64].abs() * 3
    c.pool = c.pool.abs()
    check(c, cuda, rms=False)


def test_q_scaling(cuda):
    c = TreeCase([100], trees([9]), 2, 2, 64, HF)
    check(c, cuda, op_kw=dict(q_scaling=0.5), ref_kw=dict(q_scaling=0.5), rms=False)


def test_strided_rows(cuda):
    c = TreeCase([80, 5], trees([17, 2]), 4, 2, 64, BF, rope=2)
    pool = c.pool.to(cuda)
    args, kw = device_args(c, cuda, pool)
    wide = torch.full((c.tokens, c.qkv.shape[1] + 24), float("nan"), dtype=BF, device=cuda)
    wide[:, 8:8 + c.qkv.shape[1]] = args[0]
    args[0] = wide[:, 8:8 + c.qkv.shape[1]]
    out = make_op(c)(*args, **kw)
    torch.cuda.synchronize()
    compare(c, out, pool, *c.reference())


def test_sequences_that_do_not_fit_are_skipped(cuda):
    # one history beyond the host's bound, one beyond the block table, a missing block, an empty sequence; the others' rows
    # are right and the skipped ones' stay
    c = TreeCase([40, 50, 60, 70, 20], trees([8, 8, 8, 0, 8]), 4, 2, 64, BF, tpb=16)
    ref, bound, ref_pool = c.reference(skip=(1, 2))
    pool = c.pool.to(cuda)
    args, kw = device_args(c, cuda, pool)
    args[1] = torch.tensor([40, 2000, 60, 70, 20], dtype=torch.int32, device=cuda)
    args[4][2, 0, 1] = 0
    kw["max_past_length"] = 70
    out = torch.full((c.tokens, c.Hq * c.D), 7.0, dtype=BF, device=cuda)
    make_op(c)(*args, out=out, **kw)
    torch.cuda.synchronize()
    # the nodes of the sequence with the missing block are stored where their own block is there
    pool[:, c.table[2, 60 // 16], :, 60 % 16:] = ref_pool[:, c.table[2, 60 // 16], :, 60 % 16:].to(cuda)
    pool[:, c.table[2, 64 // 16], :, :4] = ref_pool[:, c.table[2, 64 // 16], :, :4].to(cuda)
    compare(c, out, pool, ref, bound, ref_pool)


@pytest.mark.parametrize("Hq,n", [(2, 4), (2, 12), (2, 24), (2, 40)])
def test_scores_beyond_fp32(cuda, Hq, n):
    # the first keys' scores are -1e40 / 8, -inf in fp32: weight 0; so is the only maximum the first tiles could have
    c = TreeCase([300, 130], trees([n, n]), Hq, 1, 64, BF)
    c.qkv[:, 0:Hq * 64:64] = 1e20
    c.qkv[:, Hq * 64] = 0.0
    for b, p in enumerate(c.past):
        for t in range(p):
            c.pool[0, c.table[b, t // c.tpb], :, t % c.tpb, 0] = -1e20 if t < 129 else 0.0
    check(c, cuda, rms=False)


def test_a_block_that_is_not_aligned(cuda):
    # the sequence is skipped and nothing goes to that block
    c = TreeCase([40, 50], trees([8, 8]), 4, 2, 64, BF, tpb=16)
    ref, bound, ref_pool = c.reference(skip=(1,))
    pool = c.pool.to(cuda)
    args, kw = device_args(c, cuda, pool)
    args[4][1, :, 3] += 8  # positions 48 .. 63: all of its nodes'
    out = torch.full((c.tokens, c.Hq * c.D), 7.0, dtype=BF, device=cuda)
    make_op(c)(*args, out=out, **kw)
    torch.cuda.synchronize()
    compare(c, out, pool, ref, bound, ref_pool)


def test_rows_that_overlap_are_refused(cuda):
    c = TreeCase([40], trees([4]), 4, 2, 64, BF)
    args, kw = device_args(c, cuda, c.pool.to(cuda))
    rows = args[0]
    for bad in (rows[:1].expand(4, -1), rows.view(-1).as_strided(rows.shape, (8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            make_op(c)(bad, *args[1:], **kw)


def test_repeats_are_equal_and_other_streams(cuda):
    c = TreeCase([900, 40, 333], trees([30, 64, 5]), 8, 2, 128, BF, F8, rope=2)
    pool = c.pool.to(cuda)
    args, kw = device_args(c, cuda, pool)
    op = make_op(c)
    first = op(*args, **kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(op(*args, **kw))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(bits(o), bits(first))


def test_captured_into_a_graph(cuda):
    c = TreeCase([900, 40, 333], trees([30, 64, 5]), 8, 2, 128, HF, rope=2)
    pool = c.pool.to(cuda)
    args, kw = device_args(c, cuda, pool)
    op = make_op(c)
    want = op(*args, **kw)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        op(*args, out=out, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            op(*args, out=out, **kw)
    torch.cuda.synchronize()
    q0, past0 = args[0].clone(), args[1].clone()
    for step in range(3):  # new values and shorter histories in the same buffers, eager work in between
        args[0].copy_(q0 * (1 + 0.25 * step))
        args[1].copy_(torch.clamp(past0 - 7 * step, min=0))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(bits(got), bits(op(*args, **kw))), f"replay {step}"
        torch.cuda.synchronize()


def test_against_the_decode_kernel(cuda):
    # a chain of one token is the generation step the framework had: same inputs, same cache line
    import test_gpu_attention as ta  # noqa: F401  (the plugin's own parity tests)
    c = TreeCase([130, 66], [[-1], [-1]], 8, 2, 128, BF, rope=2)
    pool, pool2 = c.pool.to(cuda), c.pool.to(cuda)
    args, kw = device_args(c, cuda, pool)
    out = make_op(c)(*args, **kw)
    ptr = c.pointers(pool2)[None]
    plg = F.make_gpt_attention_plugin(num_heads=8, num_kv_heads=2, head_size=128, dtype="bfloat16", position_embedding_type=2,
                                      rotary_embedding_dim=128, tokens_per_block=c.tpb)
    past, cap = torch.tensor(c.past, dtype=torch.int32), c.max_blocks * c.tpb
    i32 = torch.int32
    ref = F.gpt_attention(
        plg, qkv=args[0][:, None], sequence_length=(past + 1).to(cuda), host_past_key_value_lengths=past,
        host_max_attention_window_sizes=torch.tensor([cap], dtype=i32), host_sink_token_length=torch.zeros(1, dtype=i32),
        context_lengths=past.to(cuda), cache_indirection=torch.zeros(2, 1, cap, dtype=i32, device=cuda),
        host_request_types=torch.ones(2, dtype=i32), kv_cache_block_pointers=ptr.to(cuda), host_kv_cache_block_pointers=ptr)
    torch.cuda.synchronize()
    # two kernels, each within its own bound of the definition
    _, bound, _ = c.reference()
    assert ((out.double() - ref[:, 0].double()).abs().cpu() <= 2 * bound).all()
    assert ((pool.double() - pool2.double()).abs() <= 2 * UNIT[BF] * pool.double().abs() + 1e-3).all()
