"""Tree attention against limits derived from the roundings of its own arithmetic (speculative_precision), and at the ends of
the number formats it works in."""
import pytest
import torch

import speculative_precision as S
from speculative_reference import TreeCase, UNIT, pack_rows
from test_gpu_tree_attention import device_args, make_op, trees

pytestmark = pytest.mark.gpu
BF, HF, I8, F8 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
SCALE = {BF: 1.0, HF: 1.0, I8: 4.0 / 127, F8: 0.5}


def run(c, dev, op_kw=None, **call):
    """(out, pool) after the call, on the CPU."""
    pool = c.pool.to(dev)
    args, kw = device_args(c, dev, pool)
    kw.update(call)
    out = make_op(c, **(op_kw or {}))(*args, **kw)
    torch.cuda.synchronize()
    return out.cpu(), pool.cpu()


def holds(c, dev, op_kw=None, q_scaling=1.0, **call):
    out, pool = run(c, dev, op_kw, **call)
    wrong = S.wrong_with(out, *S.definition(c, pool, q_scaling))
    assert wrong is None, wrong
    return out


def put(c, half, b, t, d, value):
    """Element d of all kv heads of token t of sequence b's history."""
    c.pool[half, c.table[b, t // c.tpb], :, t % c.tpb, d] = value


# ------------------------------------------------------------------------------------------------ precision
@pytest.mark.parametrize("dtype,kv", [(BF, BF), (HF, HF), (BF, I8), (HF, I8), (BF, F8), (HF, F8)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (8, 1, 128), (6, 2, 64), (2, 1, 256), (3, 1, 80)])
@pytest.mark.parametrize("q_factor", [1.0, 4.0])
def test_precision(cuda, dtype, kv, Hq, Hkv, D, q_factor):
    c = TreeCase([300, 130], trees([20, 12]), Hq, Hkv, D, dtype, kv, rope=2, kv_scale=SCALE[kv], seed=D)
    c.qkv[:, :Hq * D] = (c.qkv[:, :Hq * D].float() * q_factor).to(dtype)
    holds(c, cuda)


@pytest.mark.parametrize("splits", [0, 1, 3, 24])
@pytest.mark.parametrize("Hq,n", [(1, 7), (4, 8), (8, 16), (8, 40)])  # one workgroup shape each
def test_precision_over_parts(cuda, splits, Hq, n):
    c = TreeCase([1500, 64, 700], trees([n, 1, n]), Hq, 1, 128, BF, rope=2)
    c.qkv[:, :Hq * 128] = (c.qkv[:, :Hq * 128].float() * 4).to(BF)
    holds(c, cuda, op_kw=dict(multi_block_mode=splits))


@pytest.mark.parametrize("dtype,kv", [(BF, BF), (HF, HF), (HF, I8)])
@pytest.mark.parametrize("splits", [1, 4])
def test_maxima_that_keep_growing(cuda, dtype, kv, splits):
    # scores of several hundred whose maximum grows along the keys, and all of them negative: every rescale shows
    c = TreeCase([400, 100], trees([13, 4]), 2, 1, 64, dtype, kv, kv_scale=1 / 8 if kv == I8 else 1.0)
    for b, past in enumerate(c.past):
        for t in range(past):
            row = c.pool[0, c.table[b, t // c.tpb], :, t % c.tpb]
            row.copy_((row.float() * (0.1 + 6.0 * t / past)).clamp(-127, 127).to(kv))
    c.qkv[:, :2 * 64] = (c.qkv[:, :2 * 64].float() * 4).to(dtype)
    holds(c, cuda, op_kw=dict(multi_block_mode=splits))
    c.qkv[:, :2 * 64] = -c.qkv[:, :2 * 64].abs()
    c.pool = c.pool.abs() if kv != I8 else c.pool.float().abs().clamp(max=127).to(kv)
    holds(c, cuda, op_kw=dict(multi_block_mode=splits))


@pytest.mark.parametrize("ns,kv", [([257, 3], BF), ([513, 1], F8), ([1024], HF), ([700, 64], I8)])
def test_large_trees(cuda, ns, kv):
    dtype = HF if kv in (HF, I8) else BF
    c = TreeCase([100, 20][:len(ns)], trees(ns, 5), 2, 1, 64, dtype, kv, tpb=32, kv_scale=SCALE[kv], rope=2)
    holds(c, cuda)


# ------------------------------------------------------------------------------------------------ far weights
@pytest.mark.parametrize("kv", [HF, I8, F8, BF])
@pytest.mark.parametrize("splits", [1, 5])
def test_a_key_far_ahead_keeps_the_others(cuda, kv, splits):
    # key 0 is 26 binary orders ahead of about 5000 others and its value is 0: the result is what the others add up to, whose
    # weights, 2^-26 of the largest, fall below fp16's smallest number where the largest is 1.  A weight held as 2^-16 in fp16
    # is off by 2^-25 at most (2^-9 of it), in bf16 by 2^-8 of it; a score of 18 by 2^-16 (q in two bf16 parts) and fp32: 2^-11
    dtype = BF if kv == BF else HF
    c = TreeCase([5000], trees([8]), 2, 1, 64, dtype, kv, kv_scale=1.0)
    c.qkv.zero_()
    c.qkv[:, :128:64] = 8.0   # q: (8, 0, ...), score = k_0
    c.pool[0] = torch.zeros(1).to(c.kv_dtype)
    c.pool[1] = torch.full((1,), 64.0).to(c.kv_dtype)
    c.qkv[:, 3 * 64:] = 64.0  # v of the nodes
    put(c, 0, 0, 0, 0, 18.0)
    for d in range(64):
        put(c, 1, 0, 0, d, 0.0)
    out, pool = run(c, cuda, op_kw=dict(multi_block_mode=splits))
    ref = S.definition(c, pool)[0]
    assert ref.abs().min() > 1e-3
    assert ((out.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -11 + UNIT[dtype]) * ref).all(), (out[0, 0].item(), ref[0, 0].item())


# ------------------------------------------------------------------------------------------------ scores at and beyond the ends of fp32
@pytest.mark.parametrize("D", [64, 128, 80, 48])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [3, 12, 40])
def test_infinite_keys_that_are_seen(cuda, D, dtype, n):
    # a history key and a node's key of -inf in one place: weight 0 for the queries that are positive there, NaN (a score of
    # +inf) for the others.  Head sizes that fill the kernel's rows and ones that do not, first and last element
    c = TreeCase([130, 20], trees([n, n]), 4, 2, D, dtype)
    q = c.qkv.view(c.tokens, 8, D)
    for head, sign in ((0, 1), (1, 1), (2, 1), (3, -1)):
        for d in (0, D - 1):
            q[:, head, d] = (sign * q[:, head, d].float().abs().clamp_min(0.1)).to(dtype)
    put(c, 0, 0, 3, 0, -float("inf"))
    put(c, 0, 0, 100, D - 1, -float("inf"))
    q[c.offsets[1] + 1, 4:6, D - 1] = -float("inf")
    out = holds(c, cuda)
    rows = slice(0, n)
    assert torch.isfinite(out[rows, :3 * D]).all() and out[rows, 3 * D:].isnan().all()


@pytest.mark.parametrize("qv,kvalue", [(1e21, -1e21), (1e23, -1e20), (3e38, -3e38), (-1e25, 1e22)])
@pytest.mark.parametrize("Hq,n,splits", [(2, 4, 0), (2, 12, 0), (2, 40, 3), (4, 40, 0)])
def test_finite_inputs_whose_scores_overflow(cuda, qv, kvalue, Hq, n, splits):
    # some keys' scores are far below -3e38, the others' are 0: weight 0, and the others share the result
    c = TreeCase([300, 130], trees([n, n]), Hq, 1, 64, BF)
    c.qkv[:, 0:Hq * 64:64] = qv
    c.qkv[:, Hq * 64] = 0.0
    for b, p in enumerate(c.past):
        for t in range(p):
            put(c, 0, b, t, 0, kvalue if t % 3 == 0 or t < 70 else 0.0)
    out = holds(c, cuda, op_kw=dict(multi_block_mode=splits))
    assert torch.isfinite(out).all()


def test_infinite_queries(cuda):
    # q = +inf in one place where two keys are positive, against keys that are negative there: +inf among the scores, NaN; where
    # no key is positive all scores are -inf and nothing has a weight: the row is 0
    for keys, nan in (((), False), ((3, 40), True)):
        c = TreeCase([70], trees([4]), 1, 1, 64, BF)
        c.qkv[:, 5] = float("inf")
        c.qkv[:, 64 + 5] = -1.0
        for t in range(70):
            put(c, 0, 0, t, 5, 1.0 if t in keys else -1.0)
        out, _ = run(c, cuda)
        assert out.isnan().all() if nan else (out == 0).all()


@pytest.mark.parametrize("n,splits", [(4, 1), (12, 1), (12, 4), (60, 1), (60, 4)])
@pytest.mark.parametrize("big", [1e16, 1e18])
def test_scores_far_below_zero(cuda, n, splits, big):
    # all scores equal, at -1e31 and -1e35: the weights are equal, whatever the scores' size
    c = TreeCase([500], trees([n]), 2, 1, 64, BF)
    c.qkv[:, :192] = 0.0
    c.qkv[:, [0, 64]] = big
    c.qkv[:, 128] = -big
    c.pool[0] = 0.0
    c.pool[0, ..., 0] = -big
    out, pool = run(c, cuda, op_kw=dict(multi_block_mode=splits))
    # equal weights: P is a power of 2 or one number for all keys, so the result is the mean but for the fp32 sums
    for rows, cols, q, k, v, hidden in S.heads(c, 0, pool):
        w = (~hidden).double() / (~hidden).sum(1, keepdim=True)
        # (P's one rounding is in the sums of all keys, 2^-8, and the result's own)
        assert ((out[rows, cols].double() - w @ v).abs() <= 2 * UNIT[BF] * (w @ v).abs() + 2.0 ** -16 * (w @ v.abs())).all()


@pytest.mark.parametrize("dtype,kv,factor", [(BF, I8, 1.0), (BF, F8, 1.0), (BF, F8, 1e6), (HF, HF, 1.0), (HF, F8, 1.0)])
@pytest.mark.parametrize("n,splits", [(3, 1), (12, 3), (60, 1)])
def test_queries_beyond_fp16(cuda, dtype, kv, factor, n, splits):
    # q times its scale is beyond 65504 in two places, of which the larger decides: cut off there both would be equal, and the
    # other key, with the larger element, would win
    c = TreeCase([100], trees([n]), 2, 1, 64, dtype, kv, kv_scale=1.0)
    q_scaling = 1.0 if dtype == BF else 1.0 / 512
    c.qkv[:, :128] = (c.qkv[:, :128].float() * 0.1).to(dtype)
    c.qkv[:, [0, 64]] = 3.0e6 * factor if dtype == BF else 30000.0
    c.qkv[:, [1, 65]] = 1.0e6 * factor if dtype == BF else 10000.0
    c.qkv[:, 128:192] = 0.0
    c.pool[0] = torch.zeros(1).to(c.kv_dtype)
    put(c, 0, 0, 7, 0, 1.0)
    put(c, 0, 0, 40, 1, 2.0)
    out = holds(c, cuda, op_kw=dict(multi_block_mode=splits, q_scaling=q_scaling), q_scaling=q_scaling)
    v = c.pool[1, c.table[0, 0], 0, 7]
    assert torch.equal(out[:, :64], v.to(dtype).expand(n, -1))


# ------------------------------------------------------------------------------------------------ NaN into 8-bit caches
@pytest.mark.parametrize("kv,low", [(I8, -128), (F8, -448.0)])
def test_nan_into_an_8_bit_cache_is_its_lowest_value(cuda, kv, low):
    # like every kernel of the framework that writes these caches; infinities saturate.  No row but those that see the node changes
    c = TreeCase([70], trees([9]), 4, 2, 64, BF, kv, kv_scale=1 / 32)
    k, v = 4 * 64, 6 * 64
    seen = [0b1, 0b11, 0b101, 0b1001, 0b10001, 0b100001, 0b1000001, 0b10000001, 0b100000001]
    c.mask[:] = pack_rows(seen, c.words)
    clean, clean_pool = run(c, cuda)
    for i, at in ((3, v + 5), (5, k + 70)):
        c.qkv[i, at] = float("nan")
    c.qkv[6, v + 9], c.qkv[6, v + 10] = float("inf"), float("-inf")
    out, pool = run(c, cuda)
    value = lambda half, node, h, d: pool[half, c.table[0, (70 + node) // c.tpb], h, (70 + node) % c.tpb, d].float().item()
    assert value(1, 3, 0, 5) == low and value(0, 5, 1, 6) == low
    assert value(1, 6, 0, 9) == (127 if kv == I8 else 448) and value(1, 6, 0, 10) == low
    same = [0, 1, 2, 4, 7, 8]
    assert torch.equal(out[same].view(torch.int16), clean[same].view(torch.int16)) and torch.isfinite(out).all()
    held = c.qkv.clone()
    held[held.isnan()] = low / 32
    c.qkv = held
    wrong = S.wrong_with(out, *S.definition(c, pool))
    assert wrong is None, wrong


# ------------------------------------------------------------------------------------------------ maxima whose step is coarse
@pytest.mark.parametrize("dtype,kv", [(BF, I8), (BF, F8), (HF, HF), (BF, BF)])
@pytest.mark.parametrize("log2_score", [12, 20, 22.5, 23.5, 24.5, 25.5, 26.5, 27.5, 28.5, 29.5, 31, 40])
@pytest.mark.parametrize("n,splits", [(3, 1), (60, 1), (60, 3)])
def test_one_key_far_ahead_of_all_at_any_size(cuda, dtype, kv, log2_score, n, splits):
    # the largest score is 2^log2_score binary orders, where fp32 counts in steps of up to 2^17; the rest lies as far behind
    c = TreeCase([200], trees([n]), 2, 1, 64, dtype, kv, kv_scale=1.0)
    q_scaling = 1.0 if dtype == BF else 2.0 ** -24
    value = 2.0 ** log2_score / (0.125 * 1.4426950408889634) * q_scaling / 2
    c.qkv[:, :192] = 0.0
    c.qkv[:, [0, 64]] = value
    c.pool[0] = torch.zeros(1).to(c.kv_dtype)
    put(c, 0, 0, 7, 0, 1.0)
    put(c, 0, 0, 150, 0, 2.0)  # in another tile: the maximum doubles
    out, _ = run(c, cuda, op_kw=dict(multi_block_mode=splits, q_scaling=q_scaling))
    if not torch.isfinite(c.qkv).all():  # (fp16 does not hold the query of the last case: inf * 0 is NaN)
        assert dtype == HF and log2_score == 40 and out.isnan().all()
        return
    v = c.pool[1, c.table[0, 150 // c.tpb], 0, 150 % c.tpb]
    assert torch.equal(out[:, :64], v.to(dtype).expand(n, -1))


@pytest.mark.parametrize("dtype,kv", [(BF, I8), (HF, HF), (BF, BF)])
@pytest.mark.parametrize("top", [1000, 30000, 500000])
def test_a_maximum_that_moves_a_little_at_large_scores(cuda, dtype, kv, top):
    # key 7 at `top` binary orders, key 150 a few above it: the rescale has to move sums and maximum by the same step
    c = TreeCase([200], trees([12]), 1, 1, 64, dtype, kv, kv_scale=1.0)
    q_scaling = 2.0 ** -8
    c.qkv[:, :128] = 0.0
    unit = 0.125 * 1.4426950408889634 / q_scaling  # of a score per q k
    c.qkv[:, 0], c.qkv[:, 1] = top / unit / 64, 20.3 / unit
    c.pool[0] = torch.zeros(1).to(c.kv_dtype)
    for t, extra in ((7, 0.0), (150, 1.0)):
        put(c, 0, 0, t, 0, 64.0)
        put(c, 0, 0, t, 1, extra)
    out, pool = run(c, cuda, op_kw=dict(q_scaling=q_scaling))
    ref = S.definition(c, pool, q_scaling)[0]
    # key 150 is 2^20 ahead; key 7's share, 2^-20, is below the result's rounding
    assert ((out.double() - ref).abs() <= UNIT[dtype] * ref.abs() + 2.0 ** -18 * ref.abs().max()).all()
