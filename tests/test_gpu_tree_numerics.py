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
    wrong = S.verdict(out, *S.definition(c, pool, q_scaling))
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
