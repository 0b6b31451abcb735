"""CPU: the limits that the tree-attention tests hold the kernel to accept its arithmetic and reject a cheaper one."""
import numpy as np
import pytest
import torch

import speculative_precision as S
from speculative_reference import TreeCase, random_tree

BF, HF, I8, F8 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def case(dtype, kv, D, past=(300, 130), n=(20, 12), q_factor=4.0, **kw):
    rs = np.random.RandomState(D)
    scale = 4.0 / 127 if kv == I8 else 0.5 if kv == F8 else 1.0
    c = TreeCase(list(past), [random_tree(rs, m) for m in n], 4, 2, D, dtype, kv, kv_scale=scale, seed=D, **kw)
    # scores four times as wide as unit variance gives: an error of q then outweighs those of P and of the result
    c.qkv[:, :4 * D] = (c.qkv[:, :4 * D].float() * q_factor).to(dtype)
    return c


@pytest.mark.parametrize("dtype,kv", [(BF, BF), (HF, HF), (HF, I8), (HF, F8), (BF, I8), (BF, F8)])
@pytest.mark.parametrize("D", [64, 128])
def test_limits_accept_the_arithmetic(dtype, kv, D):
    c = case(dtype, kv, D)
    pool = c.reference()[2]
    assert S.wrong_with(S.model(c, pool), *S.definition(c, pool)) is None


@pytest.mark.parametrize("dtype,kv", [(BF, BF), (HF, HF), (HF, I8), (HF, F8)])
@pytest.mark.parametrize("D", [64, 128])
def test_limits_reject_a_query_in_one_part(dtype, kv, D):
    c = case(dtype, kv, D)
    pool = c.reference()[2]
    assert S.wrong_with(S.model(c, pool, q_parts=1), *S.definition(c, pool)) is not None


def test_limits_reject_zeros_and_a_lost_rescale():
    c = case(BF, BF, 64, q_factor=40.0)
    pool = c.reference()[2]
    ref, bound, var = S.definition(c, pool)
    assert S.wrong_with(S.model(c, pool), ref, bound, var) is None
    assert S.wrong_with(torch.zeros_like(ref), ref, bound, var) is not None
    assert ((ref.abs() <= bound).double().mean() < 0.05)


def test_definition_is_the_one_of_the_other_tests():
    c = TreeCase([70, 130], [random_tree(np.random.RandomState(1), n) for n in (9, 21)], 4, 2, 64, BF, I8, rope=1, kv_scale=1 / 32, bias=True)
    ref, _, pool = c.reference()
    assert torch.allclose(S.definition(c, pool)[0], ref, rtol=1e-12, atol=1e-12)
