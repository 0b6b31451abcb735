"""Tree attention in 64 bits with the error that the kernel's own arithmetic may make, and a CPU model of that arithmetic.

The kernel holds q, times score scale and log2(e), in two parts of the type its products run in (one part for a bf16 result over
an 8-bit cache), the scores and both sums in fp32, and rounds the weights P and the result once each.  With u half a step of a
type, relative:
  * q: two parts leave u_c^2, one part u_c; the rotation and the scale run in fp32 (8 roundings of 2^-24 at most);
  * a score moves by at most (that) * A, A = max over the visible keys of sum_d |q_d k_d| / sqrt(D), and by the fp32 sums' 64
    roundings of A and of the running maximum they start from; in fp16 a part below its normal range is off by 2^-25 at most;
  * a weight moves by the factor exp(2 * that), by u_c of P, and by 2^-16 of the sums;
  * the result is rounded once: u of itself.
Independent roundings, uniform over a step: variance (step / 2)^2 / 3 each, which `variance` adds up."""
import math

import torch

from speculative_reference import UNIT, angles, rotate

BF, HF = torch.bfloat16, torch.float16


def compute_type(c):
    return c.dtype if c.kv_dtype == c.dtype else HF


def parts(c):
    return 1 if c.kv_dtype != c.dtype and c.dtype == BF else 2


def heads(c, b, pool, q_scaling=1.0):
    """For every query head of sequence b: (rows of the result, columns, q / sqrt(D) [n, D], k, v [keys, D] double, hidden)."""
    Hq, Hkv, D, G, tpb = c.Hq, c.Hkv, c.D, c.Hq // c.Hkv, c.tpb
    lo, n, past = int(c.offsets[b]), c.n[b], c.past[b]
    x = c.qkv[lo:lo + n].double()
    if c.bias is not None:
        x = x + c.bias.double()
    x = x.view(n, Hq + 2 * Hkv, D)[:, :Hq]
    if c.rope:
        x = rotate(x, angles(past + c.depth[lo:lo + n], c.rot_dim, **c.rope_args), c.rope, c.rot_dim)
    raw = pool.view(torch.int8) if c.kv_dtype == torch.float8_e4m3fn else pool
    blocks = torch.from_numpy(c.table[b, :-(-(past + n) // tpb)])
    hidden = ~c.seen(b)
    for h in range(Hkv):
        k, v = (raw[half, blocks, h].reshape(-1, D)[:past + n].view(pool.dtype).double() * c.kv_scale for half in range(2))
        for g in range(G):
            at = (h * G + g) * D
            yield slice(lo, lo + n), slice(at, at + D), x[:, h * G + g] / (math.sqrt(D) * q_scaling), k, v, hidden


def weights(q, k, hidden):
    s = q @ k.t()
    s[hidden] = -math.inf
    empty = hidden.all(1)
    s[empty] = 0.0
    w = torch.softmax(s, -1)
    w[hidden] = 0.0
    return s, w


def definition(c, pool, q_scaling=1.0):
    """(out, bound, variance), each [tokens, Hq * D] double, NaN outside the sequences; `pool` after the call."""
    u, uc, one = UNIT[c.dtype], UNIT[compute_type(c)], parts(c) == 1
    out = torch.full((c.tokens, c.Hq * c.D), float("nan"), dtype=torch.float64)
    bound, variance = out.clone(), out.clone()
    for b in range(len(c.past)):
        if c.n[b] == 0:
            continue
        for rows, cols, q, k, v, hidden in heads(c, b, pool, q_scaling):
            s, w = weights(q, k, hidden)
            o = w @ v
            # keys of weight 0 (in 64 bits) add nothing, however their scores are rounded
            dead = hidden | (w == 0)
            A = (q.abs() @ torch.nan_to_num(k, posinf=0.0, neginf=0.0).abs().t()).masked_fill(dead, 0.0).amax(1, keepdim=True)
            top = s.masked_fill(dead, 0.0).abs().amax(1, keepdim=True)
            moved = ((uc if one else uc * uc) + 2.0 ** -21) * A + 64 * 2.0 ** -24 * (A + top)
            if compute_type(c) == HF:
                ks = (k / c.kv_scale).abs().sum(1)
                moved = moved + math.log(2) * 2.0 ** -25 * torch.where(torch.isfinite(ks), ks, torch.zeros_like(ks)).max()
            av = w @ v.abs()
            out[rows, cols] = o
            bound[rows, cols] = (torch.expm1(2 * moved) + uc + 2.0 ** -16) * av + u * o.abs() + 1e-7
            var = uc * uc / 3 * (w * w) @ (v * v) + u * u / 3 * o * o
            if one:  # q's rounding moves all scores of a row together: out changes by sum_t w_t (e . k_t) (v_t - o)
                kv = torch.einsum("it,td,tj->idj", w, k, v) - (w @ k)[:, :, None] * o[:, None]
                var = var + torch.einsum("id,idj->ij", (uc * q) ** 2 / 3, kv * kv)
            variance[rows, cols] = var
    return out, bound, variance


def model(c, pool, q_parts=None):
    """What the kernel's arithmetic gives with q in `q_parts` parts: every rounding it chooses, the sums exact."""
    C, q_parts = compute_type(c), q_parts or parts(c)
    out = torch.full((c.tokens, c.Hq * c.D), float("nan"), dtype=torch.float64)
    for b in range(len(c.past)):
        for rows, cols, q, k, v, hidden in heads(c, b, pool):
            z = q * (math.log2(math.e) * c.kv_scale)
            held = z.to(C).double()
            if q_parts == 2:
                held = held + (z - held).to(C).double()
            s = held @ (k / c.kv_scale).t()
            s[hidden] = -math.inf
            p = torch.exp2(s - s.amax(1, keepdim=True))
            out[rows, cols] = (p.to(C).double() @ v / p.sum(1, keepdim=True)).to(c.dtype).double()
    return out


def wrong_with(out, ref, bound, variance):
    """None, or what is wrong with `out` [tokens, Hq * D] against the definition."""
    live = ~bound.isnan().all(1)
    o, r, t, var = out.double()[live], ref[live], bound[live], variance[live]
    fine = torch.isfinite(r)
    if not torch.equal(o.isnan(), r.isnan()) or not torch.equal(o[~fine & ~r.isnan()], r[~fine & ~r.isnan()]):
        return "infinities or NaN in other places"
    err = (o - r).abs()[fine]
    if not (err <= t[fine]).all():
        return f"error {err.max().item():.3g}, {(err / t[fine]).max().item():.3g} times its bound"
    # (the mean over a thousand or more roundings stays within a tenth of its expectation, which is at most 0.74 of the limit:
    # a value's step is 1 to 1/2 of what `variance` takes)
    if err.numel() >= 1000:
        ratio = (err.square().mean() / var[fine].mean()).sqrt().item()
        if ratio > 1:
            return f"rms error {ratio:.3g} times that of the roundings"
    return None
