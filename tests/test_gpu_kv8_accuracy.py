"""Attention over the paged 8-bit cache: outputs of 16 bits as good as their own rounding, for every number of rows; V of zeros and
of very different size.

The reference is the softmax in 64 bits over the K and V that q4hip_kv8_read gives.
"""
import math

import numpy as np
import pytest
import torch

import q4hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": (q4hip.F32, torch.float32), "f16": (q4hip.F16, torch.float16), "bf16": (q4hip.BF16, torch.bfloat16)}


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def exact(q, K, V, have, rows, most=False):
    """[len(rows)][heads][head_dim] in 64 bits: attention of the given rows of q [n][heads][head_dim], the first of which lies at
    `have`, over K, V [positions][kv heads][head_dim]; most: the largest probabilities instead."""
    n, H, hd = q.shape
    G, L = H // K.shape[1], K.shape[0]
    out = torch.empty(len(rows), H, hd, dtype=torch.float64, device="cuda")
    seen = torch.arange(L, device="cuda")[None] <= have + torch.tensor(rows, device="cuda")[:, None]
    for h in range(H):
        s = torch.mm(q[rows, h].double(), K[:, h // G].double().t().contiguous()) / math.sqrt(hd)
        p = torch.softmax(torch.where(seen, s, s.new_full((), -math.inf)), 1)
        out[:, h] = p.amax(1, keepdim=True) if most else torch.mm(p, V[:, h // G].double().contiguous())
    return out


def attend(q, k, v, have, KVH, hd):
    """(outputs, K, V the cache stands for) of the rows q [n][heads * head_dim] of one sequence, behind `have` positions of
    k, v [have + n][KVH * hd]."""
    n, L = q.shape[0], k.shape[0]
    typ = next(a for a, t in TYPES.values() if t == q.dtype)
    kv = q4hip.Kv8(1, q.shape[1] // hd, KVH, hd, 1, L, -(-L // 32), L)
    out = torch.empty_like(q)
    zero, hold, more, all_ = ints([0]), ints([have]), ints([n]), ints([L])
    torch.cuda.synchronize()
    kv.plan(zero.data_ptr(), all_.data_ptr(), L)
    kv.append(0, k.data_ptr(), v.data_ptr(), typ, KVH * hd, KVH * hd)
    kv.plan(hold.data_ptr(), more.data_ptr(), n)
    kv.attend(0, q.data_ptr(), out.data_ptr(), typ, q.shape[1], q.shape[1])
    seq, pos = ints(np.zeros(L)), ints(np.arange(L))
    K, V = (torch.empty(L, KVH, hd, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    kv.read(0, seq.data_ptr(), pos.data_ptr(), L, K.data_ptr(), V.data_ptr())
    return out.view(n, -1, hd), K, V


def some(n):
    return sorted(set(np.linspace(0, n - 1, 40).astype(int).tolist()))


def quotient(H, KVH, hd, have, add, dtype, size):
    """The root of the mean square of the outputs' error over that of their rounding alone, on columns of different size."""
    t = TYPES[dtype][1]
    g = torch.Generator(device="cuda")
    g.manual_seed(H + hd + add)
    cols = torch.exp(0.5 * torch.randn(2, KVH * hd, generator=g, device="cuda"))
    k, v = ((torch.randn(have + add, KVH * hd, generator=g, device="cuda") * c).to(t) for c in cols)
    q = (size * torch.randn(add, H * hd, generator=g, device="cuda")).to(t)
    out, K, V = attend(q, k, v, have, KVH, hd)
    rows = some(add)
    want = exact(q.view(add, H, hd), K, V, have, rows)
    err = (out[rows].double() - want).square().sum()
    rounding = (want.to(t).double() - want).square().sum()
    return float((err / rounding).sqrt())


@pytest.mark.parametrize("dtype,most", [("f16", 1.03), ("bf16", 1.003)])
@pytest.mark.parametrize("H,KVH,hd,have,add", [
    (14, 2, 64, 131072, 1),          # a token, its pages shared
    (12, 2, 128, 3000, 1),
    (14, 2, 64, 4000, 3),            # a turn of a few rows
    (32, 8, 128, 4000, 40),          # units of 32 rows
    (20, 20, 64, 4000, 4100),        # tiles
    (8, 1, 128, 60000, 700)])
def test_outputs_are_as_good_as_their_rounding(H, KVH, hd, have, add, dtype, most):
    """What the kernel adds before it rounds, d, makes the quotient 1 + d / r at most, r the rounding.  Relative to an output, r
    is 2^-12 to 2^-11 of fp16 over sqrt(3), some 2e-4, and 8 times that of bf16.  d has three parts, each of random sign among the
    positions, so that they cancel as the values do and stay relative to the output: the weights' two fp16 numbers, 2^-22;
    the fp32 scores' rounding, here of S = 0.05 * scale * sum |q K| < 0.05 * 4 of the products' 128 summands plus K's 128
    codes, (128 + 8) 2^-24 * 5 S at the very most, 8e-6, in the mean of random signs a tenth of it; the sums' fp32 roundings,
    sqrt(n / 32) 2^-24 / sqrt(32) of what they hold, < 2e-6.  So d < 4e-6: d / r < 0.02 of fp16 and < 0.0025 of bf16.  One fp16
    number for the weights, off by up to 2^-11, makes the quotient 1.3 to 1.4 of fp16 and 1.005 to 1.008 of bf16."""
    assert quotient(H, KVH, hd, have, add, dtype, 0.05) < most


def test_a_long_token_with_weights_far_apart():
    """Queries of size 1 on keys of size 1.3: weights from 2^-14 to 1 of the largest.  d as above, but for the scores, whose
    sums hold 128 scale |sum of q| * 0.12 = 15 * 0.125 * 8: roundings of 2^-25 of that in 32 steps of random sign make
    sqrt(32) 2^-25 * 15 = 2.5e-6.  d < 6e-6: below 1.03.  Code + 128 in the sums of V makes it 1.28."""
    assert quotient(14, 2, 64, 131072, 1, "f16", 1.0) < 1.03


@pytest.mark.parametrize("dtype,lead,size", [("f32", 0.0, 1.0), ("f16", 0.0, 1.0), ("bf16", 0.0, 1.0), ("f16", 0.0, 3e4),
                                             ("f32", 0.0, 1e15), ("bf16", 0.0, 1e30), ("f32", 1e-28, 1.0), ("bf16", 1e-28, 1e25),
                                             ("f32", 1e25, 1e-20), ("bf16", 1e25, 1e-20)])
@pytest.mark.parametrize("H,KVH,hd,add", [(14, 2, 64, 1),          # a token, its pages shared
                                          (14, 2, 64, 3),
                                          (12, 2, 128, 40),        # units of 32 rows
                                          (20, 20, 64, 4100),      # tiles
                                          (20, 10, 128, 4100)])
@pytest.mark.parametrize("rise", [0.0, 40.0])
def test_values_of_very_different_size(H, KVH, hd, add, dtype, lead, size, rise):
    """20,000 positions whose V has the size `lead`, zeros among them, then 400 and the rows of size `size`; the scores of the last 10 of
    the 400 are higher by `rise`.  With A = sum_j p_j |V_j| of a row and column, L positions, and the error of a score
    ds = S ((hd + 8) 2^-24 + 2^-22), S the largest scale * sum_d |q_d| (|K_jd| + 128 k_j) (k_j: K's scale, at most 2 / 127 of a
    page's largest, so that 128 k_j < 2.02 max|K|): the probabilities' errors make A (e^(2 ds) - 1), the sums' A (L / 32 + 48) 2^-23,
    the two fp16 numbers of a weight A 2^-22, and what is below fp16 at 2^-38 of the largest p_j v_j, v_j the V scale, for each
    position times its code, L 2^-38 max p max|V|.  Then `out` is rounded.  A V whose share is lost in l, or one that makes l infinite,
    is off by whole multiples of A."""
    t = TYPES[dtype][1]
    g = torch.Generator(device="cuda")
    g.manual_seed(add)
    have, L = 20400, 20400 + add
    k, v = (torch.randn(L, KVH * hd, generator=g, device="cuda") for _ in range(2))
    v[:20000] *= lead
    v[20000:] *= size
    q = 0.05 * torch.randn(add, H * hd, generator=g, device="cuda")
    if rise:
        q.view(add, H, hd)[:, :, 0] = 1
        k.view(L, KVH, hd)[:, :, 0] = 0
        k.view(L, KVH, hd)[20390:20400, :, 0] = rise * math.sqrt(hd)
    q, k, v = (x.to(t) for x in (q, k, v))
    out, K, V = attend(q, k, v, have, KVH, hd)
    rows = some(add)
    y = q.view(add, H, hd)
    want, A, p = exact(y, K, V, have, rows), exact(y, K, V.abs(), have, rows), exact(y, K, V, have, rows, most=True)
    S = hd ** -0.5 * y[rows].double().abs().sum(2, keepdim=True) * 3.02 * K.double().abs().max()
    bound = A * (torch.expm1(2 * S * ((hd + 8) * 2.0 ** -24 + 2.0 ** -22)) + (L / 32 + 48) * 2.0 ** -23 + 2.0 ** -22)
    bound = bound + L * 2.0 ** -38 * p * V.double().abs().max()
    bound = bound + (want.abs() + bound) * torch.finfo(t).eps / 2
    err = (out[rows].double() - want).abs()
    assert (err <= bound).all(), float((err / bound).nan_to_num(1e9).max())
