"""Attention over the paged 8-bit cache in 16 bits: outputs as good as their own rounding, for every number of rows.

The reference is the softmax in 64 bits over the K and V that q4hip_kv8_read gives.
"""
import math

import numpy as np
import pytest
import torch

import q4hip

pytestmark = pytest.mark.gpu

TYPES = {"f16": (q4hip.F16, torch.float16), "bf16": (q4hip.BF16, torch.bfloat16)}


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def exact(q, K, V, have, rows):
    """[len(rows)][heads][head_dim] in 64 bits: attention of the given rows of q [n][heads][head_dim], the first of which lies at
    `have`, over K, V [positions][kv heads][head_dim]."""
    n, H, hd = q.shape
    G, L = H // K.shape[1], K.shape[0]
    out = torch.empty(len(rows), H, hd, dtype=torch.float64, device="cuda")
    seen = torch.arange(L, device="cuda")[None] <= have + torch.tensor(rows, device="cuda")[:, None]
    for h in range(H):
        s = torch.mm(q[rows, h].double(), K[:, h // G].double().t().contiguous()) / math.sqrt(hd)
        p = torch.softmax(torch.where(seen, s, s.new_full((), -math.inf)), 1)
        out[:, h] = torch.mm(p, V[:, h // G].double().contiguous())
    return out


def quotient(H, KVH, hd, have, add, dtype, size):
    """The root of the mean square of the outputs' error over that of their rounding alone, on columns of different size."""
    typ, t = TYPES[dtype]
    g = torch.Generator(device="cuda")
    g.manual_seed(H + hd + add)
    L = have + add
    kv = q4hip.Kv8(1, H, KVH, hd, 1, L, -(-L // 32), L)
    cols = torch.exp(0.5 * torch.randn(2, KVH * hd, generator=g, device="cuda"))
    k, v = ((torch.randn(L, KVH * hd, generator=g, device="cuda") * c).to(t) for c in cols)
    q = (size * torch.randn(add, H * hd, generator=g, device="cuda")).to(t)
    out = torch.empty_like(q)
    zero, hold, more, all_ = ints([0]), ints([have]), ints([add]), ints([L])
    torch.cuda.synchronize()
    kv.plan(zero.data_ptr(), all_.data_ptr(), L)
    kv.append(0, k.data_ptr(), v.data_ptr(), typ, KVH * hd, KVH * hd)
    kv.plan(hold.data_ptr(), more.data_ptr(), add)
    kv.attend(0, q.data_ptr(), out.data_ptr(), typ, H * hd, H * hd)
    seq, pos = ints(np.zeros(L)), ints(np.arange(L))
    K, V = (torch.empty(L, KVH, hd, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    kv.read(0, seq.data_ptr(), pos.data_ptr(), L, K.data_ptr(), V.data_ptr())
    rows = sorted(set(np.linspace(0, add - 1, 40).astype(int).tolist()))
    want = exact(q.view(add, H, hd), K, V, have, rows)
    err = (out.view(add, H, hd)[rows].double() - want).square().sum()
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
