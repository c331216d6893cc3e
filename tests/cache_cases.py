"""Inputs and 64-bit references of the cache operators' tests (torch, on the GPU)."""
import math

import numpy as np
import torch

DT = {0: torch.float16, 1: torch.bfloat16}
HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}  # of the 16-bit type, relative
# P is rounded to fp16 (2^-11 of p at most), for bf16 caches too where there are many rows and 16 keys' largest value lies in
# [2^-8, 2^16): those values then go through fp16, exact but below 2^-14, where they are off by at most 2^-25, under 2^-17
# of that largest.  Else P is the bf16 of p and the bf16 of what that left over, 2^-16 of p.
P_STEP = {0: 2.0 ** -11, 1: 2.0 ** -11}
V_STEP = {0: 0.0, 1: 2.0 ** -25}


def randn(seed, *shape, dtype=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(DT[dtype]).cuda()


def i32(a):
    return torch.as_tensor(np.asarray(a, np.int32)).cuda()


def random_tree(seed, batch, n):
    """see [batch][n][n] (a token sees itself and its ancestors) and its words."""
    rs = np.random.default_rng(seed)
    see = np.zeros((batch, n, n), bool)
    for b in range(batch):
        for i in range(n):
            parent = i - 1 - int(rs.integers(0, 4))
            if parent >= 0:
                see[b, i] = see[b, parent]
            see[b, i, i] = True
    return see, words(see)


def words(see):
    batch, n, _ = see.shape
    w = (n + 31) // 32
    bits = np.zeros((batch, n, w * 32), np.uint64)
    bits[:, :, :n] = see
    out = (bits.reshape(batch, n, w, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return torch.from_numpy(out.astype(np.uint32).view(np.int32)).cuda()


def attend(q, k, v, see, dtype):
    """q [rows][dim], k, v [keys][dim], see [rows][keys] -> (o, weights, bound on |error| of an fp32 o, relative bound on
    the weights' error) in 64 bits.

    A score sums dim products in fp32: it is off by at most dim * 2^-24 * sum |q k| / sqrt(dim), the row's largest of
    which is e; a weight e^s and the sum it is divided by are off by that relatively, plus 2^-21 for the exponential and
    the division, plus keys * 2^-24 for the sum.  Then o is off by those and P's rounding, times sum_j p_j |v_j|, and by V's
    own."""
    q, k, v = q.double(), k.double(), v.double()
    dim, keys = q.shape[1], max(k.shape[0], 1)
    scale = 1.0 / math.sqrt(dim)
    if k.shape[0] == 0:
        z = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
        return z, torch.zeros(q.shape[0], 0, dtype=torch.float64, device=q.device), z, torch.zeros(q.shape[0], 1, device=q.device)
    s = (q @ k.T * scale).masked_fill(~see, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))
    e = ((q.abs() @ k.abs().T) * scale * see).amax(-1, keepdim=True) * dim * 2.0 ** -24
    rel = 2.0 * e + 2.0 ** -21 + keys * 2.0 ** -24
    return p @ v, p, (rel + keys * 2.0 ** -24 + P_STEP[dtype]) * (p @ v.abs()) + V_STEP[dtype], rel
