"""What values do to mako_attention_tree and mako_attention_decode_weights in each of their layouts: up to 128 rows a kv
head, more, and 256-wide heads.

The bound on an output is that of cache_cases.attend with P's rounding as the type has it.  bf16: P is the bf16 of p and the
bf16 of what that left over, 2^-16 of p.  fp16: P is fp16, 2^-11 of p, and as it is held 2^7 up in steps of 2^-24 at least,
2^-32 of the largest weight where p is small.  V is exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# n_tok, heads, kv_heads, dim
NARROW = [(9, 8, 2, 64), (9, 8, 2, 128)]
WIDE = [(40, 8, 2, 64), (40, 8, 2, 128)]
BROAD = [(9, 8, 2, 256), (40, 8, 2, 256)]
LAYOUTS = NARROW + WIDE + BROAD


def want_rows(q, k, v, cached, new, see, dtype):
    """o and its bound for one sequence: q [n][heads][dim], k, v [kv][S][dim], see [n][n]."""
    import cache_cases as C
    import torch
    n, H, D = q.shape
    G = H // k.shape[0]
    o = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    vis = torch.cat([torch.ones(new, cached, dtype=torch.bool), torch.from_numpy(see[:new, :new])], 1).cuda()
    for h in range(H):
        kk, vv = k[h // G, :cached + new], v[h // G, :cached + new]
        o[:new, h], p, _, rel = C.attend(q[:new, h], kk, vv, vis, dtype)
        size = vv.double().abs()
        tol[:new, h] = (rel + (cached + new) * 2.0 ** -24 + (2.0 ** -16 if dtype else 2.0 ** -11)) * (p @ size)
        if not dtype:
            tol[:new, h] += 2.0 ** -32 * (vis.double() @ size)
    return o, tol


def call(ctx, q, k, v, lens, new, mask, ctas=0):
    """o [batch][n_tok][heads][dim]."""
    import cache_cases as C
    import mako_attn
    import torch
    B, n, H, D = q.shape
    KV, S = k.shape[1:3]
    o = torch.full((B, n, H * D), 5.0, device="cuda")
    ctx.set_option(mako_attn.OPT_GRID_CTAS, ctas)
    try:
        ctx.attention_tree(q, k, v, o, B, n, C.i32(new), C.i32(lens), max(lens), H, KV, D, S, mask)
    finally:
        ctx.set_option(mako_attn.OPT_GRID_CTAS, 0)
    torch.cuda.synchronize()
    assert ctx.device_error() == 0
    return o.view(B, n, H, D)


def inputs(dtype, n_tok, heads, kv_heads, dim, lens, seed=1):
    import cache_cases as C
    B, S = len(lens), max(lens) + n_tok + 30
    q = C.randn(seed, B, n_tok, heads, dim, dtype=dtype)
    k, v = (C.randn(seed + i, B, kv_heads, S, dim, dtype=dtype) for i in (1, 2))
    return (q, k, v) + C.random_tree(seed + 3, B, n_tok)


def inside(o, q, k, v, lens, new, see, dtype, columns=slice(None)):
    for b in range(len(lens)):
        want, tol = want_rows(q[b], k[b], v[b], lens[b], new[b], see[b], dtype)
        over = ((o[b].double() - want).abs() - tol - 1e-45)[:new[b]][..., columns]
        assert over.max() <= 0, (b, float(over.max()))


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n_tok,heads,kv_heads,dim", LAYOUTS)
def test_values_of_unseen_drafts(ctx, dtype, n_tok, heads, kv_heads, dim):
    """A drafted token's finite values, large, small or zero, leave the bits of rows that do not see it as they are, also
    where it shares sixteen keys with cached ones."""
    lens, new = [190, 0, 257], [n_tok, n_tok - 1, n_tok]
    q, k, v, see, mask = inputs(dtype, n_tok, heads, kv_heads, dim, lens)
    base = call(ctx, q, k, v, lens, new, mask)
    j = 1
    for value in (2.0 ** 15, 0.0) if dtype == 0 else (2.0 ** 17, -2.0 ** 100, 2.0 ** -30, 0.0):
        k2, v2 = k.clone(), v.clone()
        for b in range(3):
            k2[b, :, lens[b] + j] *= 30.0
            v2[b, :, lens[b] + j] = value
        got = call(ctx, q, k2, v2, lens, new, mask)
        for b in range(3):
            blind = np.flatnonzero(~see[b, :new[b], j])
            assert blind.size
            assert (got[b, blind] == base[b, blind]).all(), (value, b)


@pytest.mark.parametrize("n_tok,heads,kv_heads,dim", LAYOUTS)
def test_small_columns(ctx, n_tok, heads, kv_heads, dim):
    """bf16 value columns that are small beside the others, from ones that fp16 still holds to ones far below it: each is
    as exact as the large ones.  First in all keys, then in every third group of sixteen."""
    import torch
    lens, new = [500, 33], [n_tok, n_tok - 2]
    q, k, v0, see, mask = inputs(1, n_tok, heads, kv_heads, dim, lens)
    scales = torch.tensor([1.0, 2.0 ** -12, 2.0 ** -16, 2.0 ** -18, 2.0 ** -20, 2.0 ** -26, 2.0 ** -60, 0.0],
                          device="cuda").repeat(dim // 8)
    group = torch.arange(v0.shape[2], device="cuda")[:, None] // 16
    for scale in (scales, torch.where(group % 3 == 1, scales, 1.0)):
        v = (v0.float() * scale).to(torch.bfloat16)
        inside(call(ctx, q, k, v, lens, new, mask), q, k, v, lens, new, see, 1)
