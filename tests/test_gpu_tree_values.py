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


def spoil(v, lens, dim, kv=1):
    """Non-finite values in cached rows: columns and what every row that sees them gets there.  Keys of several tiles, the
    first and the last cached one among them."""
    inf, nan = float("inf"), float("nan")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = [0, n // 3, n // 2, n - 1]
        v[b, kv, at[0], 2] = inf
        v[b, kv, at[1], 5] = -inf
        v[b, kv, at[2], 5] = -inf
        v[b, kv, at[0], 9], v[b, kv, at[3], 9] = inf, -inf
        v[b, kv, at[2], 33], v[b, kv, at[3], 33] = inf, nan
        v[b, kv, at[3], dim - 1] = inf
    return {2: inf, 5: -inf, 9: nan, 33: nan, dim - 1: inf}


def same(a, value):
    import torch
    return (torch.isnan(a) if value != value else a == value).all()


@pytest.mark.parametrize("ctas", [0, 2])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n_tok,heads,kv_heads,dim", LAYOUTS)
def test_cached_infinities(ctx, dtype, n_tok, heads, kv_heads, dim, ctas):
    """An infinite cached value makes its column infinite with its sign in every row of its kv head, whatever the weight it
    has there; both signs, or NaN, make it NaN.  A drafted infinity of the other sign makes it NaN for those that see it."""
    import torch
    lens, new = [700, 0, 257], [n_tok, n_tok - 1, n_tok]
    q, k, v, see, mask = inputs(dtype, n_tok, heads, kv_heads, dim, lens)
    q = q * 6  # weights from 1 to far below fp16's smallest
    G = heads // kv_heads
    clean = v.clone()
    columns = spoil(v, lens, dim)
    o = call(ctx, q, k, v, lens, new, mask, ctas)
    for b in (0, 2):
        for d, value in columns.items():
            assert same(o[b, :new[b], G:2 * G, d], value), (b, d)
    rest = [d for d in range(dim) if d not in columns]
    inside(o, q, k, clean, lens, new, see, dtype, rest)
    for b in (0, 2):
        v[b, 1, lens[b] + 1, 2] = float("-inf")
        v[b, 1, lens[b] + 1, 5] = float("-inf")
    o = call(ctx, q, k, v, lens, new, mask, ctas)
    for b in (0, 2):
        sees = torch.from_numpy(see[b, :new[b], 1]).cuda()
        got = o[b, :new[b], G:2 * G]
        assert same(got[sees][..., 2], float("nan")) and same(got[~sees][..., 2], float("inf"))
        assert same(got[..., 5], float("-inf"))


@pytest.mark.parametrize("ctas", [0, 2])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_cached_infinities_with_weights(ctx, dtype, dim, ctas):
    """The same for the decode with weights, whose weights are those of finite values, bit for bit."""
    import cache_cases as C
    import mako_attn
    import torch
    lens, H, KV = [700, 0, 257, 1], 8, 2
    q = C.randn(1, 4, H, dim, dtype=dtype) * 6
    k, clean = C.randn(2, 4, KV, 700, dim, dtype=dtype), C.randn(3, 4, KV, 700, dim, dtype=dtype)
    v = clean.clone()
    columns = spoil(v, lens[:3], dim)

    def decode(v):
        o, w = torch.full((4, H * dim), 5.0, device="cuda"), torch.zeros(4, KV, 700, device="cuda")
        ctx.set_option(mako_attn.OPT_GRID_CTAS, ctas)
        try:
            ctx.attention_decode_weights(q, k, v, o, w, C.i32(lens), 700, H, KV, dim, 700)
        finally:
            ctx.set_option(mako_attn.OPT_GRID_CTAS, 0)
        torch.cuda.synchronize()
        assert ctx.device_error() == 0
        return o.view(4, H, dim), w

    base, w0 = decode(clean)
    o, w = decode(v)
    assert torch.equal(w, w0)
    rest = [d for d in range(dim) if d not in columns]
    assert torch.equal(o[..., rest], base[..., rest]) and torch.equal(o[:, :4], base[:, :4])
    for b in (0, 2):
        for d, value in columns.items():
            assert same(o[b, 4:, d], value), (b, d)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
def test_merged_streams_repeat(ctx, dtype, dim):
    """Segments of one tile (whose second stream has none) to three, many a CTA: each of many calls gives the same bits,
    within the bound."""
    import torch
    lens = [int(n) for n in np.random.default_rng(3).integers(0, 380, 60)]
    new = [5] * 60
    q, k, v, see, mask = inputs(dtype, 5, 8, 4, dim, lens)
    base = call(ctx, q, k, v, lens, new, mask, 7)
    inside(base, q, k, v, lens, new, see, dtype)
    for ctas in (7, 3, 29, 0):
        first = call(ctx, q, k, v, lens, new, mask, ctas)
        for _ in range(10):
            assert torch.equal(call(ctx, q, k, v, lens, new, mask, ctas), first)


@pytest.mark.parametrize("ctas", [0, 1, 3])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n_tok,heads,kv_heads,dim", LAYOUTS)
def test_values_that_are_not_finite(ctx, dtype, n_tok, heads, kv_heads, dim, ctas):
    """NaN and infinities past the draft and in drafted values and keys: rows that do not see them keep their bits, rows
    that do are infinite or NaN in those columns, or NaN whole for a key."""
    import torch
    lens, new, j, G = [190, 0, 700], [n_tok, n_tok - 1, n_tok], 1, heads // kv_heads
    q, k, v, see, mask = inputs(dtype, n_tok, heads, kv_heads, dim, lens)
    base = call(ctx, q, k, v, lens, new, mask, ctas)
    inside(base, q, k, v, lens, new, see, dtype)
    for b in range(3):
        k[b, :, lens[b] + new[b]:] = float("nan")
        v[b, :, lens[b] + new[b]:] = float("inf")
    assert torch.equal(call(ctx, q, k, v, lens, new, mask, ctas), base)
    k2, v2 = k.clone(), v.clone()
    for b in range(3):
        v2[b, 1, lens[b] + j, 3] = float("nan")
        v2[b, 1, lens[b] + j, dim - 1] = float("-inf")
        v2[b, 1, lens[b] + n_tok - 2, dim - 1] = float("inf")
        k2[b, 0, lens[b] + j] = float("nan")
    got = call(ctx, q, k, v2, lens, new, mask, ctas)
    rest = [d for d in range(dim) if d not in (3, dim - 1)]
    for b in range(3):
        s, t = (torch.from_numpy(see[b, :new[b], x]).cuda() for x in (j, n_tok - 2))
        g, w = got[b, :new[b]], base[b, :new[b]]
        assert torch.equal(g[:, :G], w[:, :G]) and torch.equal(g[..., rest], w[..., rest])
        assert torch.equal(g[~s][..., 3], w[~s][..., 3]) and torch.equal(g[~s & ~t], w[~s & ~t])
        assert same(g[s][:, G:2 * G, 3], float("nan")) and same(g[s & ~t][:, G:2 * G, dim - 1], float("-inf"))
        assert same(g[s & t][:, G:2 * G, dim - 1], float("nan")) and same(g[t & ~s][:, G:2 * G, dim - 1], float("inf"))
    got = call(ctx, q, k2, v, lens, new, mask, ctas)
    for b in range(3):
        s = torch.from_numpy(see[b, :new[b], j]).cuda()
        g, w = got[b, :new[b]], base[b, :new[b]]
        assert torch.equal(g[~s], w[~s]) and torch.equal(g[:, G:], w[:, G:]) and same(g[s][:, :G], float("nan"))


@pytest.mark.parametrize("ctas", [0, 1, 3])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n_tok,heads,kv_heads,dim", LAYOUTS)
def test_maxima_that_move(ctx, dtype, n_tok, heads, kv_heads, dim, ctas):
    """Scores that rise by more than 8 from tile to tile, for some rows and not for others, so that sums and outputs are
    rescaled on the way; and scores in the thousands."""
    import torch
    lens, new = [900, 130], [n_tok, n_tok]
    q, k, v, see, mask = inputs(dtype, n_tok, heads, kv_heads, dim, lens)
    inside(call(ctx, q * 20, k * 10, v, lens, new, mask, ctas), q * 20, k * 10, v, lens, new, see, dtype)
    # keys along one direction, growing with their row; every other token looks that way, the others away from it
    along = (torch.arange(k.shape[2], device="cuda") / 100.0)[:, None].to(k.dtype)
    k = (0.1 * k + along).contiguous()
    sign = torch.tensor([1.0, -1.0], device="cuda").repeat(n_tok)[:n_tok, None, None].to(q.dtype)
    q = (0.5 * q + sign).contiguous()
    inside(call(ctx, q, k, v, lens, new, mask, ctas), q, k, v, lens, new, see, dtype)


@pytest.mark.parametrize("exponent", [25.1, 20.5, 16.3])
@pytest.mark.parametrize("dtype,n_tok,heads,dim", [(0, 5, 2, 128), (0, 70, 2, 128), (1, 5, 2, 128), (1, 70, 2, 128),
                                                   (0, 70, 2, 64), (1, 70, 2, 64), (0, 5, 2, 256), (1, 70, 2, 256)])
def test_many_small_weights(ctx, dtype, n_tok, heads, dim, exponent):
    """One key of weight 1 beside 32768 of 2^-exponent, all of one CTA, and values of 1: o is 1.  The products are added to a
    sum of 24 bits, which is never above o's own, and what lies below its last bit is cut off: 2^-23 of it a key at most,
    2^-8 in all.  P's own error is 2^-11 of each of the small ones, 2^-6 for the first exponent, whose share of the sum
    is below 2^-10: 2^-11 at most."""
    import cache_cases as C
    L = 32769
    q = C.randn(1, 1, n_tok, heads, dim, dtype=dtype) * 0 + 1
    k = C.randn(2, 1, 1, L + n_tok + 30, dim, dtype=dtype) * 0
    k[0, 0, 0] = exponent * 0.6931471805599453 / dim ** 0.5
    o = call(ctx, q, k, k * 0 + 1, [L], [n_tok], None, 1)
    assert ((o.double() - 1).abs() <= 2.0 ** -8 + 2.0 ** -11).all()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,scale", [(8, 2, 1.0), (7, 1, 1.0), (40, 2, 1.0), (8, 8, 12.0)])
def test_decode_with_weights_is_decode(ctx, dtype, dim, heads, kv_heads, scale):
    """The decode with weights gives softmax's output within the bound of two-part weights for bf16, and what
    attention_decode gives over the same cache, whose own error is bounded alike, within both bounds; the weights of a kv
    head sum to its query heads."""
    import cache_cases as C
    import torch
    lens, G = [1500, 0, 77, 1], heads // kv_heads
    q = C.randn(1, 4, heads, dim, dtype=dtype) * scale
    k, v = C.randn(2, 4, kv_heads, 1500, dim, dtype=dtype), C.randn(3, 4, kv_heads, 1500, dim, dtype=dtype)
    a, d = (torch.full((4, heads * dim), 3.0, device="cuda") for _ in range(2))
    w = torch.zeros(4, kv_heads, 1500, device="cuda")
    ctx.attention_decode_weights(q, k, v, a, w, C.i32(lens), 1500, heads, kv_heads, dim, 1500)
    ctx.attention_decode(q, k, v, d, C.i32(lens), 1500, heads, kv_heads, dim, 1500)
    for b, n in enumerate(lens):
        if n == 0:
            assert (a[b] == 0).all() and (d[b] == 0).all() and (w[b] == 0).all()
            continue
        want, tol = want_rows(q[b][None], k[b], v[b], n - 1, 1, np.ones((1, 1), bool), dtype)
        x, y = (t[b].view(1, heads, dim).double() for t in (a, d))
        assert ((x - want).abs() <= tol).all() and ((x - y).abs() <= 2 * tol).all()
        # each weight within 2^-11 of itself for scores of tens in fp32 (dim * 2^-24 * 2 * sum |q k| / sqrt(dim))
        assert ((w[b].double().sum(-1) - G).abs() <= G * 2.0 ** -11).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n_tok,heads,kv_heads", [(1, 8, 8), (5, 8, 2), (33, 6, 2), (64, 8, 2), (129, 2, 1)])
def test_two_part_weights(ctx, monkeypatch, dim, n_tok, heads, kv_heads):
    """bf16 within the bound of P in two parts and exact values, at the sizes of the tests of shapes: one part would be
    2^-9 off."""
    import cache_cases as C
    import test_gpu_cache_evict as E
    import test_gpu_tree as T
    monkeypatch.setattr(C, "P_STEP", {0: 2.0 ** -11, 1: 2.0 ** -16})
    monkeypatch.setattr(C, "V_STEP", {0: 0.0, 1: 0.0})
    T.run(ctx, 1, n_tok, heads, kv_heads, dim, [700, 0, 129], seed=n_tok + dim)
    T.run(ctx, 1, n_tok, heads, kv_heads, dim, [0, 1500, 3, 200, 700], new=[n_tok, 5, 1, 0, n_tok], k_stride=1800, ctas=3)
    E.check_weights(ctx, 1, heads, kv_heads, dim, [700, 0, 129, -4, 1, 3000], seed=heads + dim)
