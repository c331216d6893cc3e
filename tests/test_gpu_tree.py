"""mako_attention_tree against softmax in 64 bits; the bound on each value's error is cache_cases.attend's, plus half a
step where o is 16-bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def want_rows(q, k, v, cached, new, see, dtype):
    """o and its bound for one sequence: q [n][heads][dim], k, v [kv][S][dim]."""
    import cache_cases as C
    import torch
    n, H, D = q.shape
    KV = k.shape[0]
    G = H // KV
    o = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    vis = torch.cat([torch.ones(new, cached, dtype=torch.bool), torch.from_numpy(see[:new, :new])], 1).cuda()
    for h in range(H):
        kk, vv = k[h // G, :cached + new], v[h // G, :cached + new]
        # what no token of a row sees is no part of its sum
        o[:new, h], _, tol[:new, h], _ = C.attend(q[:new, h], kk, vv, vis, dtype)
    return o.view(n, H * D), tol.view(n, H * D)


def run(ctx, dtype, n_tok, heads, kv_heads, dim, lens, new=None, chain=False, out16=False, seed=0, k_stride=None,
        max_len=None, see=None, ctas=0):
    import cache_cases as C
    import mako_attn
    import torch
    B = len(lens)
    top = max(max(lens), 0) if max_len is None else max_len
    S = k_stride or top + n_tok
    q = C.randn(seed, B, n_tok, heads, dim, dtype=dtype)
    k, v = (C.randn(seed + i, B, kv_heads, S, dim, dtype=dtype) for i in (1, 2))
    if see is None:
        see, mask = C.random_tree(seed, B, n_tok)
    else:
        mask = C.words(see)
    if chain:
        see, mask = np.tril(np.ones((B, n_tok, n_tok), bool)), None
    o = torch.full((B, n_tok, heads * dim), 77.0, dtype=C.DT[dtype] if out16 else torch.float32, device="cuda")
    ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, int(out16))
    ctx.set_option(mako_attn.OPT_GRID_CTAS, ctas)
    try:
        ctx.attention_tree(q, k, v, o, B, n_tok, None if new is None else C.i32(new), C.i32(lens), top, heads, kv_heads,
                           dim, S, mask)
    finally:
        ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, 0)
        ctx.set_option(mako_attn.OPT_GRID_CTAS, 0)
    torch.cuda.synchronize()
    assert ctx.device_error() == 0
    for b in range(B):
        nn = n_tok if new is None else min(max(new[b], 0), n_tok)
        want, tol = want_rows(q[b], k[b], v[b], min(max(lens[b], 0), top), nn, see[b], dtype)
        got = o[b].double()
        if out16:
            tol = tol * (1 + C.HALF_STEP[dtype]) + C.HALF_STEP[dtype] * want.abs() + 2.0 ** -25
        over = ((got - want).abs() - tol - 1e-30)[:nn]
        assert nn == 0 or over.max() <= 0, (b, float(over.max()), float((got - want)[:nn].abs().max()))
        assert (o[b, nn:] == 77.0).all()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n_tok,heads,kv_heads", [(1, 8, 8), (5, 8, 2), (16, 4, 1), (33, 6, 2), (64, 8, 2), (100, 7, 1)])
def test_shapes(ctx, dtype, dim, n_tok, heads, kv_heads):
    run(ctx, dtype, n_tok, heads, kv_heads, dim, [700, 0, 129], seed=n_tok + dim)


@pytest.mark.parametrize("cached", [0, 1, 62, 63, 64, 65, 127, 128, 129, 255, 256, 1000])
def test_lengths(ctx, cached):
    run(ctx, 1, 9, 4, 2, 128, [cached], seed=cached)
    run(ctx, 0, 37, 4, 1, 64, [cached], seed=cached)
    run(ctx, 0, 3, 16, 2, 256, [cached], seed=cached)


@pytest.mark.parametrize("n_tok", [1, 2, 31, 32, 33, 127, 128, 129, 255, 256])
def test_token_counts(ctx, n_tok):
    run(ctx, 1, n_tok, 2, 1, 128, [300, 5], chain=True, seed=n_tok)
    run(ctx, 0, n_tok, 2, 2, 64, [300, 5], seed=n_tok)


@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (5, 1), (12, 4), (40, 1), (129, 1), (24, 24)])
def test_head_groups(ctx, heads, kv_heads):
    run(ctx, 1, 6, heads, kv_heads, 64, [200, 77], seed=heads)
    run(ctx, 1, 6, heads, kv_heads, 256, [200, 77], seed=heads)


def test_ragged_batch(ctx):
    run(ctx, 0, 20, 8, 2, 128, [3000, 0, -7, 900, 64, 1], new=[20, 3, 1, 0, 35, -2], k_stride=3100)
    # a length above max_kv_len is read as max_kv_len
    run(ctx, 1, 4, 4, 2, 128, [500, 100], k_stride=600, max_len=300)


@pytest.mark.parametrize("dtype", [0, 1])
def test_long_and_16bit(ctx, dtype):
    run(ctx, dtype, 16, 8, 2, 128, [20000, 3, 9000], out16=True)
    run(ctx, dtype, 64, 8, 2, 128, [20001, 11], out16=True)
    run(ctx, dtype, 37, 16, 2, 256, [5001, 11], out16=True)


@pytest.mark.parametrize("ctas", [1, 2, 3, 7, 31])
@pytest.mark.parametrize("dtype,dim,n_tok,heads", [(0, 64, 9, 4), (1, 128, 9, 8), (1, 128, 70, 8), (0, 64, 70, 4), (1, 256, 21, 8)])
def test_few_ctas(ctx, ctas, dtype, dim, n_tok, heads):
    """Many pieces a CTA, whole and cut at either end, of one tile and of many."""
    run(ctx, dtype, n_tok, heads, 2, dim, [0, 1500, 3, 200, 0, 64, 127, 128, 700], new=[n_tok, 5, 1, 0, n_tok, 2, n_tok, 3, 1],
        k_stride=1600, ctas=ctas, seed=ctas)


def test_many_sequences(ctx):
    rs = np.random.default_rng(0)
    run(ctx, 1, 3, 4, 2, 64, [int(x) for x in rs.integers(0, 600, 200)], new=[int(x) for x in rs.integers(0, 4, 200)])


def test_rows_that_see_nothing(ctx):
    """Tokens whose mask words are 0 (over an empty cache: the row is 0; over a full one: the cached keys only), and
    mask bits past the drafted tokens."""
    see = np.zeros((2, 40, 40), bool)
    see[:, ::3, 5] = True
    run(ctx, 0, 40, 4, 2, 128, [0, 150], see=see)
    see = np.ones((2, 40, 40), bool)
    run(ctx, 1, 40, 4, 2, 128, [0, 150], see=see, new=[7, 33])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n_tok", [4, 48])
def test_unseen_values_have_no_effect(ctx, dtype, dim, n_tok):
    """NaN and infinities in cache rows past the draft, and in drafted keys and values that a token does not see, leave
    its row's bits as they are; a row that sees a NaN value is NaN there."""
    import cache_cases as C
    import torch
    B, H, KV, S = 2, 4, 2, 400
    lens, new = [190, 0], [n_tok, n_tok - 1]
    q = C.randn(1, B, n_tok, H, dim, dtype=dtype)
    k, v = C.randn(2, B, KV, S, dim, dtype=dtype), C.randn(3, B, KV, S, dim, dtype=dtype)
    see, mask = C.random_tree(4, B, n_tok)

    def call(k, v):
        o = torch.full((B, n_tok, H * dim), 5.0, device="cuda")
        ctx.attention_tree(q, k, v, o, B, n_tok, C.i32(new), C.i32(lens), 190, H, KV, dim, S, mask)
        return o

    base = call(k, v)
    k2, v2 = k.clone(), v.clone()
    for b in range(B):
        k2[b, :, lens[b] + new[b]:] = float("nan")
        v2[b, :, lens[b] + new[b]:] = float("inf")
    assert torch.equal(call(k2, v2), base)
    for b in range(B):
        j = 1
        v2[b, 1, lens[b] + j, 3] = float("nan")
        v2[b, 1, lens[b] + j, dim - 1] = float("-inf")
    got = call(k2, v2)
    for b in range(B):
        sees = torch.from_numpy(see[b, :new[b], 1]).cuda()
        g, w = got[b, :new[b]].view(-1, H, dim), base[b, :new[b]].view(-1, H, dim)
        assert torch.equal(g[:, :H // KV], w[:, :H // KV])
        assert torch.equal(g[~sees], w[~sees])
        hit = g[sees][:, H // KV:]
        assert torch.isnan(hit[..., 3]).all() and (hit[..., dim - 1] == float("-inf")).all()
        rest = [d for d in range(dim) if d not in (3, dim - 1)]
        assert torch.equal(hit[..., rest], w[sees][:, H // KV:][..., rest])
    # a key of NaN: rows that see it are NaN, others as before
    k2, v2 = k.clone(), v.clone()
    for b in range(B):
        k2[b, 0, lens[b] + 1] = float("nan")
    got = call(k2, v2)
    for b in range(B):
        sees = torch.from_numpy(see[b, :new[b], 1]).cuda()
        g, w = got[b, :new[b]].view(-1, H, dim), base[b, :new[b]].view(-1, H, dim)
        assert torch.equal(g[~sees], w[~sees]) and torch.equal(g[:, H // KV:], w[:, H // KV:])
        assert torch.isnan(g[sees][:, :H // KV]).all()


@pytest.mark.parametrize("dim,n_tok", [(64, 5), (128, 5), (64, 70), (128, 70), (256, 5)])
def test_value_ranges(ctx, dim, n_tok):
    """bf16 values far outside fp16's range and at its ends, alike in all keys and by groups of 16 keys, and zero."""
    import cache_cases as C
    import torch
    H, KV, L = 4, 2, 500
    q, k = C.randn(1, 1, n_tok, H, dim, dtype=1), C.randn(2, 1, KV, L + n_tok, dim, dtype=1)
    v0 = C.randn(3, 1, KV, L + n_tok, dim, dtype=1)
    see, mask = C.random_tree(4, 1, n_tok)
    groups = torch.arange(L + n_tok, device="cuda")[:, None] // 16 % 4
    mixed = torch.tensor([2.0 ** -40, 1.0, 2.0 ** 30, 2.0 ** -9], device="cuda")[groups]
    for scale in (2.0 ** -60, 2.0 ** -11, 2.0 ** -9, 2.0 ** 13, 2.0 ** 14, 2.0 ** 60, 0.0, mixed):
        v = (v0.float() * scale).to(torch.bfloat16)
        o = torch.full((1, n_tok, H * dim), 3.0, device="cuda")
        ctx.attention_tree(q, k, v, o, 1, n_tok, None, C.i32([L]), L, H, KV, dim, L + n_tok, mask)
        want, tol = want_rows(q[0], k[0], v[0], L, n_tok, see[0], 1)
        if not torch.is_tensor(scale) and scale < 2.0 ** -11:
            tol = tol - C.V_STEP[1]  # such values never go through fp16
        assert ((o[0].double() - want).abs() <= tol).all(), scale


@pytest.mark.parametrize("dtype", [0, 1])
def test_seen_values_that_are_not_finite(ctx, dtype):
    """A cached key's NaN value, seen by all, makes its column NaN in every row and no other."""
    import cache_cases as C
    import torch
    n, H, KV, D, L = 5, 4, 2, 128, 300
    q, k, v = C.randn(1, 1, n, H, D, dtype=dtype), C.randn(2, 1, KV, L + n, D, dtype=dtype), C.randn(3, 1, KV, L + n, D, dtype=dtype)
    v[0, 1, 70, 9] = float("nan")
    o = torch.zeros(1, n, H * D, device="cuda")
    ctx.attention_tree(q, k, v, o, 1, n, None, C.i32([L]), L, H, KV, D, L + n)
    bad = torch.isnan(o.view(n, H, D))
    assert bad[:, 2:, 9].all() and bad.sum() == n * 2


@pytest.mark.parametrize("dtype", [0, 1])
def test_large_scores(ctx, dtype):
    """Scores in the thousands: one key takes almost all weight, the maximum moves from tile to tile."""
    import cache_cases as C
    import torch
    n, H, KV, D, L = 12, 4, 2, 128, 900
    q = C.randn(1, 1, n, H, D, dtype=dtype) * 20
    k, v = C.randn(2, 1, KV, L + n, D, dtype=dtype) * 10, C.randn(3, 1, KV, L + n, D, dtype=dtype)
    see, mask = C.random_tree(4, 1, n)
    o = torch.zeros(1, n, H * D, device="cuda")
    ctx.attention_tree(q, k, v, o, 1, n, None, C.i32([L]), L, H, KV, D, L + n, mask)
    want, tol = want_rows(q[0], k[0], v[0], L, n, see[0], dtype)
    assert ((o[0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,n_tok", [(0, 5), (0, 70), (1, 5), (1, 70)])
def test_many_small_weights(ctx, dtype, n_tok):
    """One key of weight 1 beside 32768 of 2^-25.1, all of one CTA, and values of 1: o is 1.  The small ones are 2^-10.1 of
    the sum together.  Each P is off by 2^-6 of itself at most; the product's fp32 sum, near 2^7 in steps of 2^-16, takes
    them 16 at a time, near 2^-14, and loses a step at most, a quarter: less than 2^-12 in all."""
    import cache_cases as C
    import mako_attn
    import torch
    D, L = 128, 32769
    q = torch.ones(1, n_tok, 1, D, dtype=C.DT[dtype], device="cuda")
    k = torch.zeros(1, 1, L + n_tok, D, dtype=C.DT[dtype], device="cuda")
    k[0, 0, 0] = 1.5390625
    v = torch.ones_like(k)
    o = torch.zeros(1, n_tok, D, device="cuda")
    ctx.set_option(mako_attn.OPT_GRID_CTAS, 1)
    try:
        ctx.attention_tree(q, k, v, o, 1, n_tok, None, C.i32([L]), L, 1, 1, D, L + n_tok)
    finally:
        ctx.set_option(mako_attn.OPT_GRID_CTAS, 0)
    assert ((o.double() - 1).abs() <= 2.0 ** -11).all()


def test_chain_of_one_is_decode(ctx):
    """One drafted token of each sequence gives what the single-token decode gives over the same keys, within both
    kernels' bounds."""
    import cache_cases as C
    import torch
    B, H, KV, D, S = 3, 8, 2, 128, 2000
    lens = [1500, 0, 77]
    q, k, v = C.randn(1, B, 1, H, D), C.randn(2, B, KV, S, D), C.randn(3, B, KV, S, D)
    a, d = torch.zeros(B, 1, H * D, device="cuda"), torch.zeros(B, H * D, device="cuda")
    ctx.attention_tree(q, k, v, a, B, 1, None, C.i32(lens), 1500, H, KV, D, S)
    ctx.attention_decode(q, k, v, d, C.i32([x + 1 for x in lens]), 1501, H, KV, D, S)
    for b in range(B):
        _, tol = want_rows(q[b], k[b], v[b], lens[b], 1, np.ones((1, 1), bool), 0)
        assert ((a[b] - d[b]).abs().double() <= 2 * tol).all()


def test_far_rows(ctx):
    """A cache whose rows lie past 2^32 bytes and 2^31 values."""
    import cache_cases as C
    import torch
    B, KV, S, D, n, H = 3, 8, 400000, 256, 2, 8  # 2.5e9 values
    k = torch.zeros(B, KV, S, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    lens = [300, 5, 399990]
    small = C.randn(2, KV, 304, D)
    k[0, :, :304], v[0, :, :304] = small, small.flip(1)
    # the last sequence: keys of zero but for the drafted rows, whose scores decide
    k[2, :, 399990:399992] = 40.0
    v[2, :, 399990:399992] = C.randn(3, KV, 2, D)
    q = C.randn(1, B, n, H, D)
    q[2] = 1.0
    o = torch.zeros(B, n, H * D, device="cuda")
    ctx.attention_tree(q, k, v, o, B, n, None, C.i32(lens), 399990, H, KV, D, S)
    want, tol = want_rows(q[0], k[0], v[0], 300, n, np.tril(np.ones((n, n), bool)), 0)
    assert ((o[0].double() - want).abs() <= tol).all()
    # e^(640 - 0) against 399990: the drafted values alone remain
    last = v[2, :, 399990:399992].double()
    assert ((o[2, 0].double() - last[:, 0].reshape(-1)).abs() <= 2.0 ** -11 * last[:, 0].reshape(-1).abs() + 1e-6).all()
    mean = last.mean(1).reshape(-1)
    assert ((o[2, 1].double() - mean).abs() <= 2.0 ** -10 * last.abs().mean(1).reshape(-1) + 1e-6).all()
    del k, v
    torch.cuda.empty_cache()


def test_refusals(ctx):
    import mako_attn
    import torch
    h = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    o = torch.zeros(1 << 14, device="cuda")
    ok = dict(q=h, k=h, v=h, o=o, batch=1, n_tok=2, n_new=None, kv_len=n, max_kv_len=6, heads=2, kv_heads=1, dim=128,
              k_stride=8, mask=None)
    ctx.attention_tree(**ok)
    for bad, text in [(dict(dim=80), "heads of 80"), (dict(heads=3, kv_heads=2), "3 heads over 2"),
                      (dict(n_tok=257, k_stride=1000), "257 drafted"), (dict(max_kv_len=7), "max_kv_len 7"),
                      (dict(max_kv_len=0xFFFFFFFF), "max_kv_len"), (dict(batch=65536), "65536 sequences"),
                      (dict(v=None), "null"), (dict(kv_len=None), "null"), (dict(o=o[1:]), "unaligned"),
                      (dict(k=h[1:]), "unaligned")]:
        with pytest.raises(mako_attn.MakoError, match=text):
            ctx.attention_tree(**{**ok, **bad})
    ctx.attention_tree(**{**ok, "batch": 0})
    ctx.attention_tree(**{**ok, "n_tok": 0})
