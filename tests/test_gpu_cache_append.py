"""mako_cache_append against its formulas in 64 bits.

Bar: the kernel computes in fp32 and rounds once.  A value v of a pair (a, b) is off by at most half a step of the
16-bit type at v, plus the fp32 error: the norm's sum of squares of up to 256 values, its root and two products, the angle (a reduced
turn rounded to fp32: 2 pi 2^-25; sincospi a few units in the last place) and the rotation's three roundings together
stay under 2^-18 of hypot(a, b) * amplitude (a sum of 64 roundings of 2^-24 at most).  Rows outside the written range
keep their bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}  # of fp16, bf16, relative
TINY = {0: 2.0 ** -25, 1: 0.0}             # half of fp16's smallest step
FILL = 0x7BFF


def tdev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def filled(shape, dtype):
    import torch
    t = torch.full(shape, FILL, dtype=torch.int16, device="cuda")
    return t.view(torch.bfloat16 if dtype == 1 else torch.float16)


def values(t):
    return t.float().cpu().numpy().astype(np.float64)


def bits(t):
    import torch
    return t.view(torch.int16).cpu().numpy().view(np.uint16)


def formula(u, w, eps, angle, amplitude, layout, rot):
    """One token's heads u [heads][dim] in 64 bits: (values, hypot of each value's pair)."""
    u = u.astype(np.float64)
    if w is not None:
        u = u / np.sqrt(np.mean(u * u, -1, keepdims=True) + eps) * w.astype(np.float64)
    out, size = u.copy(), np.abs(u)
    half = rot // 2
    i = np.arange(half)
    a, b = (i, i + half) if layout == 1 else (2 * i, 2 * i + 1)
    c, s = np.cos(angle) * amplitude, np.sin(angle) * amplitude
    out[:, a], out[:, b] = u[:, a] * c - u[:, b] * s, u[:, b] * c + u[:, a] * s
    size[:, a] = size[:, b] = np.hypot(u[:, a], u[:, b]) * amplitude
    return out, size


def check(ctx, dtype, batch, n_tok, heads, kv_heads, dim, rot, layout, k_stride, lens, n_new=None, pos=None, norm=True,
          gap=0, amplitude=1.0, seed=0):
    import torch
    rng = np.random.default_rng(seed)
    q_stride = dim + gap
    q_col0 = gap
    k_col0 = q_col0 + heads * q_stride
    v_col0 = k_col0 + kv_heads * dim + gap
    ld = v_col0 + kv_heads * dim + gap
    x = (rng.standard_normal((batch * n_tok, ld)) * 3).astype(np.float32)
    freq = 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    wq, wk = (rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2)) if norm else (None, None)
    eps = 1e-6
    q = filled((batch, n_tok, heads, dim), dtype)
    k, v = filled((batch, kv_heads, k_stride, dim), dtype), filled((batch, kv_heads, k_stride, dim), dtype)
    lens = np.asarray(lens, np.int32)
    dn = None if n_new is None else tdev(np.asarray(n_new, np.int32))
    dp = None if pos is None else tdev(np.asarray(pos, np.int32))
    ctx.cache_append(tdev(x), ld, q_col0, q_stride, k_col0, v_col0, batch, n_tok, dn, tdev(lens), dp, heads, kv_heads,
                     dim, rot, layout, tdev(freq) if rot else None, amplitude, None if wq is None else tdev(wq),
                     None if wk is None else tdev(wk), eps, q, k, v, k_stride)
    torch.cuda.synchronize()
    wrote_q = np.zeros((batch, n_tok, heads, dim), bool)
    wrote = np.zeros((batch, kv_heads, k_stride, dim), bool)
    gq, gk, gv = values(q), values(k), values(v)

    def near(got, want, size, what):
        over = np.abs(got - want) - HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -10) - 2.0 ** -18 * size - TINY[dtype]
        assert over.max() <= 0, (what, float(over.max()))

    for b in range(batch):
        for i in range(n_tok):
            if n_new is not None and i >= n_new[b]:
                continue
            row = max(int(lens[b]), 0) + i
            at = row if pos is None else int(pos[b][i])
            angle = at * freq
            t = x[b * n_tok + i]
            uq = np.stack([t[q_col0 + h * q_stride:][:dim] for h in range(heads)])
            uk = t[k_col0:k_col0 + kv_heads * dim].reshape(kv_heads, dim)
            uv = t[v_col0:v_col0 + kv_heads * dim].reshape(kv_heads, dim).astype(np.float64)
            near(gq[b, i], *formula(uq, wq, eps, angle, amplitude, layout, rot), "q")
            wrote_q[b, i] = True
            if row < k_stride:
                near(gk[b, :, row], *formula(uk, wk, eps, angle, amplitude, layout, rot), "k")
                near(gv[b, :, row], uv, 0 * uv, "v")
                wrote[b, :, row] = True
    assert (bits(q)[~wrote_q] == FILL).all()
    assert (bits(k)[~wrote] == FILL).all() and (bits(v)[~wrote] == FILL).all()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("layout", [1, 2])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 30), (128, 128), (128, 0), (128, 32), (128, 126), (256, 256),
                                     (256, 64), (256, 192), (256, 2)])
def test_rotation(ctx, dtype, layout, dim, rot):
    check(ctx, dtype, 2, 3, 5, 1, dim, rot, layout, 40, [7, 0], amplitude=1.25, seed=dim + rot)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (9, 3), (32, 8), (130, 10)])
def test_head_counts(ctx, heads, kv_heads):
    check(ctx, 1, 1, 2, heads, kv_heads, 128, 128, 1, 16, [3])
    check(ctx, 0, 1, 1, heads, kv_heads, 256, 128, 1, 16, [3], norm=False)


@pytest.mark.parametrize("gap", [1, 2, 3, 4, 128])
def test_odd_columns_and_strides(ctx, gap):
    check(ctx, 1, 2, 2, 4, 2, 128, 64, 2, 16, [3, 5], gap=gap)
    check(ctx, 0, 2, 2, 4, 2, 64, 64, 1, 16, [3, 5], gap=gap)


def test_ragged_far_and_full(ctx):
    # a sequence without new tokens, one with more than n_tok, negative lengths, a cache that ends inside the draft
    check(ctx, 0, 5, 6, 4, 2, 128, 128, 1, 20, [17, -3, 20, 0, 30], n_new=[6, 2, 6, 0, 9])
    rng = np.random.default_rng(3)
    check(ctx, 0, 3, 4, 4, 2, 128, 128, 1, 64, [0, 10, 60], n_new=[4, 3, 4],
          pos=rng.integers(900000, 1100000, (3, 4)))
    check(ctx, 0, 1, 2, 2, 1, 64, 32, 2, 8, [1], pos=[[-5, 2 ** 31 - 1]])


def test_many_tokens(ctx):
    check(ctx, 1, 2, 300, 2, 1, 128, 128, 1, 310, [10, 4])


def test_infinities_stay_in_their_head(ctx):
    """A head whose projection holds NaN or an infinity leaves the others' bits as they are."""
    import torch
    H, KV, D = 4, 2, 128
    x = torch.randn(2, (H + 2 * KV) * D, device="cuda")
    freq = tdev(10000.0 ** (-2.0 * np.arange(D // 2) / D))
    w = torch.ones(D, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(x):
        q = torch.zeros(1, 2, H, D, dtype=torch.float16, device="cuda")
        k, v = (torch.zeros(1, KV, 4, D, dtype=torch.float16, device="cuda") for _ in range(2))
        ctx.cache_append(x, x.shape[1], 0, D, H * D, (H + KV) * D, 1, 2, None, lens, None, H, KV, D, D, 1, freq, 1.0, w, w,
                         1e-6, q, k, v, 4)
        return q, k, v

    a = call(x)
    y = x.clone()
    y[0, 5], y[0, D * H + 7] = float("inf"), float("nan")
    c = call(y)
    assert torch.equal(a[0][0, 0, 1:], c[0][0, 0, 1:]) and torch.equal(a[0][0, 1], c[0][0, 1])
    assert torch.equal(a[1][0, 1], c[1][0, 1]) and torch.equal(a[1][0, 0, 1], c[1][0, 0, 1])
    assert torch.equal(a[2], c[2])
    assert not torch.isfinite(c[0][0, 0, 0].float()).all() and torch.isnan(c[1][0, 0, 0].float()).all()


def test_refusals(ctx):
    import mako_attn
    import torch
    t = torch.zeros(4096, device="cuda")
    h = torch.zeros(4096, dtype=torch.float16, device="cuda")
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    f = torch.zeros(64, dtype=torch.float64, device="cuda")
    ok = dict(x=t, ld=512, q_col0=0, q_stride=128, k_col0=256, v_col0=384, batch=1, n_tok=1, n_new=None, kv_len=n,
              pos=None, heads=2, kv_heads=1, dim=128, rot=128, layout=1, freq=f, amplitude=1.0, wq=None, wk=None,
              eps=0.0, q=h, k=h[1024:], v=h[2048:], k_stride=8)
    ctx.cache_append(**ok)
    for bad, text in [(dict(dim=96), "heads of 96"), (dict(heads=3, kv_heads=2), "3 heads over 2"),
                      (dict(kv_heads=0), "over 0 kv heads"), (dict(rot=129), "129 rotated"),
                      (dict(rot=130), "130 rotated"), (dict(layout=0), "layout 0"), (dict(freq=None), "freq"),
                      (dict(amplitude=float("nan")), "amplitude"), (dict(wq=t), "eps 0"),
                      (dict(wk=t, eps=float("inf")), "eps"), (dict(q_stride=127), "stride 127"),
                      (dict(v_col0=385), "v at 385"), (dict(k_col0=0xFFFFFFFF), "k at"), (dict(ld=511), "511 floats"),
                      (dict(x=None), "null"), (dict(kv_len=None), "null"), (dict(q=h[1:]), "unaligned"),
                      (dict(batch=65536, n_tok=65536), "65536 sequences")]:
        with pytest.raises(mako_attn.MakoError, match=text):
            ctx.cache_append(**{**ok, **bad})
    ctx.cache_append(**{**ok, "batch": 0})
    ctx.cache_append(**{**ok, "n_tok": 0})
