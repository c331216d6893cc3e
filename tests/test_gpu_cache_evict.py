"""mako_attention_decode_weights against softmax in 64 bits, and mako_cache_evict, bit for bit, against a selection by
sorting."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def check_weights(ctx, dtype, heads, kv_heads, dim, lens, k_stride=None, out16=False, max_len=None, seed=0, scale=1.0, ctas=0):
    import cache_cases as C
    import mako_attn
    import torch
    B, G = len(lens), heads // kv_heads
    top = max(max(lens), 0) if max_len is None else max_len
    S = k_stride or max(top, 1)
    q = C.randn(seed, B, heads, dim, dtype=dtype) * scale
    k, v = (C.randn(seed + i, B, kv_heads, S, dim, dtype=dtype) for i in (1, 2))
    w = torch.rand(B, kv_heads, S, generator=torch.Generator().manual_seed(seed)).cuda()
    before = w.clone()
    for b in range(B):  # rows no call may read
        k[b, :, min(max(lens[b], 0), top):] = float("nan")
        v[b, :, min(max(lens[b], 0), top):] = float("nan")
    o = torch.full((B, heads * dim), 9.0, dtype=C.DT[dtype] if out16 else torch.float32, device="cuda")
    ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, int(out16))
    ctx.set_option(mako_attn.OPT_GRID_CTAS, ctas)
    try:
        ctx.attention_decode_weights(q, k, v, o, w, C.i32(lens), top, heads, kv_heads, dim, S)
        again, w2 = o.clone(), before.clone()
        ctx.attention_decode_weights(q, k, v, again, w2, C.i32(lens), top, heads, kv_heads, dim, S)
    finally:
        ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, 0)
        ctx.set_option(mako_attn.OPT_GRID_CTAS, 0)
    torch.cuda.synchronize()
    assert torch.equal(o, again) and torch.equal(w, w2)
    assert ctx.device_error() == 0
    for b in range(B):
        L = min(max(lens[b], 0), top)
        assert torch.equal(w[b, :, L:], before[b, :, L:])
        for h in range(kv_heads):
            see = torch.ones(G, L, dtype=torch.bool, device="cuda")
            want, p, tol, rel = C.attend(q[b, h * G:(h + 1) * G], k[b, h, :L], v[b, h, :L], see, dtype)
            got = o[b].view(heads, dim)[h * G:(h + 1) * G].double()
            if out16:
                tol = tol * (1 + C.HALF_STEP[dtype]) + C.HALF_STEP[dtype] * want.abs() + 2.0 ** -25
            assert ((got - want).abs() <= tol).all()
            # each head's weight within rel, one rounding for every add
            total = before[b, h, :L].double() + p.sum(0)
            bound = (rel * p).sum(0) + (G + 1) * 2.0 ** -24 * total
            assert L == 0 or ((w[b, h, :L].double() - total).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (7, 1), (40, 2)])
def test_weights(ctx, dtype, dim, heads, kv_heads):
    check_weights(ctx, dtype, heads, kv_heads, dim, [700, 0, 129, -4, 1], seed=heads + dim)


@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 255, 256, 257, 1023, 1025, 5000])
def test_weights_lengths(ctx, length):
    check_weights(ctx, 1, 8, 2, 128, [length], k_stride=length + 3, seed=length)
    check_weights(ctx, 0, 3, 1, 64, [length, 1], seed=length, out16=True)


def test_weights_long(ctx):
    check_weights(ctx, 0, 8, 2, 128, [40000, 17], seed=1)
    check_weights(ctx, 1, 16, 2, 256, [30000], k_stride=30001, seed=2, out16=True)
    check_weights(ctx, 1, 80, 1, 64, [3000], seed=3)
    check_weights(ctx, 0, 4, 2, 128, [500, 100], k_stride=600, max_len=300)
    check_weights(ctx, 1, 8, 2, 128, [4000], seed=4, scale=30.0)


@pytest.mark.parametrize("ctas", [1, 2, 5, 40])
@pytest.mark.parametrize("dtype,dim", [(0, 64), (1, 128), (0, 256)])
def test_weights_few_ctas(ctx, ctas, dtype, dim):
    check_weights(ctx, dtype, 8, 2, dim, [0, 1500, 3, 128, 0, 64, 127, 129, 700, 0], k_stride=1601, ctas=ctas, seed=ctas)


def test_weights_many_heads(ctx):
    check_weights(ctx, 0, 130, 1, 64, [700, 0, 300], seed=5)
    check_weights(ctx, 1, 260, 2, 128, [300, 129], seed=6)


def test_weights_refusals(ctx):
    import mako_attn
    import torch
    h = torch.zeros(1 << 12, dtype=torch.float16, device="cuda")
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    o = torch.zeros(1 << 12, device="cuda")
    ok = dict(q=h, k=h, v=h, o=o, weight=o[1024:], kv_len=n[:1], max_kv_len=8, heads=2, kv_heads=1, dim=128, k_stride=8)
    ctx.attention_decode_weights(**ok)
    for bad, text in [(dict(dim=80), "heads of 80"), (dict(heads=3, kv_heads=2), "3 heads over 2"),
                      (dict(max_kv_len=9), "max_kv_len 9"), (dict(weight=None), "null"), (dict(v=h[3:]), "unaligned")]:
        with pytest.raises(mako_attn.MakoError, match=text):
            ctx.attention_decode_weights(**{**ok, **bad})
    ctx.attention_decode_weights(**{**ok, "kv_len": n[:0]})


def pick(weight, length, sinks, recent, budget):
    """The rows kept of one head, ascending."""
    if length <= budget:
        return np.arange(length)
    lo, hi = sinks, length - recent
    w = weight[lo:hi].astype(np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    nan = np.isnan(weight[lo:hi])
    order = np.lexsort((np.arange(lo, hi), nan, -w))  # NaN after -inf
    return np.sort(np.concatenate([np.arange(lo), lo + order[:budget - sinks - recent], np.arange(hi, length)]))


def check_evict(ctx, dtype, kv_heads, dim, lens, sinks, recent, budget, k_stride, out_stride, weight=None, in_place=False,
                max_len=None, seed=0, alias_len=False):
    import cache_cases as C
    import torch
    B = len(lens)
    top = max(max(lens), 0) if max_len is None else max_len
    k, v = (C.randn(seed + i, B, kv_heads, k_stride, dim, dtype=dtype) for i in (1, 2))
    rs = np.random.default_rng(seed)
    if weight is None:
        weight = np.round(np.exp(2 * rs.standard_normal((B, kv_heads, k_stride))) * 64) / 64
    weight = np.ascontiguousarray(np.broadcast_to(weight, (B, kv_heads, k_stride)).astype(np.float32))
    w = torch.from_numpy(weight).cuda()
    k0, v0 = k.clone(), v.clone()
    if in_place:
        ko, vo, wo = k, v, w
    else:
        ko, vo = (torch.full((B, kv_heads, out_stride, dim), 3.0, dtype=C.DT[dtype], device="cuda") for _ in range(2))
        wo = torch.full((B, kv_heads, out_stride), 3.0, device="cuda")
    ko0, vo0, wo0 = ko.clone(), vo.clone(), wo.clone()
    kept = torch.full((B, kv_heads, budget), 12345, dtype=torch.int32, device="cuda")
    kv_len = C.i32(lens)
    new_len = kv_len if alias_len else torch.full((B,), 77, dtype=torch.int32, device="cuda")
    ctx.cache_evict(k, v, w, kv_len, top, kv_heads, dim, k_stride, sinks, recent, budget, ko, vo, wo, out_stride, kept,
                    new_len)
    torch.cuda.synchronize()
    got = kept.cpu().numpy()
    for b in range(B):
        L = min(max(lens[b], 0), top)
        assert int(new_len[b]) == min(L, budget)
        for h in range(kv_heads):
            rows = pick(weight[b, h], L, sinks, recent, budget)
            n = len(rows)
            np.testing.assert_array_equal(got[b, h, :n], rows)
            assert (got[b, h, n:] == -1).all()
            at = torch.from_numpy(rows).cuda()
            for out, src, was in ((ko, k0, ko0), (vo, v0, vo0), (wo, torch.from_numpy(weight).cuda(), wo0)):
                a, c = out[b, h].contiguous().view(torch.uint8), src[b, h][at].contiguous().view(torch.uint8)
                step = a.numel() // out.shape[2]
                assert torch.equal(a.view(-1)[:n * step], c.view(-1))
                assert torch.equal(a.view(-1)[n * step:], was[b, h].contiguous().view(torch.uint8).view(-1)[n * step:])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,kv_heads,dim", [(0, 1, 64), (1, 3, 128), (0, 2, 256)])
@pytest.mark.parametrize("lens,sinks,recent,budget", [
    ([900, 300, 299, 0, -5, 301], 4, 50, 300), ([5000], 0, 0, 1), ([2049, 2048], 0, 2000, 2000),
    ([3000, 1025], 1000, 0, 1000), ([4097, 700], 3, 500, 4096), ([70], 0, 0, 65), ([20000, 1], 8, 100, 777)])
def test_evict(ctx, in_place, dtype, kv_heads, dim, lens, sinks, recent, budget):
    S = max(max(lens), budget) + 5
    check_evict(ctx, dtype, kv_heads, dim, lens, sinks, recent, budget, S, S if in_place else budget + 3,
                in_place=in_place, seed=budget)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_weights_of_every_kind(ctx, in_place):
    """All equal, all zero of both signs, NaN, infinities, subnormals and negatives."""
    rs = np.random.default_rng(5)
    S = 1500
    kinds = [np.zeros(S), np.full(S, 0.25), np.where(rs.random(S) < 0.5, -0.0, 0.0), np.full(S, np.nan),
             np.where(rs.random(S) < 0.7, np.nan, rs.random(S)), np.where(rs.random(S) < 0.5, np.inf, -np.inf),
             rs.standard_normal(S), rs.random(S) * 1e-44, np.where(rs.random(S) < 0.9, -np.inf, np.nan)]
    for i, w in enumerate(kinds):
        check_evict(ctx, 1, 2, 128, [1500, 1400], 2, 30, 500, S, S if in_place else 500, weight=w, in_place=in_place,
                    seed=i)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_long_rows(ctx, in_place):
    """Rows of one CTA's registers and a few more, of a cluster's, and past them."""
    for n in (32768, 32769, 70001, 262144, 262145, 400000):
        check_evict(ctx, 0, 1, 64, [n, 31], 5, 300, 1234, n + 1, n + 1 if in_place else 1300, in_place=in_place, seed=n)
    check_evict(ctx, 1, 1, 64, [300000], 0, 0, 290000, 300000, 300000, weight=np.float32(0.5), in_place=in_place)


@pytest.mark.parametrize("n", [1500, 20000, 40001, 270001])
@pytest.mark.parametrize("low,high", [(1.0, 2.0), (float(np.nextafter(np.float32(2), np.float32(0))), 2.0), (0.0, 1.0),
                                      (float("nan"), 0.0), (1.0, float(np.nextafter(np.float32(1), np.float32(2)))),
                                      (-float("inf"), -1.0)])
def test_evict_counts_that_fit(ctx, n, low, high):
    """Two weights, alike but for a digit or the last bit, of which just as many have the higher one as stay, or one more
    or fewer; and no contest at all."""
    rs = np.random.default_rng(n)
    w = np.full(n, low)
    w[7 + rs.permutation(n - 37)[:400]] = high
    for budget in (437, 436, 438, 37):
        check_evict(ctx, 0, 1, 64, [n], 7, 30, budget, n, budget, weight=w)


def test_evict_capped_and_aliased_lengths(ctx):
    check_evict(ctx, 0, 2, 128, [900, 400, 1200], 4, 16, 256, 1300, 256, max_len=800)
    check_evict(ctx, 0, 4, 64, [900, 100, 1200], 4, 16, 256, 1300, 1300, in_place=True, alias_len=True)
    check_evict(ctx, 0, 4, 64, [900, 100, 1200], 4, 16, 256, 1300, 300, alias_len=True)


def test_evict_refusals(ctx):
    import mako_attn
    import torch
    k, v, ko, vo = (torch.zeros(4096, dtype=torch.float16, device="cuda") for _ in range(4))
    w, wo = torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = torch.zeros(64, dtype=torch.int32, device="cuda")
    ok = dict(k=k, v=v, weight=w, kv_len=n, max_kv_len=16, kv_heads=1, dim=64, k_stride=16, sinks=1, recent=2, budget=8,
              k_out=ko, v_out=vo, weight_out=wo, out_stride=8, kept=kept, new_len=n.clone())
    ctx.cache_evict(**ok)
    for bad, text in [(dict(dim=100), "heads of 100"), (dict(budget=0), "budget 0"), (dict(sinks=7), "7 sinks"),
                      (dict(sinks=0xFFFFFFFF), "sinks"), (dict(out_stride=7), "7 output rows"),
                      (dict(max_kv_len=17), "max_kv_len 17"), (dict(k_out=k), "partly"), (dict(weight_out=w), "partly"),
                      (dict(k_out=k, v_out=v, weight_out=w), "partly"), (dict(k_out=vo), "partly"),
                      (dict(k_out=v), "partly"), (dict(kept=None), "null"), (dict(new_len=None), "null"),
                      (dict(v_out=vo[4:]), "unaligned"), (dict(kv_heads=0), "0 kv heads")]:
        with pytest.raises(mako_attn.MakoError, match=text):
            ctx.cache_evict(**{**ok, **bad})
    ctx.cache_evict(**{**ok, "kv_len": n[:0]})
