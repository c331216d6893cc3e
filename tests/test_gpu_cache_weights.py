"""Accumulated attention weights over the life of a bounded cache: appended tokens begin at 0 whatever their row held,
evictions keep the sums of the rows they keep."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

H, KV, D = 8, 2, 64
LD = (H + 2 * KV) * D


def append(ctx, x, q, k, v, lens, rows, weight=None, n_new=None):
    """Tokens without norm or rotation."""
    ctx.cache_append(x, LD, 0, D, H * D, (H + KV) * D, q.shape[0], q.shape[1], n_new, lens, None, H, KV, D, 0, 1, None, 1.0,
                     None, None, 1.0, q, k, v, rows, weight=weight)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (10, 10, 128), (9, 9, 256), (1, 1, 64)])
def test_written_rows_are_cleared(ctx, heads, kv_heads, dim):
    """The entries of the rows written and no others; a row past the cache and a sequence without new tokens clear
    nothing; without the argument nothing is touched."""
    import cache_cases as C
    import torch
    B, n, S = 4, 6, 20
    lens, new = [3, 17, -2, 9], [6, 6, 2, 0]
    ld = (heads + 2 * kv_heads) * dim
    x = torch.randn(B * n, ld, device="cuda")
    q = torch.zeros(B, n, heads, dim, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(B, kv_heads, S, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for weight in (torch.full((B, kv_heads, S), 7.0, device="cuda"), None):
        q.zero_(), k.zero_(), v.zero_()
        ctx.cache_append(x, ld, 0, dim, heads * dim, (heads + kv_heads) * dim, B, n, C.i32(new), C.i32(lens), None, heads,
                         kv_heads, dim, 0, 1, None, 1.0, None, None, 1.0, q, k, v, S, weight=weight)
        torch.cuda.synchronize()
        for b in range(B):
            first = max(lens[b], 0)
            wrote = np.zeros(S, bool)
            wrote[first:first + new[b]] = True
            assert torch.equal((k[b] != 0).any(-1).any(0).cpu(), torch.from_numpy(wrote))
            if weight is not None:
                want = torch.where(torch.from_numpy(wrote), 0.0, 7.0).expand(kv_heads, S)
                assert torch.equal(weight[b].cpu(), want)


def pick(weight, length, sinks, recent, budget):
    if length <= budget:
        return np.arange(length)
    middle = np.arange(sinks, length - recent)
    order = np.lexsort((middle, -weight[middle]))
    return np.sort(np.concatenate([np.arange(sinks), middle[order[:budget - sinks - recent]],
                                   np.arange(length - recent, length)]))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("captured", [True, False])
def test_bounded_cache(ctx, in_place, captured):
    """Append, decode with weights, evict when full, again and again: every sum is that of the tokens that still are in the
    cache, as a host's bookkeeping by token has them, and each eviction keeps the rows that these sums name.  In place,
    or between two caches in turn; the decode step eager or replayed from a graph."""
    import cache_cases as C
    import torch
    rows, budget, sinks, recent, top = 96, 40, 2, 8, 64
    g = torch.Generator().manual_seed(5)

    def cache():
        return [torch.full((1, KV, rows, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)] + [
            torch.zeros(1, KV, rows, device="cuda")]

    caches = [cache(), cache()]
    kv_len = C.i32([0])
    x = torch.zeros(1, LD, device="cuda")
    q = torch.zeros(1, 1, H, D, dtype=torch.float16, device="cuda")
    o = torch.zeros(1, H * D, device="cuda")
    kept = torch.zeros(1, KV, budget, dtype=torch.int32, device="cuda")

    def step(k, v, w):
        append(ctx, x, q, k, v, kv_len, rows, weight=w)
        kv_len.add_(1)
        ctx.attention_decode_weights(q[:, 0], k, v, o, w, kv_len, rows, H, KV, D, rows)

    graphs = []
    for c in caches if captured else []:
        step(*c)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(*c)
    for c in caches:
        c[2].zero_()
    kv_len.zero_()
    at, length, sums, evicted = 0, 0, [np.zeros(0), np.zeros(0)], 0
    for _ in range(200):
        k, v, w = caches[at]
        x.copy_(torch.randn(1, LD, generator=g) * 2)
        if captured:
            graphs[at].replay()
        else:
            step(k, v, w)
        length += 1
        for h in range(KV):
            see = torch.ones(H // KV, length, dtype=torch.bool, device="cuda")
            _, p, _, _ = C.attend(q[0, 0, h * 4:h * 4 + 4], k[0, h, :length], v[0, h, :length], see, 0)
            sums[h] = np.append(sums[h], 0.0) + p.sum(0).cpu().numpy()
            # fp32 scores of a few units: 2^-15 of each weight and step is ample for 200 steps, 2^-24 a step for the adds
            got = w[0, h, :length].double().cpu().numpy()
            assert (np.abs(got - sums[h]) <= 2.0 ** -13 * sums[h] + 1e-12).all()
        if length == top:
            before = w.clone()
            out = caches[at if in_place else 1 - at]
            ctx.cache_evict(k, v, w, kv_len, rows, KV, D, rows, sinks, recent, budget, *out, rows, kept, kv_len)
            torch.cuda.synchronize()
            for h in range(KV):
                take = pick(before[0, h].cpu().numpy().astype(np.float64), length, sinks, recent, budget)
                np.testing.assert_array_equal(kept[0, h].cpu().numpy(), take)
                sums[h] = sums[h][take]
            length, evicted = budget, evicted + 1
            at = at if in_place else 1 - at
    assert evicted == 6 and ctx.device_error() == 0
    graphs.clear()
