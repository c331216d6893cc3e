"""The cache operators together, as a server uses them: prompts appended, decode steps that accumulate weights, an
eviction into a smaller cache and later in place, drafted trees appended at their true positions and attended, the
accepted ones appended again; then the same calls captured in CUDA graphs, on another stream, and with the projection
behind the attention.  Every attention's output is compared with softmax in 64 bits over the cache as it then stands."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, H, KV, D, DT = 2, 8, 2, 128, 1
LD = (H + 2 * KV) * D
EPS = 1e-6


def freqs():
    import mako_attn as M
    import torch
    return torch.from_numpy(M.rope_freqs(D, 10000.0, M.ROPE_PARTS, 4.0, 2048.0, 1.0, 32.0)).cuda()


class Server:
    """One layer's cache and the calls on it."""

    def __init__(self, ctx, rows, seed=0):
        import torch
        self.ctx, self.rows = ctx, rows
        g = torch.Generator().manual_seed(seed)
        self.randn = lambda *s: torch.randn(*s, generator=g).cuda()
        self.k, self.v = (torch.full((B, KV, rows, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.weight = torch.zeros(B, KV, rows, device="cuda")
        self.kv_len = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.freq, self.w = freqs(), 1.0 + 0.1 * self.randn(D)

    def append(self, x, n, pos=None, n_new=None, stream=None):
        import torch
        q = torch.zeros(B, n, H, D, dtype=torch.bfloat16, device="cuda")
        self.ctx.cache_append(x, LD, 0, D, H * D, (H + KV) * D, B, n, n_new, self.kv_len, pos, H, KV, D, D, 1, self.freq,
                              1.1, self.w, self.w, EPS, q, self.k, self.v, self.rows, stream=stream)
        return q

    def expect(self, q, b, h, keys, see):
        """o and its bound of head h's rows q [n][H][D] over the cache's first `keys` rows."""
        import cache_cases as C
        kv = h // (H // KV)
        return C.attend(q[b, :, h], self.k[b, kv, :keys], self.v[b, kv, :keys], see, DT)

    def check(self, o, q, keys, see):
        """o [B][n][H * D] against 64 bits; keys[b], see[b] [n][keys]."""
        for b in range(B):
            for h in range(H):
                want, p, tol, rel = self.expect(q, b, h, keys[b], see[b].cuda())
                got = o[b].view(-1, H, D)[:, h].double()
                assert ((got - want).abs() <= tol + 1e-30).all(), (b, h, float((got - want).abs().max()))


def test_serving_loop(ctx):
    import cache_cases as C
    import torch
    s = Server(ctx, 700)
    lens = [600, 250]
    prompt = s.randn(B * 600, LD)
    s.append(prompt, 600, n_new=C.i32(lens))
    s.kv_len = C.i32(lens)
    # decode steps: each token is appended, then attends itself and all before it
    total = [np.zeros((KV, 700)) for _ in range(B)]
    for step in range(3):
        q = s.append(s.randn(B, LD), 1)
        s.kv_len += 1
        lens = [n + 1 for n in lens]
        o = torch.zeros(B, H * D, device="cuda")
        s.ctx.attention_decode_weights(q[:, 0].contiguous(), s.k, s.v, o, s.weight, s.kv_len, max(lens), H, KV, D, s.rows)
        s.check(o.view(B, 1, H * D), q, lens, [torch.ones(1, n, dtype=torch.bool) for n in lens])
        for b in range(B):
            for h in range(H):
                p = s.expect(q, b, h, lens[b], torch.ones(1, lens[b], dtype=torch.bool, device="cuda"))[1]
                total[b][h // (H // KV), :lens[b]] += p[0].cpu().numpy()
    for b in range(B):  # the weights' sums, within 2^-12 of each (scores of a few units in fp32, three steps, four heads)
        got = s.weight[b].cpu().numpy()
        assert (np.abs(got - total[b]) <= 2.0 ** -12 * total[b] + 1e-12).all()
        assert abs(got.sum() - 3 * H) < 1e-3
    # eviction into a cache of 300 rows
    small = Server(ctx, 300, seed=1)
    kept = torch.zeros(B, KV, 200, dtype=torch.int32, device="cuda")
    new_len = torch.zeros(B, dtype=torch.int32, device="cuda")
    s.ctx.cache_evict(s.k, s.v, s.weight, s.kv_len, max(lens), KV, D, s.rows, 4, 50, 200, small.k, small.v, small.weight,
                      300, kept, new_len)
    assert new_len.tolist() == [200, 200]
    for b in range(B):
        for h in range(KV):
            at = kept[b, h].long()
            assert (at[1:] > at[:-1]).all() and at[:4].tolist() == [0, 1, 2, 3]
            assert at[-50:].tolist() == list(range(lens[b] - 50, lens[b]))
            assert torch.equal(small.k[b, h, :200], s.k[b, h, at]) and torch.equal(small.v[b, h, :200], s.v[b, h, at])
            assert torch.equal(small.weight[b, h, :200], s.weight[b, h, at])
            rest = s.weight[b, h, 4:lens[b] - 50].cpu().numpy()
            assert set(at[4:-50].tolist()) == set((4 + np.lexsort((np.arange(rest.size), -rest))[:146]).tolist())
    small.kv_len = new_len
    # a drafted tree: positions go on from the true lengths, rows from the evicted cache's
    n = 12
    see, mask = C.random_tree(7, B, n)
    depth = see.sum(-1) - 1
    pos = C.i32(np.asarray(lens)[:, None] + depth)
    x = s.randn(B * n, LD)
    q = small.append(x, n, pos)
    o = torch.zeros(B, n, H * D, device="cuda")
    small.ctx.attention_tree(q, small.k, small.v, o, B, n, None, small.kv_len, 200, H, KV, D, 300, mask)
    vis = [torch.cat([torch.ones(n, 200, dtype=torch.bool), torch.from_numpy(see[b])], 1) for b in range(B)]
    small.check(o, q, [200 + n] * B, vis)
    # the path of the deepest token is accepted: its tokens appended again give the rows they had as drafts
    for b in range(B):
        path = np.flatnonzero(see[b, int(depth[b].argmax())])
        drafted = small.k[b, :, 200 + path].clone()
        again = torch.zeros(B * n, LD, device="cuda")
        again[b * n:b * n + len(path)] = x[b * n + torch.from_numpy(path).cuda()]
        new = [0, 0]
        new[b] = len(path)
        place = np.zeros((B, n))
        place[b, :len(path)] = lens[b] + np.arange(len(path))
        small.append(again, n, C.i32(place), C.i32(new))
        assert torch.equal(small.k[b, :, 200:200 + len(path)], drafted)
    # and in place, back to 150 rows
    before = small.k.clone()
    kept = torch.zeros(B, KV, 150, dtype=torch.int32, device="cuda")
    small.ctx.cache_evict(small.k, small.v, small.weight, small.kv_len, 200, KV, D, 300, 4, 50, 150, small.k, small.v,
                          small.weight, 300, kept, small.kv_len)
    assert small.kv_len.tolist() == [150, 150]
    for b in range(B):
        for h in range(KV):
            assert torch.equal(small.k[b, h, :150], before[b, h, kept[b, h].long()])
    assert ctx.device_error() == 0


def test_graph_outlives_larger_calls():
    """A captured step replays right after later, larger calls have grown the context's scratch, and beside a second
    graph of the same context."""
    import cache_cases as C
    import mako_attn
    import torch
    ctx = mako_attn.Context(0)

    def make(n, length, seed):
        S = length + n
        t = dict(q=C.randn(seed, 1, n, H, D, dtype=DT), k=C.randn(seed + 1, 1, KV, S, D, dtype=DT),
                 v=C.randn(seed + 2, 1, KV, S, D, dtype=DT), o=torch.zeros(1, n, H * D, device="cuda"),
                 od=torch.zeros(1, H * D, device="cuda"), w=torch.zeros(1, KV, S, device="cuda"),
                 len=C.i32([length]), kept=torch.zeros(1, KV, 64, dtype=torch.int32, device="cuda"),
                 ko=torch.zeros(1, KV, 64, D, dtype=C.DT[DT], device="cuda"),
                 vo=torch.zeros(1, KV, 64, D, dtype=C.DT[DT], device="cuda"), wo=torch.zeros(1, KV, 64, device="cuda"),
                 new=C.i32([0]))

        def calls():
            ctx.attention_tree(t["q"], t["k"], t["v"], t["o"], 1, n, None, t["len"], length, H, KV, D, S)
            ctx.attention_decode_weights(t["q"][:, 0], t["k"], t["v"], t["od"], t["w"], t["len"], length, H, KV, D, S)
            ctx.cache_evict(t["k"], t["v"], t["w"], t["len"], length, KV, D, S, 2, 8, 64, t["ko"], t["vo"], t["wo"], 64,
                            t["kept"], t["new"])
        return t, calls

    def outputs(t):
        return [t[x].clone() for x in ("o", "od", "w", "kept", "ko", "vo", "wo", "new")]

    t1, calls1 = make(4, 500, 1)
    t2, calls2 = make(40, 9000, 11)
    calls1()
    torch.cuda.synchronize()
    g1 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        calls1()
    calls2()  # more rows, more keys: the scratch grows
    torch.cuda.synchronize()
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        calls2()
    for t, g, calls in ((t1, g1, calls1), (t2, g2, calls2), (t1, g1, calls1)):
        for x in ("q", "k", "v"):
            t[x].copy_(C.randn(99, *t[x].shape, dtype=DT))
        t["w"].zero_()
        g.replay()
        torch.cuda.synchronize()
        got = outputs(t)
        t["w"].zero_()
        for x in ("o", "od", "ko", "vo", "wo", "kept"):
            t[x].zero_()
        calls()
        torch.cuda.synchronize()
        for a, b in zip(got, outputs(t)):
            assert torch.equal(a, b)
    assert ctx.device_error() == 0
    del g1, g2
    ctx.close()


def test_other_stream_and_projection(ctx):
    """The calls on a stream of their own, ordered by events, with 16-bit output feeding the output projection."""
    import cache_cases as C
    import mako_attn
    import torch
    s = Server(ctx, 400, seed=5)
    side = torch.cuda.Stream()
    n, length = 8, 300
    x0, x1 = s.randn(B * length, LD), s.randn(B * n, LD)
    w = C.randn(3, 256, H * D, dtype=DT)
    y = torch.zeros(B * n, 256, device="cuda")
    o = torch.zeros(B, n, H * D, dtype=torch.bfloat16, device="cuda")
    lens = C.i32([length] * B)
    side.wait_stream(torch.cuda.current_stream())
    ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, 1)
    try:
        with torch.cuda.stream(side):
            s.append(x0, length)
            s.kv_len = lens
            q = s.append(x1, n)
            ctx.attention_tree(q, s.k, s.v, o, B, n, None, lens, length, H, KV, D, 400)
            ctx.proj(w, o, y, B * n, H * D, 256)
    finally:
        ctx.set_option(mako_attn.OPT_OUTPUT_16BIT, 0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    see = torch.cat([torch.ones(n, length, dtype=torch.bool), torch.ones(n, n, dtype=torch.bool).tril()], 1)
    for b in range(B):
        for h in range(H):
            want, _, tol, _ = s.expect(q, b, h, length + n, see.cuda())
            got = o[b].view(n, H, D)[:, h].double()
            assert ((got - want).abs() <= tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all()
    want = o.view(B * n, -1).double() @ w.double().T
    # fp32 sums of 1024 exact products: 1024 roundings of 2^-24 at most
    assert ((y.double() - want).abs() <= 2.0 ** -14 * (o.view(B * n, -1).double().abs() @ w.double().abs().T)).all()
    assert ctx.device_error() == 0


def test_launch_counts(ctx):
    import torch
    s = Server(ctx, 100, seed=6)
    before = ctx.launches()
    s.append(s.randn(B, LD), 1)
    assert ctx.launches() == before + 1
    torch.cuda.synchronize()
