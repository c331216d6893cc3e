// Attention for drafted tokens over a KV cache on sm_100a tensor cores (mako_attention_tree): per (sequence, kv head) the
// rows are (token, head of the group) pairs, up to thousands of keys long and few rows high.  No counterpart in the
// reference.
//
// Bound by the one read of K and V (4 * dim bytes a key and kv head, 128 rows cost 2/3 of that time in products): the
// tensor cores work on 128-row tiles however few rows there are, and everything else is arranged around streaming the
// cache.
//   - Work is cut by bytes: the tiles of all (sequence, kv head, row block) segments form one line that is divided
//     evenly over one CTA an SM, whatever the lengths; a CTA may start and end inside a segment.  Each CTA finds its place
//     on the device from kv_len (no host synchronisation).  A segment within one CTA is written at once, the pieces of a
//     cut one go to scratch (at most two a CTA) and tree_combine_kernel merges them by log-sum-exp.
//   - Warp 0 streams K and V tiles by TMA through one ring in the order of use; warp 1 issues the products; warps 2 and
//     3 load the rows of q (the first piece's, for which all wait, the softmax warps do), the latter cleans the drafted
//     values; warps 4-11 are two softmax warpgroups, a thread a row.
//   - Up to 128 rows: the two warpgroups take alternate key tiles of the same rows, each with its own S, maximum, sum and
//     O, and merge at the end (a split within the CTA).  More rows (WIDE): each takes 128 rows of every tile.  256-wide
//     heads: O alone takes half of TMEM, so one warpgroup runs with two S buffers of 64 keys.
//   - S is overwritten by P: fp16, or for bf16 the bf16 of p and of what that left over (two products, 2^-17 off instead of
//     2^-9: the sum of many rounded weights would show in fp32 outputs).  Base-2 softmax; a row's maximum moves only when
//     passed by 8.
//   - Turning bf16 V tiles into fp16 in shared memory, so that P is one part, pays only if columns that are small beside the
//     others may lose bits: with a test that fp16 holds every value exactly, 64-token trees over 8 x 16-32K keys take 248 us
//     against 249 without, and without the test 237.
//   - Keys at or past the cached length are seen by mask.  Scores that are not seen are replaced, not added to, so keys may
//     hold anything; values of those tiles are cleaned in shared memory before the product: rows behind the draft become
//     0, and so do single values that are not finite, which the rows that do see their token get back in the epilogue.
//     Infinities among the cached values, seen by all, are looked for there once a row has NaN.
//
// The same kernel serves the decode that accumulates attention weights (DEC, mako_attention_decode_weights): one token a
// sequence, its own key already counted in kv_len.  It stores the scores (4 bytes a key and head), and
// weights_finish_kernel, once each row's maximum and sum are known, turns them into the keys' weights.
//
// Every wait is bounded (clock64); on a timeout the thread records a code in p.err, waits (bounded) for its own copies and
// products in flight, and the CTA frees its TMEM and returns.
#include "common.cuh"
#include "kernels.h"
#include "tc100.cuh"

namespace mako {
namespace {

using namespace tc;

constexpr long long WAIT_LIMIT = 1ll << 31;  // clock cycles (~1 s)
// Pieces whose bad-value words are kept apart: the cleaner begins a piece once the products of the one before have all been
// issued, when the epilogue of the one three before it is over.
constexpr uint32_t BAD_RING = 4;

template <int D, bool WIDE, bool DEC>
struct TreeCfg {
    static constexpr bool DECODE = DEC;
    static constexpr int STREAMS = D == 256 ? 1 : 2;
    static constexpr int NT = 128 + 128 * STREAMS;
    static constexpr uint32_t TK = D == 256 ? 64 : 128;         // keys a tile
    static constexpr uint32_t ROWS = WIDE ? 256 : 128;          // rows a segment
    static constexpr uint32_t KBOX = TK * 128, QBOX = 128 * 128;  // 64 values of TK keys, of 128 rows
    static constexpr uint32_t SLOT = TK * D * 2;                // a K or V tile
    static constexpr uint32_t NS = D == 64 ? 10 : 5;            // ring slots
    static constexpr uint32_t QTILE = 128 * D * 2;
    static constexpr uint32_t Q = 0, RING = Q + (WIDE ? 2 : 1) * QTILE, MISC = RING + NS * SLOT;
    // barriers, the bad-value words, the merge of the two streams (narrow)
    static constexpr uint32_t BAD = MISC + 512, XCHG = BAD + BAD_RING * 32;
    static constexpr uint32_t TOTAL = XCHG + (STREAMS == 2 && !WIDE ? 2 * 128 * 8 : 0) + 1024;
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};

// mbar_wait for a whole warp in step, polling with a test that never suspends the warp: waking up from a suspended wait
// cost the products' issuer up to half its time (16-token trees of bf16 142 -> 136 us, 64-wide heads 100 -> 82).
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, long long limit)
{
    bool ok = mbar_test(bar, parity);
    if (!ok) {
        const long long t0 = clock64();
        while (!(ok = mbar_test(bar, parity)) && clock64() - t0 < limit) {
        }
    }
    return __all_sync(0xffffffffu, ok);
}

struct __align__(64) TreeParams {
    CUtensorMap tk, tv;
    const void* q;
    const void* v;
    void* o;
    float* o_part;    // [2 * grid][D / 4][ROWS][4], DEC [2 * grid][ROWS][D]
    float2* ml_part;  // [2 * grid][ROWS]: (max in log2 units, sum)
    const int32_t* kv_len;
    const int32_t* n_new;
    const uint32_t* mask;
    int* err;
    uint64_t k_hstride;  // values a kv head of the cache
    // DEC
    float* scores;    // [batch][heads][s_stride] unscaled
    float2* row_ml;   // [batch][heads]: (max in log2 units, sum) of rows written whole
    float* weight;    // [batch][kv_heads][w_stride]
    uint64_t s_stride, w_stride;
    uint32_t batch, n_tok, heads, kv_heads, group, max_len, o_type, grid;
    float scale_log2;
};

__device__ __forceinline__ uint32_t seq_cached(const TreeParams& p, uint32_t b)
{
    const int32_t l = __ldg(p.kv_len + b);
    return l > 0 ? min(uint32_t(l), p.max_len) : 0u;
}
__device__ __forceinline__ uint32_t seq_drafted(const TreeParams& p, uint32_t b)
{
    if (!p.n_new)
        return p.n_tok;
    const int32_t n = __ldg(p.n_new + b);
    return n > 0 ? min(uint32_t(n), p.n_tok) : 0u;
}

// The line of key tiles: sequence b holds kv_heads * rb segments (row blocks fastest) of `tiles` tiles each.
// toks: the tokens that have rows; drafted: those that have a key behind the cached ones (none with DEC).
struct SeqUnits {
    uint32_t cached, drafted, toks, tiles, rb;
    __device__ uint32_t units(const TreeParams& p) const { return tiles * rb * p.kv_heads; }
};
template <class C>
__device__ __forceinline__ SeqUnits seq_units(const TreeParams& p, uint32_t b)
{
    SeqUnits s;
    s.cached = seq_cached(p, b);
    s.drafted = C::DECODE ? 0u : seq_drafted(p, b);
    s.toks = C::DECODE ? 1u : s.drafted;
    s.tiles = (s.cached + s.drafted + C::TK - 1) / C::TK;
    s.rb = (p.group * s.toks + C::ROWS - 1) / C::ROWS;
    return s;
}
// Down to one tile a CTA: 8 drafted tokens over 512 keys of 8 kv heads (40 tiles) run in 11.0 us so, 13.5 with two or
// more tiles a CTA, 15.7 with four.
__device__ __forceinline__ uint32_t units_per_cta(const TreeParams& p, uint32_t total)
{
    return total ? (total + p.grid - 1) / p.grid : 1;
}

// One CTA's walk over its part of the line, segment piece by segment piece; every role walks alike.
struct Walk {
    uint32_t b;      // sequence
    uint32_t rem;    // units of it before this place
    uint32_t left;   // units this CTA has left
    bool first;      // the piece starts at the CTA's first unit
};
struct Piece {
    uint32_t b, kvh, rblk, t0, nb, cached, drafted, rows, slot;  // rows: the segment line's (group * toks)
    bool whole;
};
template <class C>
__device__ __forceinline__ bool next_piece(const TreeParams& p, Walk& w, Piece& x)
{
    while (w.left && w.b < p.batch) {
        const SeqUnits s = seq_units<C>(p, w.b);
        if (w.rem >= s.units(p)) {
            ++w.b;
            w.rem = 0;
            continue;
        }
        const uint32_t seg = w.rem / s.tiles;
        x.b = w.b;
        x.kvh = seg / s.rb;
        x.rblk = seg % s.rb;
        x.t0 = w.rem % s.tiles;
        x.nb = min(s.tiles - x.t0, w.left);
        x.rows = p.group * s.toks;
        x.cached = s.cached;
        x.drafted = s.drafted;
        x.whole = x.nb == s.tiles;
        x.slot = 2 * blockIdx.x + (w.first ? 0 : 1);
        w.rem += x.nb;
        w.left -= x.nb;
        w.first = false;
        return true;
    }
    return false;
}

// Ring positions, from the piece's first, of its tile t's K and V: K0 V0 K1 V1 ... when every tile serves both
// streams (WIDE); K0 K1 V0 K2 V1 K3 ... when tiles alternate between S buffers.
template <bool WIDE>
__device__ __forceinline__ uint32_t k_at(uint32_t t)
{
    return WIDE ? 2 * t : t < 2 ? t : 2 * t - 1;
}
template <bool WIDE>
__device__ __forceinline__ uint32_t v_at(uint32_t t, uint32_t nb)
{
    return WIDE ? 2 * t + 1 : nb == 1 ? 1 : 2 + t + min(t, nb - 2);
}

// 32 visibility bits of drafted keys first .. first + 31 (first may be negative: cached keys, seen by all) for token
// tok of sequence b with `drafted` tokens.
__device__ __forceinline__ uint32_t mask_word(const TreeParams& p, uint32_t b, uint32_t tok, uint32_t w)
{
    if (!p.mask)
        return tok >= 32 * w + 31 ? 0xFFFFFFFFu : tok < 32 * w ? 0u : (2u << (tok - 32 * w)) - 1u;
    const uint32_t nw = (p.n_tok + 31) / 32;
    return w < nw ? __ldg(p.mask + (uint64_t(b) * p.n_tok + tok) * nw + w) : 0u;
}
__device__ __forceinline__ uint32_t seen_bits(const TreeParams& p, uint32_t b, uint32_t tok, uint32_t drafted, int first)
{
    if (first <= -32)
        return 0xFFFFFFFFu;
    if (first >= int(drafted))
        return 0u;
    const uint32_t ahead = drafted - uint32_t(max(first, 0));  // drafted keys from max(first, 0) on
    uint32_t x;
    if (first < 0) {
        x = mask_word(p, b, tok, 0);
        if (ahead < 32)
            x &= (1u << ahead) - 1u;
        return x << -first | ((1u << -first) - 1u);
    }
    const uint32_t w = uint32_t(first) / 32, sh = uint32_t(first) % 32;
    x = __funnelshift_r(mask_word(p, b, tok, w), sh ? mask_word(p, b, tok, w + 1) : 0u, sh);
    return ahead < 32 ? x & ((1u << ahead) - 1u) : x;
}
__device__ __forceinline__ bool token_sees(const TreeParams& p, uint32_t b, uint32_t tok, uint32_t j)
{
    return mask_word(p, b, tok, j / 32) >> (j % 32) & 1u;
}

// The bits of the pair's 16-bit values that are not finite.
template <bool BF>
__device__ __forceinline__ uint32_t not_finite(uint32_t u)
{
    const uint32_t e = BF ? 0x7F80u : 0x7C00u;
    uint32_t m = (u & e) == e ? 0xFFFFu : 0u;
    if ((u >> 16 & e) == e)
        m |= 0xFFFF0000u;
    return m;
}

// Which of 32 columns of a row of values hold +inf, -inf, NaN: a bit each in r.x, r.y, r.z.
template <bool BF>
__device__ __forceinline__ void odd_columns(const uint16_t* row, uint3& r)
{
#pragma unroll 1
    for (uint32_t e = 0; e < 32; e += 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + e);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t h = w[i / 2] >> (i % 2 * 16), bit = 1u << (e + i);
            if ((not_finite<BF>(h) & 0xFFFFu) == 0)
                continue;
            if (h & (BF ? 0x7Fu : 0x3FFu))
                r.z |= bit;
            else if (h & 0x8000u)
                r.y |= bit;
            else
                r.x |= bit;
        }
    }
}

// The end of a piece some of whose values are not finite: in columns [c0, c1) (multiples of 32) every row (`on`) gets
// what those it sees add up to, an infinity, or NaN where there are both or a NaN.  Drafted values are named by
// the bits of bad; with `scan` the `keys` cached ones from key j0 on are read too.  Value d of this thread's row lies
// at (d / 4) * step + d % 4 from `at`.  Warp-collective; out of line, so that it costs the others no registers.
template <int D, bool BF>
__device__ __noinline__ void odd_values(const TreeParams& p, uint32_t b, uint32_t kvh, uint32_t cached, uint32_t tok,
                                        const uint32_t* bad, bool scan, uint32_t j0, uint32_t keys, uint32_t c0, uint32_t c1,
                                        bool on, void* out, uint64_t at, uint32_t step, uint32_t type)
{
    const uint16_t* const v = static_cast<const uint16_t*>(p.v) + (uint64_t(b) * p.kv_heads + kvh) * p.k_hstride;
#pragma unroll 1
    for (uint32_t c = c0; c < c1; c += 32) {
        uint3 r = make_uint3(0, 0, 0);
        if (scan) {
#pragma unroll 1
            for (uint32_t j = threadIdx.x & 31; j < keys; j += 32)
                odd_columns<BF>(v + uint64_t(j0 + j) * D + c, r);
            r = make_uint3(__reduce_or_sync(0xffffffffu, r.x), __reduce_or_sync(0xffffffffu, r.y),
                           __reduce_or_sync(0xffffffffu, r.z));
        }
        if (!on)
            continue;
#pragma unroll 1
        for (uint32_t i = 0; i < 8; ++i)
            for (uint32_t bits = bad[i]; bits; bits &= bits - 1) {
                const uint32_t j = i * 32 + __ffs(bits) - 1;
                if (token_sees(p, b, tok, j))
                    odd_columns<BF>(v + uint64_t(cached + j) * D + c, r);
            }
        for (uint32_t bits = r.x | r.y | r.z; bits; bits &= bits - 1) {
            const uint32_t e = __ffs(bits) - 1, d = c + e;
            const float z = (r.z | (r.x & r.y)) >> e & 1u ? NAN : r.x >> e & 1u ? INFINITY : -INFINITY;
            out_store1(out, at + uint64_t(d / 4) * step + d % 4, z, type);
        }
    }
}

// Thread i of n copies its share of a piece's first `rows` rows of q into shared memory and zeroes the rows up to `upto`.
template <class C, int D>
__device__ __forceinline__ void load_q(const TreeParams& p, const Piece& x, uint32_t sQ, uint32_t i, uint32_t n, uint32_t rows,
                                       uint32_t upto)
{
    constexpr uint32_t CH = D / 8;  // 16-byte chunks a row
    const uint32_t step = n / CH, c = i % CH;
    uint32_t r = i / CH, g = (x.rblk * C::ROWS + r) % p.group;
    const uint16_t* const q = static_cast<const uint16_t*>(p.q);
    const uint16_t* src =
        q + ((uint64_t(x.b) * p.n_tok + (x.rblk * C::ROWS + r) / p.group) * p.heads + x.kvh * p.group + g) * D + c * 8;
    for (; r < upto; r += step) {
        cp_async16(sQ + (r >> 7) * C::QTILE + (c >> 3) * C::QBOX + swz(r & 127, c & 7, 128), r < rows ? src : q, r < rows);
        src += step * D;
        for (g += step; g >= p.group; g -= p.group)
            src += (p.heads - p.group) * D;  // the group's heads of the next token
    }
    cp_async_commit();
    cp_async_wait<0>();
    fence_proxy_async_smem();
}

template <int D, bool BF, bool WIDE, bool DEC>
__global__ void __launch_bounds__((TreeCfg<D, WIDE, DEC>::NT), 1) tree_tc_kernel(const __grid_constant__ TreeParams p)
{
    using C = TreeCfg<D, WIDE, DEC>;
    constexpr uint32_t TK = C::TK, ROWS = C::ROWS, NS = C::NS, SC = TK;  // SC: TMEM columns of an S buffer
    constexpr uint32_t COLO = 256;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    const uint32_t sQ = base + C::Q, sR = base + C::RING, sB = base + C::MISC;
    auto full = [&](uint32_t s) { return sB + 8 * s; };
    auto empty = [&](uint32_t s) { return sB + 80 + 8 * s; };
    auto v_raw = [&](uint32_t s) { return sB + 160 + 8 * s; };  // a V tile that the cleaner still has to pass on
    auto s_full = [&](uint32_t x) { return sB + 240 + 8 * x; };
    auto p_full = [&](uint32_t x) { return sB + 256 + 8 * x; };
    auto pv_done = [&](uint32_t x) { return sB + 272 + 8 * x; };
    const uint32_t q_full = sB + 288, q_empty = sB + 296, mma_done = sB + 304;
    const uint32_t q_first = sB + 312;  // the first piece's rows of q
    volatile uint32_t* const plan = reinterpret_cast<volatile uint32_t*>(smem + C::MISC + 320);  // b, rem, left, tmem
    volatile uint32_t* const dead = plan + 4;  // a softmax warp gave up
    // P in fp16 is 2^RISE times the weight: at most 2^15 with the 2^8 by which a maximum may be passed, and that much further
    // from fp16's smallest values, where many small weights beside one large would be lost that the sum counts.
    constexpr float RISE = BF ? 0.0f : 7.0f;
    uint32_t* const bad = reinterpret_cast<uint32_t*>(smem + C::BAD);
    float2* const xchg = reinterpret_cast<float2*>(smem + C::XCHG);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the combine may be scheduled now
    if (threadIdx.x == 32) {
        for (uint32_t s = 0; s < NS; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(v_raw(s), 1);
        }
        for (uint32_t x = 0; x < 2; ++x) {
            mbar_init(s_full(x), 1);
            mbar_init(p_full(x), 128);
            mbar_init(pv_done(x), 1);
        }
        mbar_init(q_full, 64);
        mbar_init(q_first, 128 * C::STREAMS);
        mbar_init(q_empty, 1);
        mbar_init(mma_done, 1);
        *dead = 0;
        fence_barrier_init();
    }
    if (warp == 3 && lane < 8)
        bad[lane] = 0;
    if (warp == 2) {
        tmem_alloc(base + C::MISC + 332, 512);
        tmem_relinquish();
    }
    if (warp == 0) {
        // this CTA's part of the line: [u0, u1), then the sequence u0 lies in
        uint32_t units = lane < p.batch ? seq_units<C>(p, lane).units(p) : 0, total = units;
        for (uint32_t i = lane + 32; i < p.batch; i += 32)
            total += seq_units<C>(p, i).units(p);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            total += __shfl_xor_sync(0xffffffffu, total, o);
        const uint32_t per = units_per_cta(p, total), u0 = min(total, per * blockIdx.x), u1 = min(total, u0 + per);
        uint32_t at = 0;
        uint32_t b = 0, rem = 0;
        for (uint32_t i0 = 0; u0 < u1; i0 += 32) {
            uint32_t incl = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o)
                    incl += y;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at + incl > u0);
            if (hit) {
                const int l = __ffs(hit) - 1;
                b = i0 + l;
                rem = u0 - at - __shfl_sync(0xffffffffu, incl - units, l);
                break;
            }
            at += __shfl_sync(0xffffffffu, incl, 31);
            units = i0 + 32 + lane < p.batch ? seq_units<C>(p, i0 + 32 + lane).units(p) : 0;
        }
        if (lane == 0) {
            plan[0] = b;
            plan[1] = rem;
            plan[2] = u1 - u0;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, plan[3], 0);
    Walk w{plan[0], plan[1], plan[2], true};
    Piece x;
    bool ok = true;
    uint32_t n0 = 0;  // ring position of the piece's first tile

    if (warp < 4) {
        if constexpr (C::STREAMS == 2)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 104;\n" ::: "memory");
        if (warp == 0 && lane == 0) {
            // ---------------- TMA producer ----------------
            tma_prefetch_desc(&p.tk);
            tma_prefetch_desc(&p.tv);
            uint32_t loads = 0;
            while (ok && next_piece<C>(p, w, x)) {
                const int hd = int(x.b * p.kv_heads + x.kvh);
                // Tiles that no other row block reads leave L2 first: the scores and parts stay (8 x 16-32K keys with
                // weights 148 -> 141 us, one sequence of 131072 70 -> 62).
                const uint64_t hint = x.rows <= ROWS ? l2_evict_first() : l2_evict_normal();
                // loads in ring order
                for (uint32_t i = 0; i < 2 * x.nb; ++i) {
                    bool is_k;
                    uint32_t t;
                    if (WIDE) {
                        is_k = (i & 1) == 0;
                        t = i / 2;
                    } else if (i < min(x.nb, 2u)) {
                        is_k = true;
                        t = i;
                    } else if (x.nb == 1) {
                        is_k = false;
                        t = 0;
                    } else {
                        // V0 K2 V1 K3 ... V(nb-3) K(nb-1) V(nb-2) V(nb-1)
                        const uint32_t j = i - 2;
                        is_k = (j & 1) && j / 2 + 2 < x.nb;
                        t = j < 2 * (x.nb - 2) ? j / 2 + (is_k ? 2 : 0) : j - (x.nb - 2);
                    }
                    const uint32_t n = n0 + i, s = n % NS;
                    if (n >= NS && !mbar_wait(empty(s), (n / NS + 1) & 1, WAIT_LIMIT)) {
                        ok = false;
                        break;
                    }
                    // V tiles past the cached keys arrive at the cleaner, which passes them on to `full`
                    const uint32_t bar = !is_k && (x.t0 + t + 1) * TK > x.cached ? v_raw(s) : full(s);
                    mbar_expect_tx(bar, C::SLOT);
                    for (uint32_t c = 0; c < D / 64; ++c)
                        tma_load_3d_hint(sR + s * C::SLOT + c * C::KBOX, is_k ? &p.tk : &p.tv, bar, c * 64,
                                         int((x.t0 + t) * TK), hd, hint);
                    loads = n + 1;
                }
                n0 += 2 * x.nb;
            }
            if (!ok) {
                atomicExch(p.err, 41);
                // the copies in flight, the last NS loads at most, land before the CTA leaves
                for (uint32_t n = loads > NS ? loads - NS : 0; n < loads; ++n)
                    mbar_wait(full(n % NS), (n / NS) & 1, WAIT_LIMIT);
            }
        } else if (warp == 1) {
            // ---------------- UMMA issuer: the whole warp in step, one lane issues ----------------
            const uint32_t lead = elect_lane();
            // Descriptors: one 64-bit add an operand (the start address field never carries into the next).
            constexpr uint32_t F = BF ? 1u : 0u;
            const uint32_t idesc_qk = idesc_f16(F, F, 0, 0, 128, TK);
            const uint32_t idesc_pv = idesc_f16(F, F, 0, 1, 128, D);
            const uint64_t dq = sdesc(sQ, 16, 1024), dk = sdesc(sR, 16, 1024), dv = sdesc(sR, C::KBOX, 1024);
            auto qk = [&](uint32_t sbuf, uint32_t qt, uint32_t slot) {
                const uint64_t a = dq + (qt * C::QTILE >> 4), b = dk + (slot * C::SLOT >> 4);
#pragma unroll
                for (uint32_t ks = 0; ks < D / 16; ++ks)
                    umma_ss_lead(lead, tmem + sbuf * SC, a + (((ks >> 2) * C::QBOX + (ks & 3) * 32) >> 4),
                            b + (((ks >> 2) * C::KBOX + (ks & 3) * 32) >> 4), idesc_qk, ks > 0);
            };
            // P.V over the tile's 16-key groups that hold keys (the cleaner has made the last group's other rows 0)
            auto pv = [&](uint32_t sbuf, uint32_t ot, uint32_t slot, uint32_t t, bool acc) {
                const uint64_t b = dv + (slot * C::SLOT >> 4);
                const uint32_t keys = x.cached + x.drafted - (x.t0 + t) * TK, d = tmem + COLO + ot * 128, a = tmem + sbuf * SC;
                if (keys >= TK) {
#pragma unroll
                    for (uint32_t part = 0; part < (BF ? 2 : 1); ++part)
#pragma unroll
                        for (uint32_t kk = 0; kk < TK / 16; ++kk)
                            umma_ts_lead(lead, d, a + part * (TK / 2) + kk * 8, b + (kk * 2048 >> 4), idesc_pv,
                                    acc || part > 0 || kk > 0);
                } else {
                    for (uint32_t part = 0; part < (BF ? 2 : 1); ++part)
                        for (uint32_t kk = 0; kk < (keys + 15) / 16; ++kk)
                            umma_ts_lead(lead, d, a + part * (TK / 2) + kk * 8, b + (kk * 2048 >> 4), idesc_pv,
                                    acc || part > 0 || kk > 0);
                }
            };
            uint32_t pieces = 0, pc = 0;  // pc: parity of each p_full's phases so far
            auto wait_full = [&](uint32_t n) { return mbar_wait_warp(full(n % NS), (n / NS) & 1, WAIT_LIMIT); };
            auto wait_v = [&](uint32_t t) { return wait_full(n0 + v_at<WIDE>(t, x.nb)); };
            while (ok && next_piece<C>(p, w, x)) {
                x.nb = __shfl_sync(0xffffffffu, x.nb, 0);  // so that the compiler knows it to be uniform
                x.t0 = __shfl_sync(0xffffffffu, x.t0, 0);
                x.cached = __shfl_sync(0xffffffffu, x.cached, 0);
                x.drafted = __shfl_sync(0xffffffffu, x.drafted, 0);
                if (!(ok = pieces ? mbar_wait_warp(q_full, (pieces - 1) & 1, WAIT_LIMIT) : mbar_wait_warp(q_first, 0, WAIT_LIMIT)))
                    break;
                ++pieces;
                if (WIDE) {
                    if (!(ok = wait_full(n0)))
                        break;
                    fence_after();
                    for (uint32_t y = 0; y < 2; ++y) {
                        qk(y, y, n0 % NS);
                        umma_commit_lead(lead, s_full(y));
                    }
                    umma_commit_lead(lead, empty(n0 % NS));
                    if (x.nb == 1)
                        umma_commit_lead(lead, q_empty);
                    for (uint32_t t = 0; t < x.nb && ok; ++t) {
                        const uint32_t vs = (n0 + 2 * t + 1) % NS, ks = (n0 + 2 * t + 2) % NS;
                        ok = wait_v(t);
                        for (uint32_t y = 0; y < 2 && ok; ++y) {
                            if (!(ok = mbar_wait_warp(p_full(y), pc >> y & 1u, WAIT_LIMIT)))
                                break;
                            pc ^= 1u << y;
                            fence_after();
                            pv(y, y, vs, t, t > 0);
                            if (y == 1)
                                umma_commit_lead(lead, empty(vs));
                            if (t + 1 < x.nb) {
                                if (y == 0 && !(ok = wait_full(n0 + 2 * t + 2)))
                                    break;
                                qk(y, y, ks);
                                umma_commit_lead(lead, s_full(y));
                                if (y == 1) {
                                    umma_commit_lead(lead, empty(ks));
                                    if (t + 2 == x.nb)
                                        umma_commit_lead(lead, q_empty);
                                }
                            } else {
                                umma_commit_lead(lead, pv_done(y));
                            }
                        }
                    }
                } else {
                    for (uint32_t t = 0; t < min(x.nb, 2u) && ok; ++t) {
                        if (!(ok = wait_full(n0 + t)))
                            break;
                        fence_after();
                        qk(t, 0, (n0 + t) % NS);
                        umma_commit_lead(lead, s_full(t));
                        umma_commit_lead(lead, empty((n0 + t) % NS));
                        if (t + 1 == x.nb)
                            umma_commit_lead(lead, q_empty);
                    }
                    for (uint32_t t = 0; t < x.nb && ok; ++t) {
                        const uint32_t y = t & 1, vs = (n0 + v_at<WIDE>(t, x.nb)) % NS;
                        if (!(ok = wait_v(t) && mbar_wait_warp(p_full(y), pc >> y & 1u, WAIT_LIMIT)))
                            break;
                        pc ^= 1u << y;
                        fence_after();
                        pv(y, C::STREAMS == 2 ? y : 0, vs, t, C::STREAMS == 2 ? t > 1 : t > 0);
                        umma_commit_lead(lead, empty(vs));
                        if (C::STREAMS == 1) {
                            umma_commit_lead(lead, pv_done(0));  // every product, for a rescale of O
                            if (t + 1 == x.nb)
                                umma_commit_lead(lead, pv_done(1));  // the piece's last
                        } else if (t + 2 >= x.nb) {
                            umma_commit_lead(lead, pv_done(y));
                        }
                        if (t + 2 < x.nb) {
                            const uint32_t kn = n0 + k_at<WIDE>(t + 2);
                            if (!(ok = wait_full(kn)))
                                break;
                            qk(y, 0, kn % NS);
                            umma_commit_lead(lead, s_full(y));
                            umma_commit_lead(lead, empty(kn % NS));
                            if (t + 3 == x.nb)
                                umma_commit_lead(lead, q_empty);
                        }
                    }
                }
                n0 += 2 * x.nb;
            }
            if (!ok && lane == 0)
                atomicExch(p.err, 42);
            umma_commit_lead(lead, mma_done);  // every product issued above has finished before TMEM is freed
            mbar_wait_warp(mma_done, 0, WAIT_LIMIT);
        } else if (warp >= 2) {
            // ---------------- q loaders, the second also cleans the drafted values ----------------
            // Rows past the drafted ones are zero: nobody reads what S and O hold for them, but products of zeros draw less
            // power, which is what holds the clock down here.
            uint32_t pieces = 0, used = 0;  // used: parity of each slot's v_raw uses so far
            uint32_t dirty = 0;             // rows from here on are zero
            while (ok && next_piece<C>(p, w, x)) {
                if (pieces > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (pieces - 1) & 1, WAIT_LIMIT))))
                    break;
                const uint32_t rows = min(ROWS, x.rows - x.rblk * ROWS);
                uint32_t* const mybad = bad + pieces % BAD_RING * 8;
                if (pieces > 0) {  // the softmax warps load the first piece's
                    if (warp == 3 && lane < 8)
                        mybad[lane] = 0;  // before q_full, on which the piece's epilogue depends
                    load_q<C, D>(p, x, sQ, threadIdx.x - 64, 64, rows, max(rows, dirty));
                    __syncwarp();
                    mbar_arrive(q_full);
                }
                dirty = rows;
                ++pieces;
                if (warp == 2)
                    continue;
                const uint32_t first = x.cached / TK;  // the first tile with keys past the cached ones
                for (uint32_t t = first > x.t0 ? first - x.t0 : 0; t < x.nb; ++t) {
                    const uint32_t j0 = (x.t0 + t) * TK, s = (n0 + v_at<WIDE>(t, x.nb)) % NS;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(v_raw(s), used >> s & 1u, WAIT_LIMIT))))
                        break;
                    used ^= 1u << s;
                    const uint32_t r0 = x.cached > j0 ? x.cached - j0 : 0;
                    const uint32_t r1 = min(TK, x.cached + x.drafted - j0);  // rows past it are no keys
                    uint8_t* const tile = smem + C::RING + s * C::SLOT;
                    auto chunk = [&](uint32_t i) {
                        const uint32_t r = i / (D / 8), c = i % (D / 8);
                        return reinterpret_cast<uint4*>(tile + (c >> 3) * C::KBOX + swz(r, c & 7, 128));
                    };
                    for (uint32_t i = r0 * (D / 8) + lane; i < r1 * (D / 8); i += 32) {
                        uint4* const e = chunk(i);
                        const uint4 u = *e;
                        const uint4 m = make_uint4(not_finite<BF>(u.x), not_finite<BF>(u.y), not_finite<BF>(u.z),
                                                   not_finite<BF>(u.w));
                        if (m.x | m.y | m.z | m.w) {
                            *e = make_uint4(u.x & ~m.x, u.y & ~m.y, u.z & ~m.z, u.w & ~m.w);
                            const uint32_t j = j0 + i / (D / 8) - x.cached;
                            atomicOr(&mybad[j / 32], 1u << (j % 32));
                        }
                    }
                    for (uint32_t i = r1 * (D / 8) + lane; i < (r1 + 15) / 16 * 16 * (D / 8); i += 32)
                        *chunk(i) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(full(s));
                }
                n0 += 2 * x.nb;
            }
            if (!ok && lane == 0)
                atomicExch(p.err, 43);
        }
    } else {
        if constexpr (C::STREAMS == 2)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n" ::: "memory");
        // ---------------- softmax and epilogue ----------------
        const uint32_t y = (warp - 4) >> 2, ql = (warp & 3) * 32, row = ql + lane;
        const uint32_t tl = tmem + (ql << 16);
        const float scale = p.scale_log2;
        // sc: parity of each s_full's phases; pieces ended with tiles of this stream; tiles of all pieces so far
        uint32_t pieces = 0, sc = 0, ends = 0, products = 0;
        while (ok && next_piece<C>(p, w, x)) {
            if (pieces == 0) {
                load_q<C, D>(p, x, sQ, threadIdx.x - 128, 128 * C::STREAMS, min(ROWS, x.rows - x.rblk * ROWS), ROWS);
                mbar_arrive(q_first);
            }
            const uint32_t live_rows = x.rows;
            const uint32_t rbase = x.rblk * ROWS + (WIDE ? y * 128 : 0), r = rbase + row;
            const bool live = r < live_rows, warp_live = rbase + ql < live_rows;
            const uint32_t tok = DEC ? 0u : min(r, live_rows - 1) / p.group;
            float m = -INFINITY, l = 0.0f;
            uint32_t mine = 0;  // tiles of this stream so far
            const uint32_t step = WIDE || C::STREAMS == 1 ? 1 : 2;
            for (uint32_t t = WIDE || C::STREAMS == 1 ? 0 : y; t < x.nb; t += step, ++mine) {
                const uint32_t sb = WIDE ? y : t & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(s_full(sb), sc >> sb & 1u, WAIT_LIMIT));
                if (!ok)
                    break;
                sc ^= 1u << sb;
                fence_after();
                uint32_t s[TK / 32][32];
                if (warp_live) {
                    if constexpr (TK == 128)
                        tmem_ld128(tl + sb * SC, s);
                    else
                        tmem_ld64(tl + sb * SC, s);
                    tmem_wait_ld();
#pragma unroll
                    for (uint32_t c = 0; c < TK / 32; ++c)
                        reg_fence(s[c]);
                    const uint32_t j0 = (x.t0 + t) * TK;
                    if (j0 + TK > x.cached) {
#pragma unroll
                        for (uint32_t c = 0; c < TK / 32; ++c) {
                            const uint32_t bits = seen_bits(p, x.b, tok, x.drafted, int(j0 + c * 32) - int(x.cached));
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(bits >> e & 1u))
                                    s[c][e] = 0xFF800000u;  // -inf
                        }
                    }
                    float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (uint32_t c = 0; c < TK; c += 8)
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e)
                            mq[e] = max3f(mq[e], __uint_as_float(s[(c + 2 * e) >> 5][(c + 2 * e) & 31]),
                                          __uint_as_float(s[(c + 2 * e + 1) >> 5][(c + 2 * e + 1) & 31]));
                    const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * scale;
                    float f = 1.0f;
                    bool resc = false;
                    if (mx > m + 8.0f) {
                        f = m == -INFINITY ? 0.0f : ex2(m - mx);
                        m = mx;
                        l *= f;
                        resc = true;
                    }
                    const float mneg = m == -INFINITY ? 0.0f : RISE - m;
                    const uint64_t scale2 = pack2(scale, scale), mneg2 = pack2(mneg, mneg);
                    uint64_t sum2[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
                    for (uint32_t c = 0; c < TK / 32; ++c) {
                        // 32 scores -> 16 columns of P (and of what rounding left over)
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float a, b;
                            unpack2(ffma2(pack2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), scale2, mneg2),
                                    a, b);
                            a = ex2(a);
                            b = ex2(b);
                            sum2[e & 1] = fadd2(sum2[e & 1], pack2(a, b));
                            if (BF) {
                                hi[e] = Elem<__nv_bfloat16>::pack(a, b);
                                lo[e] = Elem<__nv_bfloat16>::pack(a - __uint_as_float(hi[e] << 16),
                                                                  b - __uint_as_float(hi[e] & 0xFFFF0000u));
                            } else {
                                hi[e] = Elem<__half>::pack(a, b);
                            }
                        }
                        tmem_st16(tl + sb * SC + c * 16, hi);
                        if (BF)
                            tmem_st16(tl + sb * SC + TK / 2 + c * 16, lo);
                    }
                    {
                        float s0, s1, s2, s3;
                        unpack2(sum2[0], s0, s1);
                        unpack2(sum2[1], s2, s3);
                        l += (s0 + s1) + (s2 + s3);
                    }
                    // Rescale O before the next product adds to it.  Two streams: the product before was committed
                    // with this S.  One stream: wait for it here.
                    if (__any_sync(0xffffffffu, resc && mine > 0)) {
                        if (C::STREAMS == 1)
                            ok = __all_sync(0xffffffffu, mbar_wait(pv_done(0), (products + mine - 1) & 1, WAIT_LIMIT));
                        fence_after();
                        const float gsc = resc ? f : 1.0f;
#pragma unroll
                        for (uint32_t c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(tl + COLO + (C::STREAMS == 2 ? y * 128 : 0) + c * 32, o);
                            tmem_wait_ld();
                            reg_fence(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * gsc);
                            tmem_st32(tl + COLO + (C::STREAMS == 2 ? y * 128 : 0) + c * 32, o);
                        }
                    }
                    tmem_wait_st();
                }
                fence_before();
                mbar_arrive(p_full(sb));
                if (!ok)
                    break;
                if (DEC && live) {  // the row's scores, while the product runs; s_stride is a multiple of the tile
                    float* const d =
                        p.scores + (uint64_t(x.b) * p.heads + x.kvh * p.group + r) * p.s_stride + (x.t0 + t) * TK;
#pragma unroll
                    for (uint32_t c = 0; c < TK / 32; ++c)
#pragma unroll
                        for (uint32_t e = 0; e < 32; e += 8) {
                            const uint32_t u[8] = {s[c][e],     s[c][e + 1], s[c][e + 2], s[c][e + 3],
                                                   s[c][e + 4], s[c][e + 5], s[c][e + 6], s[c][e + 7]};
                            st_global_v8(d + c * 32 + e, u);
                        }
                }
            }
            // The stream's last product.  One stream: on a barrier of its own, since pv_done(0) may by now have completed
            // one phase or two since S was seen, which a wait by parity cannot tell apart.
            if (ok && mine > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(pv_done(C::STREAMS == 2 ? y : 1), ends & 1, WAIT_LIMIT));
                fence_after();
                ++ends;
                products += x.nb;
            }
            // ---- epilogue: the rows' o, or their part of it
            m -= RISE;  // what the sum and o are relative to
            const uint32_t* const mybad = bad + pieces % BAD_RING * 8;
            ++pieces;
            float f0 = 1.0f, f1 = 0.0f;  // weights of the two streams' parts (narrow)
            bool have1 = false;
            constexpr bool MERGE = C::STREAMS == 2 && !WIDE;
            if (MERGE) {
                xchg[y * 128 + row] = make_float2(m, l);
                if (!ok)
                    *dead = 1;
                fence_before();  // either half reads both streams' O, of which it has waited for one
                named_bar(1, 256);
                fence_after();
                ok = *dead == 0;  // a warp that gave up ends the walk of all, which meet at these barriers
                const float2 a = xchg[row], b = xchg[128 + row];
                const float M = fmaxf(a.x, b.x);
                f0 = a.x == -INFINITY ? 0.0f : ex2(a.x - M);
                f1 = b.x == -INFINITY ? 0.0f : ex2(b.x - M);
                have1 = x.nb > 1;
                m = M;
                l = have1 ? a.y * f0 + b.y * f1 : a.y * f0;
            }
            if (ok && warp_live) {
                const float inv = x.whole ? (l != 0.0f ? 1.0f / l : 0.0f) : 1.0f;
                const uint32_t lrow = (WIDE ? y * 128 : 0) + row;
                void* dst = x.whole ? p.o : static_cast<void*>(p.o_part);
                const uint64_t doff =
                    x.whole ? ((uint64_t(x.b) * p.n_tok + tok) * p.heads + x.kvh * p.group + r % p.group) * D
                            : (uint64_t(x.slot) * ROWS + lrow) * D;
                if (live && (!MERGE || y == 0)) {
                    if (!x.whole)
                        p.ml_part[uint64_t(x.slot) * ROWS + lrow] = make_float2(m, l);
                    else if (DEC)
                        p.row_ml[uint64_t(x.b) * p.heads + x.kvh * p.group + r] = make_float2(m, l);
                }
                uint32_t any_bad = 0;
#pragma unroll
                for (int i = 0; i < (DEC ? 0 : 8); ++i)
                    any_bad |= mybad[i];
                bool nan = false;
                // narrow: this warpgroup's half of the columns, of both parts
                constexpr uint32_t NC = MERGE ? D / 64 : D / 32;
#pragma unroll
                for (uint32_t cc = 0; cc < NC; ++cc) {
                    const uint32_t c = MERGE ? y * NC + cc : cc;
                    uint32_t o[32];
                    tmem_ld32(tl + COLO + (WIDE ? y * 128 : 0) + c * 32, o);
                    tmem_wait_ld();
                    reg_fence(o);
                    if (MERGE) {
                        uint32_t o1[32];
                        if (have1) {
                            tmem_ld32(tl + COLO + 128 + c * 32, o1);
                            tmem_wait_ld();
                            reg_fence(o1);
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float z = __uint_as_float(o[e]) * f0;
                            if (have1)
                                z = fmaf(__uint_as_float(o1[e]), f1, z);
                            o[e] = __float_as_uint(z);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        nan |= isnan(__uint_as_float(o[e]));
                    if (live && (DEC || x.whole)) {
                        out_store32(dst, doff + c * 32, o, inv, x.whole ? p.o_type : 0u);
                    } else if (live) {
                        // A part, four columns at a time with the rows side by side: a warp's store is 512 bytes in one run
                        // instead of 32 sectors of as many lines (7700 -> 4300 cycles for 128 rows of 256).
                        float4* const d = reinterpret_cast<float4*>(p.o_part) + (uint64_t(x.slot) * (D / 4) + c * 8) * ROWS + lrow;
#pragma unroll
                        for (int g = 0; g < 8; ++g)
                            d[g * ROWS] = make_float4(__uint_as_float(o[4 * g]), __uint_as_float(o[4 * g + 1]),
                                                      __uint_as_float(o[4 * g + 2]), __uint_as_float(o[4 * g + 3]));
                    }
                }
                // A cached infinity gives NaN where its weight rounds to 0 in P, or to a second part of the other sign.  Scores
                // of NaN make l NaN and the whole row.
                const bool on = live && l > 0.0f, scan = __any_sync(0xffffffffu, nan && on);
                if (scan || any_bad) {
                    const bool rows = DEC || x.whole;
                    const uint32_t c0 = MERGE ? y * (D / 2) : 0, j0 = x.t0 * TK, j1 = min(x.cached, j0 + x.nb * TK);
                    odd_values<D, BF>(p, x.b, x.kvh, x.cached, tok, mybad, scan, j0, j1 > j0 ? j1 - j0 : 0u, c0,
                                      c0 + NC * 32, on, dst, rows ? doff : (uint64_t(x.slot) * D * ROWS + lrow * 4),
                                      rows ? 4u : 4 * ROWS, x.whole ? p.o_type : 0u);
                }
            }
            fence_before();
            if (MERGE) {
                named_bar(1, 256);  // both have read both parts: the next piece's products may overwrite them
                fence_after();
            }
        }
        if (!ok && lane == 0)
            atomicExch(p.err, 44);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 2) {
        fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Where row r of (sequence b, kv head kvh) was worked on: CTAs c0 .. c1, in the rows `lrow` of their slots.
struct RowPieces {
    uint32_t c0, c1, slot0, lrow;
    template <class C>
    __device__ uint64_t at(uint32_t c) const
    {
        return uint64_t(c == c0 ? slot0 : 2 * c) * C::ROWS + lrow;
    }
};
// Warp-collective.
template <class C>
__device__ __forceinline__ void line_sums(const TreeParams& p, uint32_t b, uint32_t& before, uint32_t& total)
{
    before = total = 0;
    for (uint32_t k = threadIdx.x & 31; k < p.batch; k += 32) {
        const uint32_t n = seq_units<C>(p, k).units(p);
        total += n;
        before += k < b ? n : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
}
template <class C>
__device__ __forceinline__ RowPieces row_pieces(const SeqUnits& s, uint32_t kvh, uint32_t r, uint32_t before, uint32_t per)
{
    const uint32_t u0 = before + (kvh * s.rb + r / C::ROWS) * s.tiles, u1 = u0 + s.tiles;
    RowPieces x;
    x.c0 = u0 / per;
    x.c1 = (u1 - 1) / per;
    x.slot0 = 2 * x.c0 + (u0 % per ? 1 : 0);
    x.lrow = r % C::ROWS;
    return x;
}
// Merges 32 pieces' (max, sum), a lane a piece, into the running M and l; returns this piece's weight, f0 that of what
// was merged before.  Warp-collective.
__device__ __forceinline__ float merge_ml(float2 ml, float& M, float& l, float& f0)
{
    float m1 = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
    const float Mn = fmaxf(M, m1);
    f0 = M == -INFINITY ? 0.0f : ex2(M - Mn);
    M = Mn;
    const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
    float ls = ml.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        ls += __shfl_xor_sync(0xffffffffu, ls, o);
    l = l * f0 + ls;
    return f;
}
// Merges the pieces of one row into o (values at o0 on, DEC): the CTA's WARPS warps take every WARPS-th group of pieces and
// meet in shared memory.  parts: WARPS * (D + 2) floats.
template <int D, class C, uint32_t WARPS>
__device__ __forceinline__ void combine_row(const TreeParams& p, const RowPieces& x, uint64_t o0, float* parts)
{
    constexpr uint32_t V = D / 32;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t step = min(32u, (x.c1 - x.c0) / WARPS + 1);  // pieces a warp takes at once
    float M = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
    for (uint32_t e = 0; e < V; ++e)
        acc[e] = 0.0f;
    for (uint32_t cb = x.c0 + warp * step; cb <= x.c1; cb += WARPS * step) {
        const uint32_t n = min(step, x.c1 - cb + 1);
        float f0;
        const float f =
            merge_ml(lane < n ? p.ml_part[x.at<C>(cb + lane)] : make_float2(-INFINITY, 0.0f), M, l, f0);
#pragma unroll
        for (uint32_t e = 0; e < V; ++e)
            acc[e] *= f0;
#pragma unroll 4
        for (uint32_t k = 0; k < n; ++k) {
            const float w = __shfl_sync(0xffffffffu, f, k);
            const float* src = p.o_part + x.at<C>(cb + k) * D + lane * V;
#pragma unroll
            for (uint32_t e = 0; e < V; e += 2) {
                const float2 z = __ldcs(reinterpret_cast<const float2*>(src + e));
                acc[e] = fmaf(z.x, w, acc[e]);
                acc[e + 1] = fmaf(z.y, w, acc[e + 1]);
            }
        }
    }
    float* const mine = parts + warp * (D + 2);
    if (lane == 0) {
        mine[D] = M;
        mine[D + 1] = l;
    }
#pragma unroll
    for (uint32_t e = 0; e < V; ++e)
        mine[lane * V + e] = acc[e];
    __syncthreads();
    M = -INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < WARPS; ++k)
        M = fmaxf(M, parts[k * (D + 2) + D]);
    for (uint32_t d = threadIdx.x; d < D; d += WARPS * 32) {
        float o = 0.0f, sum = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < WARPS; ++k) {
            const float* const z = parts + k * (D + 2);
            const float f = z[D] == -INFINITY ? 0.0f : ex2(z[D] - M);
            o = fmaf(z[d], f, o);
            sum = fmaf(z[D + 1], f, sum);
        }
        out_store1(p.o, o0 + d, sum != 0.0f ? o / sum : 0.0f, p.o_type);
    }
}

// Merges the pieces of segments that several CTAs worked on by log-sum-exp; rows of segments written whole have nothing to
// do.  A CTA takes 32 rows of one segment and 32 columns, a lane a row and a warp four columns, as the parts lie.
// Which pieces there are follows from the lengths alone and is worked out before the wait for the main kernel.
constexpr uint32_t CMB_WARPS = 8;
template <int D, bool WIDE>
__global__ void __launch_bounds__(CMB_WARPS * 32) tree_combine_kernel(const __grid_constant__ TreeParams p, uint32_t blocks)
{
    using C = TreeCfg<D, WIDE, false>;
    const uint32_t b = blockIdx.y, kvh = blockIdx.x / blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t r0 = blockIdx.x % blocks * 32, r = r0 + lane;
    uint32_t before, total;
    line_sums<C>(p, b, before, total);
    const SeqUnits s = seq_units<C>(p, b);
    RowPieces x{};
    if (r0 < p.group * s.drafted)
        x = row_pieces<C>(s, kvh, r0, before, units_per_cta(p, total));
    // Every CTA waits, with rows or without: what comes next in the stream waits for this kernel alone.
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    if (x.c0 == x.c1 || r >= p.group * s.drafted)
        return;
    x.lrow += lane;
    const uint32_t col = (blockIdx.z * CMB_WARPS + warp) * 4;
    float M = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr uint32_t AT = 8;  // pieces whose loads are in flight together
    for (uint32_t cb = x.c0; cb <= x.c1; cb += AT) {
        float2 ml[AT];
        float4 z[AT];
#pragma unroll
        for (uint32_t k = 0; k < AT; ++k)
            if (cb + k <= x.c1) {
                ml[k] = p.ml_part[x.at<C>(cb + k)];
                z[k] = __ldcs(reinterpret_cast<const float4*>(p.o_part) +
                              (uint64_t(cb + k == x.c0 ? x.slot0 : 2 * (cb + k)) * (D / 4) + col / 4) * C::ROWS + x.lrow);
            } else {
                ml[k] = make_float2(-INFINITY, 0.0f);
                z[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        float Mn = M;
#pragma unroll
        for (uint32_t k = 0; k < AT; ++k)
            Mn = fmaxf(Mn, ml[k].x);
        const float f0 = M == -INFINITY ? 0.0f : ex2(M - Mn);
        M = Mn;
        l *= f0;  // l is 0, or NaN and stays so, while there is no maximum
        acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
        for (uint32_t k = 0; k < AT; ++k) {
            const float f = ml[k].x == -INFINITY ? 0.0f : ex2(ml[k].x - M);
            l = fmaf(ml[k].y, f, l);
            acc = make_float4(fmaf(z[k].x, f, acc.x), fmaf(z[k].y, f, acc.y), fmaf(z[k].z, f, acc.z), fmaf(z[k].w, f, acc.w));
        }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const uint64_t o = ((uint64_t(b) * p.n_tok + r / p.group) * p.heads + kvh * p.group + r % p.group) * D + col;
    out_store2(p.o, o, acc.x * inv, acc.y * inv, p.o_type);
    out_store2(p.o, o + 2, acc.z * inv, acc.w * inv, p.o_type);
}

// The second half of the decode with weights, for one kv head of a sequence.  CTAs below n_weight take WKEYS keys each:
// a warp a head finds the row's maximum and sum, then each thread sums 2^(s * scale - max) / sum over the group's heads,
// in their order, for four keys and adds that to their weights.  The others combine cut rows, one each, and write the zero
// rows of empty sequences.
constexpr uint32_t WNT = 256, WKEYS = 4 * WNT, WHEADS = 64;
template <int D>
__global__ void __launch_bounds__(WNT) weights_finish_kernel(const __grid_constant__ TreeParams p, uint32_t n_weight)
{
    using C = TreeCfg<D, false, true>;
    __shared__ float2 ml[WHEADS];  // (max, 1 / sum) of up to WHEADS heads at a time
    __shared__ float parts[WNT / 32 * (D + 2)];
    const uint32_t b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t before, total;
    line_sums<C>(p, b, before, total);
    const SeqUnits s = seq_units<C>(p, b);
    const uint32_t per = units_per_cta(p, total);
    asm volatile("griddepcontrol.wait;\n" ::: "memory");  // every CTA, as above
    if (blockIdx.x >= n_weight) {
        const uint32_t r = blockIdx.x - n_weight;
        const uint64_t o0 = (uint64_t(b) * p.heads + kvh * p.group + r) * D;
        if (s.tiles == 0) {
            if (threadIdx.x < D)
                out_store1(p.o, o0 + threadIdx.x, 0.0f, p.o_type);
            return;
        }
        const RowPieces x = row_pieces<C>(s, kvh, r, before, per);
        if (x.c0 == x.c1)
            return;
        combine_row<D, C, WNT / 32>(p, x, o0, parts);
        return;
    }
    const uint32_t L = s.cached, j = blockIdx.x * WKEYS + threadIdx.x * 4;
    if (blockIdx.x * WKEYS >= L)
        return;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t h0 = 0; h0 < p.group; h0 += WHEADS) {
        const uint32_t nh = min(WHEADS, p.group - h0);
        const uint64_t row0 = uint64_t(b) * p.heads + kvh * p.group + h0;
        __syncthreads();
        for (uint32_t h = warp; h < nh; h += WNT / 32) {
            const RowPieces x = row_pieces<C>(s, kvh, h0 + h, before, per);
            float M = -INFINITY, l = 0.0f, f0;
            if (x.c0 == x.c1) {
                const float2 v = p.row_ml[row0 + h];
                M = v.x;
                l = v.y;
            } else {
                for (uint32_t cb = x.c0; cb <= x.c1; cb += 32)
                    merge_ml(lane < x.c1 - cb + 1 ? p.ml_part[x.at<C>(cb + lane)] : make_float2(-INFINITY, 0.0f), M, l, f0);
            }
            if (lane == 0)
                ml[h] = M == -INFINITY ? make_float2(0.0f, l) : make_float2(M, 1.0f / l);  // no maximum: l is 0 or NaN
        }
        __syncthreads();
        if (j < L) {
            const float* sc = p.scores + row0 * p.s_stride + j;
            for (uint32_t h = 0; h < nh; ++h, sc += p.s_stride) {
                const float4 z = __ldcs(reinterpret_cast<const float4*>(sc));
                const float2 c = ml[h];
                acc[0] += ex2(fmaf(z.x, p.scale_log2, -c.x)) * c.y;
                acc[1] += ex2(fmaf(z.y, p.scale_log2, -c.x)) * c.y;
                acc[2] += ex2(fmaf(z.z, p.scale_log2, -c.x)) * c.y;
                acc[3] += ex2(fmaf(z.w, p.scale_log2, -c.x)) * c.y;
            }
        }
    }
    float* w = p.weight + (uint64_t(b) * p.kv_heads + kvh) * p.w_stride + j;
    if (j + 4 <= L && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
        float4 z = *reinterpret_cast<float4*>(w);
        z.x += acc[0];
        z.y += acc[1];
        z.z += acc[2];
        z.w += acc[3];
        *reinterpret_cast<float4*>(w) = z;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < L)
            w[e] += acc[e];
}

// The dependent second kernel: scheduled while the main kernel runs out.
template <typename... A>
cudaError_t launch_dependent(void (*kern)(A...), dim3 grid, uint32_t threads, cudaStream_t st, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int D, bool WIDE, bool DEC>
cudaError_t launch_tree_t(const TreeArgs& a, bool bf, int* err, cudaStream_t st)
{
    using C = TreeCfg<D, WIDE, DEC>;
    TreeParams p;
    if (!tile_map(&p.tk, a.k, bf, D, a.k_stride, a.batch * a.kv_heads, C::TK) ||
        !tile_map(&p.tv, a.v, bf, D, a.k_stride, a.batch * a.kv_heads, C::TK))
        return cudaErrorInvalidValue;
    p.q = a.q;
    p.v = a.v;
    p.o = a.o;
    p.o_part = a.o_part;
    p.ml_part = a.ml_part;
    p.kv_len = a.kv_len;
    p.n_new = a.n_new;
    p.mask = a.mask;
    p.err = err;
    p.k_hstride = uint64_t(a.k_stride) * D;
    p.scores = a.scores;
    p.row_ml = a.row_ml;
    p.weight = a.weight;
    p.s_stride = a.s_stride;
    p.w_stride = a.k_stride;
    p.batch = a.batch;
    p.n_tok = a.n_tok;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.group = a.heads / a.kv_heads;
    p.max_len = a.max_len;
    p.o_type = a.o_type;
    p.grid = a.ctas;
    p.scale_log2 = a.scale * kLog2e;
    auto kern = bf ? tree_tc_kernel<D, true, WIDE, DEC> : tree_tc_kernel<D, false, WIDE, DEC>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL);
    if (e != cudaSuccess)
        return e;
    kern<<<a.ctas, C::NT, C::TOTAL, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess)
        return e;
    if constexpr (DEC) {
        const uint32_t nw = (p.max_len + WKEYS - 1) / WKEYS, nc = p.group;
        return launch_dependent<const TreeParams, uint32_t>(weights_finish_kernel<D>, dim3(nw + nc, p.kv_heads, p.batch),
                                                            WNT, st, p, nw);
    } else {
        const uint32_t blocks = (p.group * p.n_tok + 31) / 32;
        return launch_dependent<const TreeParams, uint32_t>(tree_combine_kernel<D, WIDE>, dim3(blocks * p.kv_heads, p.batch, D / 4 / CMB_WARPS),
                                                            CMB_WARPS * 32, st, p, blocks);
    }
}

} // namespace

// Rows a segment: 128, or 256 where the heads are narrow enough for two 128-row O tiles in TMEM and there are more rows.
uint32_t tree_rows(uint32_t n_tok, uint32_t group, uint32_t dim) { return dim < 256 && n_tok * group > 128 ? 256 : 128; }

cudaError_t launch_tree(const TreeArgs& a, int dtype, int dim, int* err, cudaStream_t st)
{
    const bool bf = dtype == kBF16, wide = tree_rows(a.n_tok, a.heads / a.kv_heads, dim) == 256;
    switch (dim) {
    case 64:
        return wide ? launch_tree_t<64, true, false>(a, bf, err, st) : launch_tree_t<64, false, false>(a, bf, err, st);
    case 128:
        return wide ? launch_tree_t<128, true, false>(a, bf, err, st) : launch_tree_t<128, false, false>(a, bf, err, st);
    case 256:
        return launch_tree_t<256, false, false>(a, bf, err, st);
    default:
        return cudaErrorInvalidValue;
    }
}

cudaError_t launch_decode_weights(const TreeArgs& a, int dtype, int dim, int* err, cudaStream_t st)
{
    const bool bf = dtype == kBF16;
    switch (dim) {
    case 64:
        return launch_tree_t<64, false, true>(a, bf, err, st);
    case 128:
        return launch_tree_t<128, false, true>(a, bf, err, st);
    case 256:
        return launch_tree_t<256, false, true>(a, bf, err, st);
    default:
        return cudaErrorInvalidValue;
    }
}

} // namespace mako
