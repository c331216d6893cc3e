// Eviction from a KV cache by accumulated attention weight (mako_cache_evict).  No counterpart in the reference.
//
// evict_select_kernel: a CTA a (sequence, kv head), for long rows a cluster of up to 8, the weights held in registers
// as order-preserving integers (SKEYS a thread; rows past a cluster's registers are read again by every pass).  The rows
// between the sinks and the recent ones compete; the weight of the last that stays is found by a radix select of 11, 11
// and 10 bits: a histogram in shared memory, merged over the cluster.  A warp whose keys all share a digit adds them at
// once, so that rows of equal weights do not queue at one counter.  All counts are integers: the result does not depend on
// the order of the adds.  Then every warp, which owns consecutive rows, writes its kept rows' indices from the count of
// those before it, ties taken from the lowest row on.
// Rows that do not compete take the key of a NaN, 0, which is the last of all: how many have it decides nothing, so no pass
// asks again which rows compete, and a pass over a key is a handful of instructions.  The loop ends as soon as a digit's
// count fits what is left to choose.  64 rows of 16-32K keys: the last is done after 14 us (21 with a test of every key in
// every pass, four barriers a pass and the bits turned at the end), of which 3 are the load, 1 the keys, 1.2 a pass over
// them and 0.7 the search after it.  Two CTAs a row take as long (37.6 and 38.1 us for the whole call): rows that fit one
// CTA's registers take one.
// evict_copy_kernel and evict_in_place_kernel copy the kept rows.  In place, row i comes from row kept[i] >= i: a CTA owns a
// 64-byte column slice of every row and walks the rows upwards in steps, reading a whole step before it writes it, so what
// a later step reads (rows at or past its own first) has not been written yet.
#include "common.cuh"
#include "kernels.h"

#include <cooperative_groups.h>

namespace mako {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t SNT = 1024, SKEYS = 32, SBINS = 2048, SMAX_CLUSTER = 8, MNT = 256;

// Weights as integers of the same order; NaN below all others, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w)
        return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t warp_incl_scan(uint32_t x)
{
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= uint32_t(o))
            x += y;
    }
    return x;
}

// Bits k with lo <= first + k < hi.
__device__ __forceinline__ uint32_t bits_within(uint32_t first, uint32_t lo, uint32_t hi)
{
    auto under = [&](uint32_t end) {  // bits k with first + k < end
        return end <= first ? 0u : end - first >= 32 ? 0xFFFFFFFFu : (1u << (end - first)) - 1u;
    };
    return under(hi) & ~under(lo);
}

// REG: a thread's keys fit its SKEYS registers.  blockDim.x: 256 or 1024.
template <bool REG>
__global__ void __launch_bounds__(SNT) evict_select_kernel(const EvictParams p)
{
    __shared__ uint32_t hist[3][SBINS], sum[SBINS], part[3][32], found[3][2], mine[2], ranks[2][32];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank(), nt = blockDim.x, warps = nt / 32;
    const uint32_t kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the copy's CTAs wait in place for the end
    const int32_t l = p.kv_len[b];
    const uint32_t len = l > 0 ? min(uint32_t(l), p.max_len) : 0u, keep = min(len, p.budget);
    const uint64_t row = uint64_t(b) * p.kv_heads + kvh;
    int32_t* const kept = p.kept + row * p.budget;
    if (kvh == 0 && rank == 0 && tid == 0)
        p.count[b] = int32_t(keep);
    for (uint32_t i = keep + rank * nt + tid; i < p.budget; i += C * nt)
        kept[i] = -1;
    if (len <= p.budget) {  // the same for the whole cluster
        for (uint32_t i = rank * nt + tid; i < len; i += C * nt)
            kept[i] = int32_t(i);
        return;
    }
    const float* const w = p.weight + row * p.k_stride;
    const uint32_t lo = p.sinks, hi = len - p.recent;  // the rows that compete
    uint32_t want = p.budget - p.sinks - p.recent;     // how many of them stay
    // warp g of the cluster owns rows [g * 32 * nk, (g + 1) * 32 * nk), lane i's every 32nd; in registers, fours of them
    uint32_t nk = (len + C * nt - 1) / (C * nt);
    if (REG)
        nk = (nk + 3) & ~3u;
    const uint32_t first = (rank * warps + warp) * 32 * nk, j0 = first + lane;
    auto competes = [&](uint32_t j) { return j - lo < hi - lo; };  // lo <= j < hi
    // A row that does not compete has key 0, as a NaN has.  Rows are counted from the highest key down and key 0 is the
    // last, so how many have it never matters.
    auto load = [&](uint32_t j) { return competes(j) ? __ldg(w + j) : __uint_as_float(0x7FC00000u); };
    uint32_t reg[REG ? SKEYS : 1];
    if (REG) {
#pragma unroll
        for (uint32_t i = 0; i < SKEYS; i += 4) {
            if (i >= nk)
                break;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                reg[REG ? i + e : 0] = __float_as_uint(load(j0 + (i + e) * 32));
        }
    }
    for (uint32_t i = tid; i < 3 * SBINS; i += nt)
        hist[i / SBINS][i % SBINS] = 0;
    // f(i, key) over this thread's rows j0 + 32 i, the whole warp in step
    auto each = [&](auto f) {
        if (REG) {
#pragma unroll
            for (uint32_t i = 0; i < SKEYS; i += 4) {
                if (i >= nk)
                    break;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    f(i + e, reg[REG ? i + e : 0]);
            }
        } else {
            for (uint32_t i = 0; i < nk; ++i) {
                uint32_t key = weight_key(load(j0 + i * 32));
                f(i, key);
            }
        }
    };
    // The bits in which the warp's keys differ from one another, and all that any of them has.
    uint32_t ones = 0, all_ones = 0xFFFFFFFFu;
    each([&](uint32_t, uint32_t& key) {
        if (REG)
            key = weight_key(__uint_as_float(key));
        ones |= key;
        all_ones &= key;
    });
    ones = __reduce_or_sync(0xffffffffu, ones);
    const uint32_t differ = ones & ~__reduce_and_sync(0xffffffffu, all_ones);
    __syncthreads();
    // T: the key of the last that stays, digit by digit; want: how many with key T stay.  No contest: no key is above T.
    uint32_t T = want > 0 ? 0u : 0xFFFFFFFFu;
    for (uint32_t pass = 0; want > 0 && pass < 3; ++pass) {
        const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        const uint32_t fixed = pass == 0 ? 0u : 0xFFFFFFFFu << (pass == 1 ? 21 : 10);  // the digits that are known
        uint32_t* const h = hist[pass];
        if ((differ >> shift) == 0) {  // one digit, and one answer whether it counts, for the whole warp
            if (lane == 0 && ones && ((ones ^ T) & fixed) == 0)
                atomicAdd(&h[ones >> shift & (bins - 1)], 32 * nk);
        } else if (pass == 0) {
            each([&](uint32_t, uint32_t& key) {
                if (key)
                    atomicAdd(&h[key >> 21], 1u);
            });
        } else {
            each([&](uint32_t, uint32_t& key) {
                if (((key ^ T) & fixed) == 0)
                    atomicAdd(&h[key >> shift & (bins - 1)], 1u);
            });
        }
        const uint32_t* all = h;
        if (C > 1) {
            cluster.sync();
            for (uint32_t i = tid; i < bins; i += nt) {
                uint32_t n = 0;
                for (uint32_t c = 0; c < C; ++c)
                    n += cluster.map_shared_rank(h, c)[i];
                sum[i] = n;
            }
            all = sum;
        }
        __syncthreads();
        // The digit at which the count from the top reaches want: 32 groups of bins are summed a warp a group (or
        // several), then one warp finds the group and the digit in it.
        const uint32_t per = bins / 32;  // 64 or 32 bins a group, group 0 the highest
        for (uint32_t g = warp; g < 32; g += warps) {
            const uint32_t top = bins - 1 - g * per - lane;
            const uint32_t n = __reduce_add_sync(0xffffffffu, all[top] + (per == 64 ? all[top - 32] : 0u));
            if (lane == 0)
                part[pass][g] = n;
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t n = part[pass][lane], above = warp_incl_scan(n) - n;
            const int g = 31 - __clz(__ballot_sync(0xffffffffu, above < want));  // the last group not past it
            above = __shfl_sync(0xffffffffu, above, g);
            uint32_t bin = bins - 1 - g * per - lane;
            n = all[bin];
            uint32_t before = above + warp_incl_scan(n) - n;
            const uint32_t last = __shfl_sync(0xffffffffu, before + n, 31);
            if (per == 64 && last < want) {
                bin -= 32;
                n = all[bin];
                before = last + warp_incl_scan(n) - n;
            }
            if (int(lane) == 31 - __clz(__ballot_sync(0xffffffffu, before < want))) {
                uint32_t t = T | bin << shift, left = want - before;
                if (t && n == left) {  // all with these digits stay, whatever the others are
                    t -= 1;
                    left = 0;
                }
                found[pass][0] = t;
                found[pass][1] = left;
            }
        }
        __syncthreads();
        T = found[pass][0];
        want = found[pass][1];
    }
    // Lane i takes the 32 rows of the warp's i-th keys from here on.  stay: those kept without the ties, tied: the ties
    const uint32_t mine0 = first + lane * 32;
    const uint32_t comp = lane < nk ? bits_within(mine0, lo, hi) : 0u, valid = lane < nk ? bits_within(mine0, 0, len) : 0u;
    uint32_t stay = 0, tied = 0, n_sure = 0, n_tie = 0;
    if (REG) {
        each([&](uint32_t i, uint32_t& key) {
            const uint32_t a = __ballot_sync(0xffffffffu, key > T);
            stay = lane == i ? a : stay;
        });
        stay |= valid & ~comp;
        if (want > 0) {
            each([&](uint32_t i, uint32_t& key) {
                const uint32_t a = __ballot_sync(0xffffffffu, key == T);
                tied = lane == i ? a : tied;
            });
            tied &= comp;
        }
        n_sure = __popc(stay);
        n_tie = __popc(tied);
    } else {
        each([&](uint32_t i, uint32_t& key) {
            const uint32_t j = j0 + i * 32;
            n_sure += key > T || (j < len && !competes(j)) ? 1u : 0u;
            n_tie += want > 0 && key == T && competes(j) ? 1u : 0u;
        });
    }
    n_sure = __reduce_add_sync(0xffffffffu, n_sure);
    n_tie = __reduce_add_sync(0xffffffffu, n_tie);
    if (lane == 0) {
        ranks[0][warp] = n_sure;
        ranks[1][warp] = n_tie;
    }
    __syncthreads();
    uint32_t at, ties;  // before this warp: kept rows without the ties, and ties
    {
        const uint32_t a = lane < warps ? ranks[0][lane] : 0u, t = lane < warps ? ranks[1][lane] : 0u;
        const uint32_t ai = warp_incl_scan(a), ti = warp_incl_scan(t);
        at = __shfl_sync(0xffffffffu, ai - a, warp);
        ties = __shfl_sync(0xffffffffu, ti - t, warp);
        if (tid == 31) {
            mine[0] = ai;
            mine[1] = ti;
        }
    }
    if (C > 1) {
        cluster.sync();
        for (uint32_t c = 0; c < rank; ++c) {
            at += cluster.map_shared_rank(mine, c)[0];
            ties += cluster.map_shared_rank(mine, c)[1];
        }
        cluster.sync();  // no CTA leaves while others read its counts
    }
    at += min(ties, want);
    if (n_sure == 0 && (n_tie == 0 || ties >= want))
        return;
    if (REG) {
        if (n_tie) {  // the same for the warp
            const uint32_t n = __popc(tied), t0 = ties + warp_incl_scan(n) - n;
            for (uint32_t room = t0 < want ? want - t0 : 0u, k = n; k > room; --k)
                tied &= ~(0x80000000u >> __clz(tied));  // the highest go
            stay |= tied;
        }
        const uint32_t n = __popc(stay);
        at += warp_incl_scan(n) - n;
        for (; stay; stay &= stay - 1)
            kept[at++] = int32_t(mine0 + __ffs(stay) - 1);
    } else {
        const uint32_t below = (1u << lane) - 1u;
        each([&](uint32_t i, uint32_t& key) {
            const uint32_t j = j0 + i * 32;
            const bool t = key == T && competes(j);
            const uint32_t ts = __ballot_sync(0xffffffffu, t);
            const bool stays = key > T || (j < len && !competes(j)) || (t && ties + __popc(ts & below) < want);
            const uint32_t st = __ballot_sync(0xffffffffu, stays);
            if (stays)
                kept[at + __popc(st & below)] = int32_t(j);
            at += __popc(st);
            ties += __popc(ts);
        });
    }
}

// Out of place: a CTA copies CROWS rows of one kv head, 16 bytes a thread at a time, CU rows' loads in flight.
constexpr uint32_t CROWS = 64, CU = 4;
template <uint32_t CH>  // 16-byte chunks a row
__global__ void __launch_bounds__(MNT) evict_copy_kernel(const EvictParams p)
{
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    constexpr uint32_t RPI = MNT / CH;  // rows the CTA takes at once
    const uint32_t kvh = blockIdx.y, b = blockIdx.z, n = uint32_t(p.count[b]);
    const uint64_t row = uint64_t(b) * p.kv_heads + kvh;
    if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0)
        p.new_len[b] = int32_t(n);
    const int32_t* const kept = p.kept + row * p.budget;
    const uint32_t r0 = blockIdx.x * CROWS, c = threadIdx.x % CH;
    const uint4* const k = static_cast<const uint4*>(p.k) + row * p.k_stride * CH + c;
    const uint4* const v = static_cast<const uint4*>(p.v) + row * p.k_stride * CH + c;
    uint4* const ko = static_cast<uint4*>(p.k_out) + row * p.out_stride * CH + c;
    uint4* const vo = static_cast<uint4*>(p.v_out) + row * p.out_stride * CH + c;
    if (r0 + threadIdx.x < n && threadIdx.x < CROWS)
        p.weight_out[row * p.out_stride + r0 + threadIdx.x] = p.weight[row * p.k_stride + kept[r0 + threadIdx.x]];
#pragma unroll
    for (uint32_t i = 0; i < CROWS; i += RPI * CU) {
        uint4 x[CU], y[CU];
#pragma unroll
        for (uint32_t u = 0; u < CU; ++u) {
            const uint32_t o = i + u * RPI + threadIdx.x / CH, r = r0 + o;
            if (o < CROWS && r < n) {
                const uint64_t src = uint64_t(kept[r]) * CH;
                x[u] = __ldcs(k + src);
                y[u] = __ldcs(v + src);
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < CU; ++u) {
            const uint32_t o = i + u * RPI + threadIdx.x / CH, r = r0 + o;
            if (o < CROWS && r < n) {
                ko[uint64_t(r) * CH] = x[u];
                vo[uint64_t(r) * CH] = y[u];
            }
        }
    }
}

// In place: blockIdx.x < 2 * slices takes a 64-byte slice of k's or v's rows, the last one the weights.
template <typename E>
__device__ __forceinline__ void move_in_place(E* base, uint64_t pitch, const int32_t* kept, uint32_t n, uint32_t per_row)
{
    constexpr int U = 4;
    const uint32_t step = MNT / per_row * U, r = threadIdx.x / per_row, c = threadIdx.x % per_row;
    for (uint32_t r0 = 0; r0 < n; r0 += step) {
        E x[U];
        bool moves[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = r0 + u * (MNT / per_row) + r;
            const uint32_t src = i < n ? uint32_t(kept[i]) : i;
            moves[u] = src != i;
            if (moves[u])
                x[u] = base[src * pitch + c];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (moves[u])
                base[uint64_t(r0 + u * (MNT / per_row) + r) * pitch + c] = x[u];
    }
}

__global__ void __launch_bounds__(MNT) evict_in_place_kernel(const EvictParams p)
{
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const uint32_t kvh = blockIdx.y, b = blockIdx.z, n = uint32_t(p.count[b]);
    const uint64_t row = uint64_t(b) * p.kv_heads + kvh;
    if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0)
        p.new_len[b] = int32_t(n);
    const int32_t* const kept = p.kept + row * p.budget;
    const uint32_t slices = p.dim / 32, x = blockIdx.x, ch = p.dim / 8;
    if (x < 2 * slices) {
        uint4* const base = static_cast<uint4*>(x < slices ? p.k_out : p.v_out) + row * p.out_stride * ch;
        move_in_place(base + x % slices * 4, ch, kept, n, 4);
    } else {
        move_in_place(p.weight_out + row * p.out_stride, 1, kept, n, 1);
    }
}

} // namespace

cudaError_t launch_cache_evict(const EvictParams& p, cudaStream_t st)
{
    // CTAs a row: as few as hold its keys in registers, 8 at most (see above for what a cluster costs).  Rows of up to
    // 16 keys a thread of 256 take a small CTA, whose barriers are cheaper.
    uint32_t c = 1;
    while (c < SMAX_CLUSTER && uint64_t(c) * SNT * SKEYS < p.max_len)
        c *= 2;
    const uint32_t nt = p.max_len <= 256 * 16 ? 256 : SNT;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c, p.kv_heads, p.batch);
    cfg.blockDim = dim3(nt);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = c;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = uint64_t(c) * SNT * SKEYS >= p.max_len ? cudaLaunchKernelEx(&cfg, evict_select_kernel<true>, p)
                                                           : cudaLaunchKernelEx(&cfg, evict_select_kernel<false>, p);
    if (e != cudaSuccess)
        return e;
    // the copy as a programmatic dependent: scheduled while the selection runs out
    cfg.blockDim = dim3(MNT);
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    if (p.in_place) {
        cfg.gridDim = dim3(2 * (p.dim / 32) + 1, p.kv_heads, p.batch);
        return cudaLaunchKernelEx(&cfg, evict_in_place_kernel, p);
    }
    cfg.gridDim = dim3((p.budget + CROWS - 1) / CROWS, p.kv_heads, p.batch);
    return p.dim == 64    ? cudaLaunchKernelEx(&cfg, evict_copy_kernel<8>, p)
           : p.dim == 128 ? cudaLaunchKernelEx(&cfg, evict_copy_kernel<16>, p)
                          : cudaLaunchKernelEx(&cfg, evict_copy_kernel<32>, p);
}

} // namespace mako
