// Eviction from a KV cache by accumulated attention weight (mako_cache_evict).  No counterpart in the reference.
//
// evict_select_kernel: a cluster of 1 to 8 CTAs a (sequence, kv head), its weights held in registers as
// order-preserving integers (SKEYS a thread; longer rows are read again by every pass).  The rows between the sinks and
// the recent ones compete; the weight of the last that stays is found by a radix select of 11, 11 and 10 bits: a
// histogram in shared memory, merged over the cluster.  Equal digits in a warp are added once, so that rows of equal
// weights do not queue at one counter.  All counts are integers: the result does not depend on the order of the adds.
// Then every warp, which owns consecutive rows, writes its kept rows' indices from the count of those before it, ties
// taken from the lowest row on.
// evict_copy_kernel and evict_in_place_kernel copy the kept rows.  In place, row i comes from row kept[i] >= i: a CTA owns a 64-byte column
// slice of every row and walks the rows upwards in steps, reading a whole step before it writes it, so what a later step
// reads (rows at or past its own first) has not been written yet.
#include "common.cuh"
#include "kernels.h"

#include <cooperative_groups.h>

namespace mako {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t SNT = 1024, SKEYS = 32, SBINS = 2048, MNT = 256;
constexpr uint32_t SWARPS = SNT / 32, SMAX_CLUSTER = 8;

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

// Adds one to hist[bin] for every lane that counts: once for all lanes with the first one's bin, then one by one.
__device__ __forceinline__ void count_bin(uint32_t* hist, uint32_t bin, bool counts)
{
    const uint32_t lane = threadIdx.x & 31, who = __ballot_sync(0xffffffffu, counts);
    if (!who)
        return;
    const int first = __ffs(who) - 1;
    const uint32_t lead = __shfl_sync(0xffffffffu, bin, first);  // by every lane, whether it counts or not
    const bool same = counts && bin == lead;
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, same));
    if (int(lane) == first)
        atomicAdd(&hist[bin], n);
    else if (counts && !same)
        atomicAdd(&hist[bin], 1u);
}

// REG: a thread's keys fit its SKEYS registers.
template <bool REG>
__global__ void __launch_bounds__(SNT) evict_select_kernel(const EvictParams p)
{
    __shared__ uint32_t hist[SBINS], sum[SBINS], part[SWARPS], found[2], mine[2], ranks[2][SWARPS];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t l = p.kv_len[b];
    const uint32_t len = l > 0 ? min(uint32_t(l), p.max_len) : 0u, keep = min(len, p.budget);
    const uint64_t row = uint64_t(b) * p.kv_heads + kvh;
    int32_t* const kept = p.kept + row * p.budget;
    if (kvh == 0 && rank == 0 && tid == 0)
        p.count[b] = int32_t(keep);
    for (uint32_t i = keep + rank * SNT + tid; i < p.budget; i += C * SNT)
        kept[i] = -1;
    if (len <= p.budget) {  // the same for the whole cluster
        for (uint32_t i = rank * SNT + tid; i < len; i += C * SNT)
            kept[i] = int32_t(i);
        return;
    }
    const float* const w = p.weight + row * p.k_stride;
    const uint32_t lo = p.sinks, hi = len - p.recent;  // the rows that compete
    uint32_t want = p.budget - p.sinks - p.recent;     // how many of them stay
    const bool contest = want > 0;
    // warp g of the cluster owns rows [g * 32 * nk, (g + 1) * 32 * nk), lane i's every 32nd
    const uint32_t nk = (len + C * SNT - 1) / (C * SNT), j0 = (rank * SWARPS + warp) * 32 * nk + lane;
    uint32_t reg[REG ? SKEYS : 1];
    if (REG) {
#pragma unroll
        for (uint32_t i = 0; i < SKEYS; ++i)
            if (i < nk)
                reg[i] = j0 + i * 32 < len ? __float_as_uint(__ldg(w + j0 + i * 32)) : 0u;
#pragma unroll
        for (uint32_t i = 0; i < SKEYS; ++i)
            if (i < nk)
                reg[i] = weight_key(__uint_as_float(reg[i]));
    }
    // f(row, key) over this thread's rows, the whole warp in step
    auto each = [&](auto f) {
        if (REG) {
#pragma unroll
            for (uint32_t i = 0; i < SKEYS; ++i)
                if (i < nk)
                    f(j0 + i * 32, reg[REG ? i : 0]);
        } else {
            for (uint32_t i = 0; i < nk; ++i)
                f(j0 + i * 32, j0 + i * 32 < len ? weight_key(__ldg(w + j0 + i * 32)) : 0u);
        }
    };
    // T: the key of the last that stays, digit by digit; want: how many with key T stay
    uint32_t T = 0;
    for (uint32_t pass = 0; contest && pass < 3; ++pass) {
        const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (uint32_t i = tid; i < SBINS; i += SNT)
            hist[i] = 0;
        __syncthreads();
        each([&](uint32_t j, uint32_t key) {
            const bool counts = j >= lo && j < hi && (pass == 0 || key >> (shift + (pass == 1 ? 11 : 10)) == T >> (shift + (pass == 1 ? 11 : 10)));
            count_bin(hist, key >> shift & (bins - 1), counts);
        });
        const uint32_t* all = hist;
        if (C > 1) {
            cluster.sync();
            for (uint32_t i = tid; i < bins; i += SNT) {
                uint32_t n = 0;
                for (uint32_t c = 0; c < C; ++c)
                    n += cluster.map_shared_rank(hist, c)[i];
                sum[i] = n;
            }
            cluster.sync();  // no histogram is cleared before all have read it
            all = sum;
        } else {
            __syncthreads();
        }
        // the digit at which the count from the top reaches want: thread t looks at the bins - 1 - 2t th and the next
        const uint32_t b0 = bins - 1 - 2 * tid, n0 = 2 * tid < bins ? all[b0] : 0u, n1 = 2 * tid < bins ? all[b0 - 1] : 0u;
        const uint32_t incl = warp_incl_scan(n0 + n1);
        if (lane == 31)
            part[warp] = incl;
        __syncthreads();
        uint32_t above = incl - n0 - n1;
        {
            const uint32_t y = part[lane], z = warp_incl_scan(y) - y;
            above += __shfl_sync(0xffffffffu, z, warp);
        }
        if (above < want && above + n0 + n1 >= want) {
            const bool second = above + n0 < want;
            found[0] = second ? b0 - 1 : b0;
            found[1] = want - above - (second ? n0 : 0u);
        }
        __syncthreads();
        T |= found[0] << shift;
        want = found[1];
    }
    // kept rows without the ties, and ties, of this warp; then of those before it
    uint32_t nk_sure = 0, n_tie = 0;
    auto sure = [&](uint32_t j, uint32_t key) { return j < len && (j < lo || j >= hi || (contest && key > T)); };
    auto tie = [&](uint32_t j, uint32_t key) { return contest && j >= lo && j < hi && key == T; };
    each([&](uint32_t j, uint32_t key) {
        nk_sure += __popc(__ballot_sync(0xffffffffu, sure(j, key)));
        n_tie += __popc(__ballot_sync(0xffffffffu, tie(j, key)));
    });
    if (lane == 0) {
        ranks[0][warp] = nk_sure;
        ranks[1][warp] = n_tie;
    }
    __syncthreads();
    uint32_t at, ties;  // before this warp: kept rows without the ties, and ties
    {
        const uint32_t a = ranks[0][lane], t = ranks[1][lane];
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
    const uint32_t below = (1u << lane) - 1u;
    each([&](uint32_t j, uint32_t key) {
        const bool t = tie(j, key);
        const uint32_t tied = __ballot_sync(0xffffffffu, t);
        const bool stays = sure(j, key) || (t && ties + __popc(tied & below) < want);
        const uint32_t stay = __ballot_sync(0xffffffffu, stays);
        if (stays)
            kept[at + __popc(stay & below)] = int32_t(j);
        at += __popc(stay);
        ties += __popc(tied);
    });
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
    // CTAs a row: enough that a thread's keys fit its registers (8 at most), and more, down to 8 keys a thread, while
    // that leaves SMs idle.
    const uint64_t rows = uint64_t(p.batch) * p.kv_heads;
    uint32_t c = 1;
    while (c < SMAX_CLUSTER && (uint64_t(c) * SNT * SKEYS < p.max_len ||
                                (uint64_t(c) * SNT * 8 < p.max_len && 2 * c * rows <= p.num_sms)))
        c *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c, p.kv_heads, p.batch);
    cfg.blockDim = dim3(SNT);
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
