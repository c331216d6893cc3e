// Eviction from a KV cache by accumulated attention weight (mako_cache_evict).  No counterpart in the reference.
//
// evict_select_kernel: one CTA a (sequence, kv head).  The rows between the sinks and the recent ones compete; the
// weight of the last that stays is found by a radix select over the weights as order-preserving integers, eight bits a
// pass (a histogram in shared memory, integer counts, so the result does not depend on the order of the adds); then
// one ordered pass writes the kept rows' indices, ties taken from the lowest row on.
// evict_move_kernel: copies the kept rows.  In place, row i comes from row kept[i] >= i: a CTA owns a 64-byte column
// slice of every row and walks the rows upwards in steps, reading a whole step before it writes it, so what a later step
// reads (rows at or past its own first) has not been written yet.
#include "common.cuh"
#include "kernels.h"

namespace mako {
namespace {

constexpr uint32_t SNT = 1024, MNT = 256;

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

// Exclusive prefix sum of x over the CTA's SNT threads, and the total.  part: 33 words of shared memory.
__device__ __forceinline__ uint32_t block_excl_scan(uint32_t x, uint32_t* part, uint32_t& total)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t incl = warp_incl_scan(x);
    __syncthreads();
    if (lane == 31)
        part[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const uint32_t y = part[lane], z = warp_incl_scan(y);
        part[lane] = z - y;
        if (lane == 31)
            part[32] = z;
    }
    __syncthreads();
    total = part[32];
    return part[warp] + incl - x;
}

__global__ void __launch_bounds__(SNT) evict_select_kernel(const EvictParams p)
{
    __shared__ uint32_t hist[256], part[33], found[2];
    const uint32_t kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int32_t l = p.kv_len[b];
    const uint32_t len = l > 0 ? min(uint32_t(l), p.max_len) : 0u, keep = min(len, p.budget);
    const uint64_t row = uint64_t(b) * p.kv_heads + kvh;
    int32_t* const kept = p.kept + row * p.budget;
    if (kvh == 0 && tid == 0)
        p.count[b] = int32_t(keep);
    for (uint32_t i = keep + tid; i < p.budget; i += SNT)
        kept[i] = -1;
    if (len <= p.budget) {
        for (uint32_t i = tid; i < len; i += SNT)
            kept[i] = int32_t(i);
        return;
    }
    const float* const w = p.weight + row * p.k_stride;
    const uint32_t lo = p.sinks, hi = len - p.recent;  // the rows that compete
    uint32_t want = p.budget - p.sinks - p.recent;     // how many of them stay
    // T: the key of the last that stays, digit by digit; want: how many with key T stay
    uint32_t T = 0;
    if (want) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256; i += SNT)
                hist[i] = 0;
            __syncthreads();
            for (uint32_t j = lo + tid; j < hi; j += SNT) {
                const uint32_t key = weight_key(w[j]);
                if (shift == 24 || key >> (shift + 8) == T >> (shift + 8))
                    atomicAdd(&hist[key >> shift & 255u], 1u);
            }
            __syncthreads();
            // the digit at which the count from the top reaches want
            const uint32_t mine = tid < 256 ? hist[255 - tid] : 0u;
            uint32_t total;
            const uint32_t above = block_excl_scan(mine, part, total);
            if (tid < 256 && above < want && above + mine >= want) {
                found[0] = 255 - tid;
                found[1] = want - above;
            }
            __syncthreads();
            T |= found[0] << shift;
            want = found[1];
            __syncthreads();
        }
    }
    uint32_t out = 0, ties = 0;  // kept and tied rows before this step
    const bool none = p.budget == p.sinks + p.recent;
    for (uint32_t j0 = 0; j0 < len; j0 += SNT) {
        const uint32_t j = j0 + tid;
        const bool forced = j < len && (j < lo || j >= hi);
        const uint32_t key = j >= lo && j < hi && !none ? weight_key(w[j]) : 0u;
        const bool compete = j >= lo && j < hi && !none;
        const bool tie = compete && key == T;
        uint32_t nt, nk;
        const uint32_t rank = block_excl_scan(tie, part, nt);
        const bool stay = forced || (compete && key > T) || (tie && ties + rank < want);
        const uint32_t at = block_excl_scan(stay, part, nk);
        if (stay)
            kept[out + at] = int32_t(j);
        out += nk;
        ties += nt;
    }
}

// Out of place: a CTA copies `step` rows of one kv head; 16 bytes a thread at a time.
__global__ void __launch_bounds__(MNT) evict_copy_kernel(const EvictParams p, uint32_t step)
{
    const uint32_t kvh = blockIdx.y, b = blockIdx.z, n = uint32_t(p.count[b]);
    const uint64_t row = uint64_t(b) * p.kv_heads + kvh;
    if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0)
        p.new_len[b] = int32_t(n);
    const int32_t* const kept = p.kept + row * p.budget;
    const uint32_t r0 = blockIdx.x * step, r1 = min(n, r0 + step), ch = p.dim / 8;
    const uint4* const k = static_cast<const uint4*>(p.k) + row * p.k_stride * ch;
    const uint4* const v = static_cast<const uint4*>(p.v) + row * p.k_stride * ch;
    uint4* const ko = static_cast<uint4*>(p.k_out) + row * p.out_stride * ch;
    uint4* const vo = static_cast<uint4*>(p.v_out) + row * p.out_stride * ch;
    for (uint32_t i = r0 * ch + threadIdx.x; i < r1 * ch; i += MNT) {
        const uint32_t r = i / ch, c = i % ch;
        const uint64_t src = uint64_t(kept[r]) * ch + c, dst = uint64_t(r) * ch + c;
        const uint4 a = __ldcs(k + src), e = __ldcs(v + src);
        ko[dst] = a;
        vo[dst] = e;
    }
    for (uint32_t r = r0 + threadIdx.x; r < r1; r += MNT)
        p.weight_out[row * p.out_stride + r] = p.weight[row * p.k_stride + kept[r]];
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
    evict_select_kernel<<<dim3(p.kv_heads, p.batch), SNT, 0, st>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
        return e;
    if (p.in_place) {
        evict_in_place_kernel<<<dim3(2 * (p.dim / 32) + 1, p.kv_heads, p.batch), MNT, 0, st>>>(p);
    } else {
        const uint32_t step = 64;
        evict_copy_kernel<<<dim3((p.budget + step - 1) / step, p.kv_heads, p.batch), MNT, 0, st>>>(p, step);
    }
    return cudaGetLastError();
}

} // namespace mako
