// Appending projected tokens to a KV cache (mako_cache_append): fp32 projection rows -> RMS norm of q and k per head,
// rotary positions, 16-bit q rows and cache rows.  No counterpart in the reference (its producers write head tiles of
// one sequence with angles from a table: src/models/runtime.cpp:215-260).
//
// HBM-bound: 4 bytes read and 2 written a value.  One CTA a token, so that the token's angles are made once for all its
// heads: thread i makes pair i's while the heads' loads are in flight.  The angle pos * freq is taken in turns in
// double precision and reduced to [-1/2, 1/2] there -- in fp32 a position of 10^6 would leave 0.06 radians of error --
// and only the reduced turn goes through fp32 sincospi.  A warp takes up to HPW heads at a time, all their loads in
// flight together (8 of 128 values: 108 us for 2 x 8192 tokens of 32 / 8 heads, 0.85 of the copy rate; 4: 122, 2: 211),
// lane l holding values 4 l .. 4 l + 3 of every 128, so that a half rotation's partner is the same value of another
// lane (through shared memory, with its bank conflicts, the same took 182 us).
#include "common.cuh"
#include "kernels.h"

namespace mako {
namespace {

constexpr uint32_t kMaxWarps = 16;

template <typename T>
__device__ __forceinline__ void store_vals(T* dst, const float* v, int n)
{
    if (n == 4) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]));
    } else {
        *reinterpret_cast<uint32_t*>(dst) = Elem<T>::pack(v[0], v[1]);
    }
}

// D: head width; VB consecutive values of a lane (2 for 64-wide heads, else 4) in NB blocks of 32 * VB.
template <int D, typename T>
__global__ void cache_append_kernel(const AppendParams p)
{
    constexpr int VB = D == 64 ? 2 : 4, NB = D / (32 * VB), VPL = VB * NB, HPW = D == 256 ? 4 : 8;
    __shared__ float2 cs[D / 2];
    extern __shared__ float row_buf[];  // [warps][D]: a head's values where rotation partners cross lanes
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const uint32_t tok = blockIdx.x, b = tok / p.n_tok, i = tok % p.n_tok;
    if (p.n_new && int32_t(i) >= p.n_new[b])
        return;
    const int32_t len = p.kv_len[b];
    const uint64_t row = uint64_t(len > 0 ? len : 0) + i;
    const float* const x = p.x + uint64_t(tok) * p.ld;
    const uint32_t gq = (p.heads + HPW - 1) / HPW, gk = (p.kv_heads + HPW - 1) / HPW, groups = gq + 2 * gk;
    const uint32_t half = p.rot / 2;
    float* const buf = row_buf + warp * D;
    bool angles = false;
    // uniform trip count: the barrier below is reached by every warp in its first round
    for (uint32_t g0 = 0; g0 < groups; g0 += warps) {
        const uint32_t g = g0 + warp;
        const bool live = g < groups;
        // kind 0 q, 1 k, 2 v; the group's first head and its count
        const uint32_t kind = g < gq ? 0 : g < gq + gk ? 1 : 2;
        const uint32_t h0 = (kind == 0 ? g : kind == 1 ? g - gq : g - gq - gk) * HPW;
        const uint32_t nh = !live ? 0 : min(uint32_t(HPW), (kind == 0 ? p.heads : p.kv_heads) - h0);
        const uint32_t step = kind == 0 ? p.q_stride : D;
        const float* const src = x + (kind == 0 ? p.q_col0 : kind == 1 ? p.k_col0 : p.v_col0) + uint64_t(h0) * step;
        float v[HPW][VPL];
#pragma unroll
        for (int j = 0; j < HPW; ++j)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const float* const s = src + uint64_t(j) * step + n * 32 * VB + lane * VB;
                if (uint32_t(j) >= nh) {
#pragma unroll
                    for (int e = 0; e < VB; ++e)
                        v[j][n * VB + e] = 0.0f;
                } else if (VB == 4 && p.vec4) {
                    const float4 w = __ldcs(reinterpret_cast<const float4*>(s));
                    v[j][n * VB] = w.x;
                    v[j][n * VB + 1] = w.y;
                    v[j][n * VB + VB - 2] = w.z;
                    v[j][n * VB + VB - 1] = w.w;
                } else if (VB == 2 && p.vec4) {
                    const float2 w = __ldcs(reinterpret_cast<const float2*>(s));
                    v[j][n * VB] = w.x;
                    v[j][n * VB + 1] = w.y;
                } else {
#pragma unroll
                    for (int e = 0; e < VB; ++e)
                        v[j][n * VB + e] = __ldcs(s + e);
                }
            }
        if (!angles) {
            if (half) {
                const double at = double(p.pos ? int64_t(p.pos[tok]) : int64_t(row));
                for (uint32_t t = threadIdx.x; t < half; t += blockDim.x) {
                    const double turns = at * (p.freq[t] * 0.15915494309189533577);  // 1 / (2 pi)
                    float s, c;
                    sincospif(2.0f * float(turns - rint(turns)), &s, &c);
                    cs[t] = make_float2(c * p.amplitude, s * p.amplitude);
                }
            }
            __syncthreads();
            angles = true;
        }
        if (!live)
            continue;
        const float* const w = kind == 0 ? p.wq : kind == 1 ? p.wk : nullptr;
        if (w) {
            float ss[HPW];
#pragma unroll
            for (int j = 0; j < HPW; ++j) {
                ss[j] = 0.0f;
#pragma unroll
                for (int e = 0; e < VPL; ++e)
                    ss[j] = fmaf(v[j][e], v[j][e], ss[j]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int j = 0; j < HPW; ++j)
                    ss[j] += __shfl_xor_sync(0xffffffffu, ss[j], o);
            float wv[VPL];
#pragma unroll
            for (int e = 0; e < VPL; ++e)
                wv[e] = __ldg(w + (e / VB) * 32 * VB + lane * VB + e % VB);
#pragma unroll
            for (int j = 0; j < HPW; ++j) {
                const float inv = rsqrtf(ss[j] / float(D) + p.eps);
#pragma unroll
                for (int e = 0; e < VPL; ++e)
                    v[j][e] *= inv * wv[e];
            }
        }
        if (kind < 2 && half) {
            if (p.layout == 2) {  // adjacent pairs: both in this lane
#pragma unroll
                for (int e = 0; e < VPL; e += 2) {
                    const uint32_t d = (e / VB) * 32 * VB + lane * VB + e % VB;
                    if (d < p.rot) {
                        const float2 a = cs[d / 2];
#pragma unroll
                        for (int j = 0; j < HPW; ++j) {
                            const float u0 = v[j][e], u1 = v[j][e + 1];
                            v[j][e] = fmaf(u0, a.x, -u1 * a.y);
                            v[j][e + 1] = fmaf(u1, a.x, u0 * a.y);
                        }
                    }
                }
            } else if (half % VB == 0) {
                // halves a whole number of chunks (VB values) apart: the partner of this lane's chunk is a chunk of
                // another lane, or of the other block
                const uint32_t hc = half / VB;
                uint32_t from[NB];
                float cc[VPL], sn[VPL];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint32_t c = n * 32 + lane;
                    const bool first = c < hc;
                    from[n] = first ? c + hc : c < 2 * hc ? c - hc : c;
#pragma unroll
                    for (int e = 0; e < VB; ++e) {
                        const float2 a = c < 2 * hc ? cs[(first ? c : c - hc) * VB + e] : make_float2(1.0f, 0.0f);
                        cc[n * VB + e] = a.x;
                        sn[n * VB + e] = first ? -a.y : a.y;
                    }
                }
#pragma unroll
                for (int j = 0; j < HPW; ++j) {
                    float u[VPL];
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int e = 0; e < VB; ++e) {
                            const float u0 = __shfl_sync(0xffffffffu, v[j][e], from[n] % 32);
                            const float u1 = NB == 2 ? __shfl_sync(0xffffffffu, v[j][VPL - VB + e], from[n] % 32) : u0;
                            u[n * VB + e] = from[n] < 32 ? u0 : u1;
                        }
#pragma unroll
                    for (int e = 0; e < VPL; ++e)
                        if ((e / VB) * 32 + lane < 2 * hc)
                            v[j][e] = fmaf(v[j][e], cc[e], u[e] * sn[e]);
                }
            } else {  // other halves: through the warp's copy of the head
#pragma unroll
                for (int j = 0; j < HPW; ++j) {
                    if (uint32_t(j) >= nh)
                        break;
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < VPL; ++e)
                        buf[(e / VB) * 32 * VB + lane * VB + e % VB] = v[j][e];
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < VPL; ++e) {
                        const uint32_t d = (e / VB) * 32 * VB + lane * VB + e % VB;
                        if (d < p.rot) {
                            const bool first = d < half;
                            const float2 a = cs[first ? d : d - half];
                            const float u = buf[first ? d + half : d - half];
                            v[j][e] = fmaf(v[j][e], a.x, first ? -u * a.y : u * a.y);
                        }
                    }
                }
            }
        }
        if (kind && row >= p.k_stride)
            continue;
        if (kind == 1 && p.weight && lane < nh)  // a token begins without the weight of the one whose row it takes
            p.weight[(uint64_t(b) * p.kv_heads + h0 + lane) * p.k_stride + row] = 0.0f;
        T* dst;
        uint64_t dstep;
        if (kind == 0) {
            dst = static_cast<T*>(p.q) + (uint64_t(tok) * p.heads + h0) * D;
            dstep = D;
        } else {
            dstep = uint64_t(p.k_stride) * D;
            dst = static_cast<T*>(kind == 1 ? p.k : p.v) + (uint64_t(b) * p.kv_heads + h0) * dstep + row * D;
        }
#pragma unroll
        for (int j = 0; j < HPW; ++j)
            if (uint32_t(j) < nh)
#pragma unroll
                for (int n = 0; n < NB; ++n)
                    store_vals<T>(dst + j * dstep + n * 32 * VB + lane * VB, &v[j][n * VB], VB);
    }
}

template <int D, typename T>
cudaError_t launch_append_t(const AppendParams& p, cudaStream_t st)
{
    constexpr uint32_t HPW = D == 256 ? 4 : 8;
    const uint32_t groups = (p.heads + HPW - 1) / HPW + 2 * ((p.kv_heads + HPW - 1) / HPW);
    const uint32_t warps = groups < kMaxWarps ? groups : kMaxWarps;
    cache_append_kernel<D, T><<<p.batch * p.n_tok, warps * 32, warps * D * sizeof(float), st>>>(p);
    return cudaGetLastError();
}

} // namespace

cudaError_t launch_cache_append(const AppendParams& p, int dtype, int dim, cudaStream_t st)
{
    const bool bf = dtype == kBF16;
    switch (dim) {
    case 64:
        return bf ? launch_append_t<64, __nv_bfloat16>(p, st) : launch_append_t<64, __half>(p, st);
    case 128:
        return bf ? launch_append_t<128, __nv_bfloat16>(p, st) : launch_append_t<128, __half>(p, st);
    case 256:
        return bf ? launch_append_t<256, __nv_bfloat16>(p, st) : launch_append_t<256, __half>(p, st);
    default:
        return cudaErrorInvalidValue;
    }
}

} // namespace mako
