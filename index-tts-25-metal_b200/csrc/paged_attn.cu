// Causal attention of a step's fresh rows over a paged K/V cache
// (itts_paged_attention).
//
// One warp per (row, query head): the lanes share the head's dimensions, the
// keys are visited one after the other with the running maximum and sum of the
// softmax in registers, and each table entry is checked before it is followed.
// The sums of every kChunk keys are folded into the totals, so that the fp32
// rounding grows with the chunks and not with the keys.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.hpp"

namespace itts {
namespace paged {
namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kChunk = 64;

template <class T, int D>
__global__ void __launch_bounds__(128) k_attn_rows(itts_paged_attention_args a) {
    const int lane = threadIdx.x & 31, h = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (h >= a.q_heads) return;
    const int kvh = h / (a.q_heads / a.cache.heads), shift = 31 - __clz(a.cache.block_size);
    const auto start = [&](int r) { return min(max(__ldg(a.q_start + r), 0), a.rows); };
    const int t = blockIdx.x;
    // the request of row t: the last one that starts at or before it
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start(mid) <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int first = start(lo), end = start(lo + 1);
    if (t < first || t >= end) return;
    const int pos = __ldg(a.lens + lo) - end + t;
    const long long keys = min((long long)pos + 1, (long long)a.max_blocks << shift);
    constexpr int E = D / 32;
    float q[E], o[E], m = -INFINITY, l = 0.f, ot[E], mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = to_float(static_cast<const T*>(a.q)[t * a.q_row_stride + h * a.q_head_stride + lane * E + e]) * a.scale;
        o[e] = ot[e] = 0.f;
    }
    const auto fold = [&] {  // (m, l, o) into (mt, lt, ot), and start afresh
        const float mn = fmaxf(mt, m), c = mt == -INFINITY ? 0.f : expf(mt - mn), f = m == -INFINITY ? 0.f : expf(m - mn);
        lt = lt * c + l * f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            ot[e] = ot[e] * c + o[e] * f;
            o[e] = 0.f;
        }
        mt = mn;
        m = -INFINITY;
        l = 0.f;
    };
    for (long long j = 0; j < keys; ++j) {
        if (j % kChunk == kChunk - 1) fold();
        const int id = __ldg(a.table + (long long)lo * a.table_stride + (j >> shift));
        if ((unsigned)id >= (unsigned)a.cache.blocks) continue;
        const long long tok = j & (a.cache.block_size - 1);
        const T* k = static_cast<const T*>(a.cache.k) + id * a.cache.k_block_stride + tok * a.cache.k_token_stride +
                     kvh * a.cache.k_head_stride + lane * E;
        const T* v = static_cast<const T*>(a.cache.v) + id * a.cache.v_block_stride + tok * a.cache.v_token_stride +
                     kvh * a.cache.v_head_stride + lane * E;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], to_float(k[e]), s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
        l = l * c + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * to_float(v[e]);
        m = mn;
    }
    fold();
#pragma unroll
    for (int e = 0; e < E; ++e)
        put(static_cast<T*>(a.out) + t * a.out_row_stride + h * a.out_head_stride + lane * E + e,
            lt == 0.f ? 0.f : ot[e] / lt);
}

template <class T>
cudaError_t launch_rows(const itts_paged_attention_args& a, cudaStream_t s) {
    const dim3 grid(a.rows, (a.q_heads + 3) / 4);
    if (a.cache.head_dim == 64)
        k_attn_rows<T, 64><<<grid, 128, 0, s>>>(a);
    else
        k_attn_rows<T, 128><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t attention_workspace(int) { return 256; }

cudaError_t launch_attention(const itts_paged_attention_args& a, cudaStream_t s) {
    switch (a.cache.type) {
        case ITTS_PAGED_F16: return launch_rows<__half>(a, s);
        case ITTS_PAGED_BF16: return launch_rows<__nv_bfloat16>(a, s);
        default: return launch_rows<float>(a, s);
    }
}

}  // namespace paged
}  // namespace itts
