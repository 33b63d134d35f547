// Append of a step's key and value rows to a paged K/V cache
// (itts_paged_append): a scatter of rows by slot with an optional rounding to
// the cache's type.
//
// Bound by memory: every source element is read once and every destination
// element written once.  A thread moves one 16-byte piece of a key row and the
// same piece of the value row (two independent loads in flight), consecutive
// threads consecutive pieces of a row, so loads and stores are whole sectors
// in every layout.  Rows whose addresses or strides are not multiples of 16
// bytes (of 8 source elements for a rounding append) go element by element.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "paged.hpp"

namespace itts {
namespace paged {
namespace {

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// kVec consecutive elements.
template <class S, class T, int kVec>
struct Piece {
    S x[kVec];
    __device__ __forceinline__ void load(const S* p) {
        if constexpr (kVec == 1) {
            x[0] = *p;
        } else {
            constexpr int kWords = kVec * int(sizeof(S)) / 16;
            uint4 w[kWords];
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
            memcpy(x, w, sizeof x);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        T y[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            if constexpr (sizeof(S) == sizeof(T))
                y[i] = x[i];
            else
                y[i] = from_float<T>(x[i]);
        }
        if constexpr (kVec == 1) {
            *p = y[0];
        } else {
            static_assert(kVec * sizeof(T) == 16, "one 16-byte store");
            uint4 w;
            memcpy(&w, y, 16);
            *reinterpret_cast<uint4*>(p) = w;
        }
    }
};

template <class S, class T, int kVec>
__global__ void __launch_bounds__(256) k_append(itts_paged_append_args a) {
    const int per_head = a.cache.head_dim / kVec, per_row = per_head * a.cache.heads;
    const int shift = 31 - __clz(a.cache.block_size);
    const unsigned slots = unsigned(a.cache.blocks) << shift;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < (long long)a.rows * per_row; i += 256ll * gridDim.x) {
        const int row = int(i / per_row), piece = int(i - (long long)row * per_row);
        const int h = piece / per_head, d = (piece - h * per_head) * kVec;
        const unsigned slot = unsigned(__ldg(a.slots + row));
        if (slot >= slots) continue;
        Piece<S, T, kVec> k, v;
        k.load(static_cast<const S*>(a.k) + row * a.k_row_stride + h * a.k_head_stride + d);
        v.load(static_cast<const S*>(a.v) + row * a.v_row_stride + h * a.v_head_stride + d);
        const long long block = slot >> shift, token = slot & (a.cache.block_size - 1);
        k.store(static_cast<T*>(a.cache.k) + block * a.cache.k_block_stride + token * a.cache.k_token_stride +
                h * a.cache.k_head_stride + d);
        v.store(static_cast<T*>(a.cache.v) + block * a.cache.v_block_stride + token * a.cache.v_token_stride +
                h * a.cache.v_head_stride + d);
    }
}

template <class S, class T>
cudaError_t launch(const itts_paged_append_args& a, cudaStream_t s) {
    constexpr int kVec = 16 / int(sizeof(T));
    const auto whole = [](long long stride) { return stride * (long long)sizeof(S) % 16 == 0; };
    const bool wide = reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.v) % 16 == 0 &&
                      whole(a.k_row_stride) && whole(a.k_head_stride) && whole(a.v_row_stride) &&
                      whole(a.v_head_stride);
    const long long pieces = (long long)a.rows * a.cache.heads * (a.cache.head_dim / (wide ? kVec : 1));
    const unsigned grid = unsigned(min((pieces + 255) / 256, 1ll << 30));
    if (wide)
        k_append<S, T, kVec><<<grid, 256, 0, s>>>(a);
    else
        k_append<S, T, 1><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append(const itts_paged_append_args& a, cudaStream_t s) {
    const bool same = a.source_type == a.cache.type;
    switch (a.cache.type) {
        case ITTS_PAGED_F16: return same ? launch<__half, __half>(a, s) : launch<float, __half>(a, s);
        case ITTS_PAGED_BF16:
            return same ? launch<__nv_bfloat16, __nv_bfloat16>(a, s) : launch<float, __nv_bfloat16>(a, s);
        default: return launch<float, float>(a, s);
    }
}

}  // namespace paged
}  // namespace itts
