// Paged attention of few rows per request: single tokens, short drafts.
//
// Bound by the bytes of K and V, so everything serves their stream.  A CTA has
// four warps; a unit is four sub-blocks of keys, one per warp (16 keys of 16
// bits, 8 of 32), which lie in one block each.  A warp streams its sub-blocks
// through a ring of its own with 16-byte cp.async (24 KB a warp, two CTAs an
// SM: 128 KB in flight per SM where 45 KB cover the latency at full rate), and
// the ring runs on over the ends of items.  Nothing in the loop waits for
// another warp: each keeps its own running maximum, sum and output of the
// softmax, which meet in shared memory at the end of an item (the ring stage
// just consumed holds them).
//
// An item's rows are the query heads of the group, times tokens.  Up to 16 of
// them are one operand tile of mma.sync: with so few rows the tensor cores of either
// kind are idle most of the time, and the register operands of mma.sync need
// no descriptors, barriers or tensor memory.  Scores S = Q K^T come out with a
// row's keys in one quad of lanes, in the layout that the second product wants
// its left operand in.
//
// 16 bits: m16n8k16.  p is split into a 16-bit head and a 16-bit rest (two
// products), so that 2^-18 of it is lost at most, far below the rounding of the
// output; in fp16, where p is lifted to 2^15, 2^-40 of the largest weight at most.
// 32 bits: m16n8k8 on TF32 with every operand split x = hi + lo and three
// products hi hi + hi lo + lo hi, as in gemm_tma.cu; scores are summed in four
// accumulators.  The dimensions (keys, for the second product) are dealt to the
// operand's index in an order that lets a lane read four of them at once.
//
// Up to eight rows of 32 bits stay on the CUDA cores: there a row costs its own
// products only, where the tile costs sixteen rows' three times over (us, 16
// requests over 4000 keys, 16 heads on 8 of 128, CUDA cores / tile: 8 rows 98 / 139,
// 4 rows 85 / 139).  A lane holds four dimensions of
// every row's query and output; the partial scores of eight keys times R rows are
// summed over the lanes by exchanging halves (one shuffle per value, not five).
//
// A masked key gets p = 0; keys behind the length and keys of bad table entries
// are not read at all (cp.async fills zeros), so nothing that lies there can
// reach the sums.
#include <algorithm>

#include "paged_attn.cuh"

namespace itts {
namespace paged {
namespace {

constexpr int kMmaRows = 16;  // of the mma.sync operand
constexpr int kSimtMost = 8;   // rows of 32 bits that the CUDA cores take
constexpr int kFewWarps = 4;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kRingBytes = 24 * 1024;  // per warp
// Units over which a warp's sums run on.  A weight below 2^-24 of a running fp32 sum is lost to it, and every sum is
// off by up to that much: over 2^19 keys, 2^17 of a warp, with one key 17 nats ahead, fp32 results were off by 4e-3
// (2e-5 so).  After a stretch the warps' sums meet in the item's slot of the workspace, as at the end of a share: 2^-16
// for the stretch and 2^-24 for each.  Us without and with: 16 steps over 420 keys 12.2 / 12.4, 64 over 16384 322 / 324.
constexpr int kFewStretch = 256;

template <class T, int D>
struct Few {
    static constexpr int kKeys = sizeof(T) == 4 ? 8 : 16;      // of a sub-block
    static constexpr int kUnit = kKeys * kFewWarps;
    static constexpr int kHalf = kKeys * D * int(sizeof(T));   // bytes of K (and of V) in a stage
    static constexpr int kStages = kRingBytes / (2 * kHalf);
    static constexpr int kChunks = D * int(sizeof(T)) / 16;    // 16-byte chunks of a key row
    static_assert(2 * kHalf >= kMmaRows * D * 4, "a stage holds a warp's output");
};
constexpr size_t kFewSmem = size_t(kRingBytes) * kFewWarps;

// Chunk of row r that chunk c is kept at (see the reads below: every access of
// eight lanes falls on eight different banks of 16 bytes).
template <class T>
__device__ __forceinline__ int swz_k(int r, int c) {
    return sizeof(T) == 4 ? c ^ ((r & 1) << 2) : c ^ (r & 7);
}
template <class T>
__device__ __forceinline__ int swz_v(int r, int c) {
    return sizeof(T) == 4 ? c ^ (((r >> 1) & 3) << 1) : c ^ (r & 7);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <class T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const float (&a)[4], float b0, float b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
          "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// The conversion keeps every NaN a NaN, which adding to the bits (rn_tf32) would not.
__device__ __forceinline__ float cvt_tf32(float x) {
    uint32_t y;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
    return __uint_as_float(y);
}
// One product of fp32 operands split into TF32 hi and lo.
__device__ __forceinline__ void mma8x3(float (&d)[4], const float (&ah)[4], const float (&al)[4], float x0, float x1) {
    const float h0 = cvt_tf32(x0), h1 = cvt_tf32(x1);
    mma8(d, ah, rn_tf32(x0 - h0), rn_tf32(x1 - h1));
    mma8(d, al, h0, h1);
    mma8(d, ah, h0, h1);
}

// What two values in 16 bits stand for.
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Rows of queries in the registers of a warp: lane (g, c) = (lane / 4, lane % 4).
template <class T, int D>
struct Query;

template <class T, int D>
struct Query {  // 16 bits: A fragments of m16n8k16
    uint32_t f[D / 16][4];
    __device__ __forceinline__ void load(const T* r0, const T* r1, int c, float sign) {
        const uint32_t flip = sign < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[k][2 * i] = r0 ? __ldg(reinterpret_cast<const uint32_t*>(r0 + 16 * k + 8 * i) + c) ^ flip : 0u;
                f[k][2 * i + 1] = r1 ? __ldg(reinterpret_cast<const uint32_t*>(r1 + 16 * k + 8 * i) + c) ^ flip : 0u;
            }
        }
    }
};
template <int D>
struct Query<float, D> {  // 32 bits: dimension 16 j + 4 c + i, split when used
    float4 x[D / 16][2];
    __device__ __forceinline__ void load(const float* r0, const float* r1, int c, float sign) {
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            x[j][0] = r0 ? __ldg(reinterpret_cast<const float4*>(r0) + 4 * j + c) : z;
            x[j][1] = r1 ? __ldg(reinterpret_cast<const float4*>(r1) + 4 * j + c) : z;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                x[j][i] = make_float4(x[j][i].x * sign, x[j][i].y * sign, x[j][i].z * sign, x[j][i].w * sign);
        }
    }
};

__device__ __forceinline__ void split4(const float (&x)[4], float (&h)[4], float (&l)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = cvt_tf32(x[i]);
        l[i] = rn_tf32(x[i] - h[i]);
    }
}

// Partial sums v[0 .. N) of 32 or 16 lanes (those that differ in the bits of `off`
// and below) are summed; N times the lane's part of the group is the index of
// what a lane is left with: one value, or N / group of them.
template <int N>
__device__ __forceinline__ void sum_exchange(float (&v)[N], int off, int lane) {
    int n = N;
#pragma unroll
    for (int step = 0; step < 5; ++step) {
        if (off == 0) break;
        if (n > 1) {
            n /= 2;
            const bool up = lane & off;
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (i < n) {
                    const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
                }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
        }
        off >>= 1;
    }
}

// The arithmetic of a warp on one item of R rows: query, running maximum and sum,
// output.  begin() at an item's start, unit() for a sub-block in the ring, end() leaves
// (maximum, sum) and outputs of rows 0 .. rows in shared memory, chunk c of row r
// of four floats at c ^ (r & 7).

// R = 16: one tile of mma.sync.  Lane (g, c) = (lane / 4, lane % 4) holds rows g, g + 8.
template <class T, int D, int R>
struct Rows {
    static_assert(R == kMmaRows, "");
    using F = Few<T, D>;
    static constexpr bool kSwizzled = true;
    Query<T, D> q;
    float m[2], l[2], o[D / 8][4];
    int lim[2];  // keys that the lane's rows see
    // row(r): query of row r, or null; seen(r): keys that it sees
    template <class Row, class Seen>
    __device__ __forceinline__ void begin(const Row& row, const Seen& seen, float sign, int lane) {
        const int g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            lim[j] = seen(g + 8 * j);
            m[j] = -INFINITY;
            l[j] = 0.f;
        }
        q.load(row(g), row(g + 8), c, sign);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    }
    __device__ __forceinline__ void unit(const unsigned char* stage, uint32_t stage_u, int key0, bool named, float scale2,
                                         int lane) {
        constexpr int KS = F::kKeys;
        const int g = lane >> 2, c = lane & 3;
        const uint32_t kb = stage_u, vb = stage_u + F::kHalf;
        constexpr int NT = KS / 8;
        float sc[NT][4];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
            const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t f[4];  // keys 0-7 (both halves of 16 dimensions), keys 8-15
                ldsm4(f, kb + kr * (F::kChunks * 16) + swz_k<T>(kr, 2 * k + kc) * 16);
                mma16<T>(sc[0], q.f[k], f[0], f[1]);
                mma16<T>(sc[1], q.f[k], f[2], f[3]);
            }
        } else {
            float part[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) part[t][0] = part[t][1] = part[t][2] = part[t][3] = 0.f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const float4 kx = *reinterpret_cast<const float4*>(stage + g * (F::kChunks * 16) +
                                                                   swz_k<T>(g, 4 * j + c) * 16);
                const float4 q0 = q.x[j][0], q1 = q.x[j][1];
                float h[4], lo[4];
                split4({q0.x, q1.x, q0.y, q1.y}, h, lo);
                mma8x3(part[j & 3], h, lo, kx.x, kx.y);
                split4({q0.z, q1.z, q0.w, q1.w}, h, lo);
                mma8x3(part[j & 3], h, lo, kx.z, kx.w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[0][e] = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
        }

        // the softmax's running maximum and sum; a row's keys are in the four lanes of a quad
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = key0 + 8 * t + 2 * c + (e & 1);
                if (!named || key >= lim[e >> 1]) sc[t][e] = -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], sc[t][e]);
            }
        float ref[2], cor[2];
        bool moved = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 1));
            mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 2));
            const float mn = fmaxf(m[j], mx[j] * scale2);
            moved |= mn > m[j];
            ref[j] = mn == -INFINITY ? 0.f : mn;
            cor[j] = ex2(m[j] - ref[j]);
            ref[j] -= lift<T>(0);
            m[j] = mn;
            l[j] *= cor[j];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
                o[j][0] *= cor[0];
                o[j][1] *= cor[0];
                o[j][2] *= cor[1];
                o[j][3] *= cor[1];
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][e] = ex2(fmaf(sc[t][e], scale2, -ref[e >> 1]));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float sum = sc[0][2 * j] + sc[0][2 * j + 1];
            if constexpr (NT == 2) sum += sc[1][2 * j] + sc[1][2 * j + 1];
            l[j] += sum;
        }

        if constexpr (sizeof(T) == 2) {
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // (row g, keys 2c..), (row g + 8, ..), the same of keys 8 + 2c
                const float y0 = sc[x >> 1][2 * (x & 1)], y1 = sc[x >> 1][2 * (x & 1) + 1];
                ph[x] = pack2<T>(y0, y1);
                const float2 r = unpack2<T>(ph[x]);
                pl[x] = pack2<T>(y0 - r.x, y1 - r.y);
            }
            const int vr = lane & 15, vc = lane >> 4;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                uint32_t f[4];  // keys 0-7, 8-15 of dimensions 0-7, then of 8-15
                ldsm4t(f, vb + vr * (F::kChunks * 16) + swz_v<T>(vr, 2 * d + vc) * 16);
                // fresh sums, added here: see the products of 32 bits below (over 2^20 keys 1.5e-3 of the result)
                float y[2][4] = {};
                mma16<T>(y[0], pl, f[0], f[1]);
                mma16<T>(y[1], pl, f[2], f[3]);
                mma16<T>(y[0], ph, f[0], f[1]);
                mma16<T>(y[1], ph, f[2], f[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[2 * d][e] += y[0][e];
                    o[2 * d + 1][e] += y[1][e];
                }
            }
        } else {
            // operand index c is key 2c, c + 4 is key 2c + 1; column n of tile 4 q + t is dimension 32 q + 4 n + t
            float h[4], lo[4];
            split4({sc[0][0], sc[0][2], sc[0][1], sc[0][3]}, h, lo);
#pragma unroll
            for (int qd = 0; qd < D / 32; ++qd) {
                const unsigned char* base = stage + F::kHalf;
                const float4 v0 = *reinterpret_cast<const float4*>(base + (2 * c) * (F::kChunks * 16) +
                                                                   swz_v<T>(2 * c, 8 * qd + g) * 16);
                const float4 v1 = *reinterpret_cast<const float4*>(base + (2 * c + 1) * (F::kChunks * 16) +
                                                                   swz_v<T>(2 * c + 1, 8 * qd + g) * 16);
                // each sub-block's sums start afresh and are added here: the tensor core's own accumulation does
                // not round to nearest, which showed over a thousand keys (1.6e-6 of the result, 0.5e-6 so)
                float y[4][4] = {};
                mma8x3(y[0], h, lo, v0.x, v1.x);
                mma8x3(y[1], h, lo, v0.y, v1.y);
                mma8x3(y[2], h, lo, v0.z, v1.z);
                mma8x3(y[3], h, lo, v0.w, v1.w);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * qd + t][e] += y[t][e];
            }
        }
    }
    __device__ __forceinline__ void end(float* dst, float2* ml, int rows, int lane) {
        const int g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
            l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
            const int r = g + 8 * j;
            if (r < rows) {
                if (c == 0) ml[r] = make_float2(m[j], l[j]);
                float* to = dst + r * D;
                const int x = (r & 7) << 2;  // floats of a row are kept in chunks of four at chunk ^ (r & 7)
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int d = 0; d < D / 8; ++d)
                        *reinterpret_cast<float2*>(to + ((8 * d + 2 * c) ^ x)) = make_float2(o[d][2 * j], o[d][2 * j + 1]);
                } else {
#pragma unroll
                    for (int qd = 0; qd < D / 32; ++qd)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *reinterpret_cast<float4*>(to + ((32 * qd + 8 * c + 4 * e) ^ x)) =
                                make_float4(o[4 * qd][2 * j + e], o[4 * qd + 1][2 * j + e], o[4 * qd + 2][2 * j + e],
                                            o[4 * qd + 3][2 * j + e]);
                }
            }
        }
    }
};

// R <= 8 rows of fp32 on the CUDA cores.  Lanes of a key: 32 (head_dim 128) or 16, four
// dimensions each; kE rows of the scores per lane after the exchange: lane = (key, row).
template <int D, int R>
struct Rows32 {
    using F = Few<float, D>;
    static constexpr bool kSwizzled = false;
    static constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes, kIter = 8 / kAtOnce, kE = R > 4 ? R / 4 : 1;
    static_assert(F::kKeys == 8, "");
    float4 q[R], o[R];
    float m[kE], l[kE];
    int lim[kE];
    // row of this lane's e-th score, and the lane (of a key's four) that holds row r
    static __device__ __forceinline__ int row_of(int lane, int e) { return (lane & 3) * R / 4 + e; }
    static __device__ __forceinline__ int lane_of(int r) { return r * 4 / R; }
    template <class Row, class Seen>
    __device__ __forceinline__ void begin(const Row& row, const Seen& seen, float sign, int lane) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float* p = row(r);
            const float4 y = p ? __ldg(reinterpret_cast<const float4*>(p) + lane % kLanes) : make_float4(0.f, 0.f, 0.f, 0.f);
            q[r] = make_float4(y.x * sign, y.y * sign, y.z * sign, y.w * sign);
            o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            lim[e] = seen(row_of(lane, e));
            m[e] = -INFINITY;
            l[e] = 0.f;
        }
    }
    __device__ __forceinline__ void unit(const unsigned char* stage, uint32_t, int key0, bool named, float scale2,
                                         int lane) {
        const float4* k = reinterpret_cast<const float4*>(stage) + lane;
        const float4* v = reinterpret_cast<const float4*>(stage + F::kHalf) + lane;
        float s[kIter * R];
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const float4 x = k[32 * i];  // key kAtOnce i + lane / kLanes
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float2 y = fma2(make_float2(x.z, x.w), make_float2(q[r].z, q[r].w),
                                      make_float2(x.x * q[r].x, x.y * q[r].y));
                s[i * R + r] = y.x + y.y;
            }
        }
        sum_exchange(s, kLanes / 2, lane);
        const int key = key0 + (D == 128 ? lane >> 2 : 2 * ((lane >> 2) & 3) + (lane >> 4));
        float ref[kE], cor[kE];
        bool moved = false;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            if (!named || key >= lim[e]) s[e] = -INFINITY;
            float mx = s[e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float mn = fmaxf(m[e], mx * scale2);
            moved |= mn > m[e];
            ref[e] = mn == -INFINITY ? 0.f : mn;
            cor[e] = ex2(m[e] - ref[e]);
            m[e] = mn;
            s[e] = ex2(fmaf(s[e], scale2, -ref[e]));
            l[e] = fmaf(l[e], cor[e], s[e]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float f = __shfl_sync(0xffffffffu, cor[r % kE], lane_of(r));
                o[r] = make_float4(o[r].x * f, o[r].y * f, o[r].z * f, o[r].w * f);
            }
        }
        const int half = D == 128 ? 0 : lane & 16;
        float4 y[R];  // of this sub-block, added to the running sums at once
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
            const float4 x = v[32 * i];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float p = __shfl_sync(0xffffffffu, s[r % kE], half + 4 * i + lane_of(r));
                if (i == 0) {
                    y[r] = make_float4(p * x.x, p * x.y, p * x.z, p * x.w);
                } else {
                    const float2 a = fma2(make_float2(p, p), make_float2(x.x, x.y), make_float2(y[r].x, y[r].y));
                    const float2 b = fma2(make_float2(p, p), make_float2(x.z, x.w), make_float2(y[r].z, y[r].w));
                    y[r] = make_float4(a.x, a.y, b.x, b.y);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) o[r] = make_float4(o[r].x + y[r].x, o[r].y + y[r].y, o[r].z + y[r].z, o[r].w + y[r].w);
    }
    __device__ __forceinline__ void end(float* dst, float2* ml, int rows, int lane) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
            const int r = row_of(lane, e);
            if (lane < 4 && r < rows && lane == lane_of(r)) ml[r] = make_float2(m[e], l[e]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (D == 64) {
                o[r].x += __shfl_xor_sync(0xffffffffu, o[r].x, 16);
                o[r].y += __shfl_xor_sync(0xffffffffu, o[r].y, 16);
                o[r].z += __shfl_xor_sync(0xffffffffu, o[r].z, 16);
                o[r].w += __shfl_xor_sync(0xffffffffu, o[r].w, 16);
            }
            if (r < rows && lane < kLanes) reinterpret_cast<float4*>(dst + r * D)[lane ^ (r & 7)] = o[r];
        }
    }
};
template <int D>
struct Rows<float, D, 1> : Rows32<D, 1> {};
template <int D>
struct Rows<float, D, 2> : Rows32<D, 2> {};
template <int D>
struct Rows<float, D, 4> : Rows32<D, 4> {};
template <int D>
struct Rows<float, D, 8> : Rows32<D, 8> {};

template <class T, int D, int R>
__global__ void __launch_bounds__(kFewThreads, 2) k_attn_few(const __grid_constant__ Attn a) {
    using F = Few<T, D>;
    using Math = Rows<T, D, R>;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ PlanSmem<kFewThreads> plan_smem;
    __shared__ float2 ml[kFewWarps][R], kept[2][R];
    constexpr int S = F::kStages, KS = F::kKeys;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* my_ring = ring + warp * kRingBytes;
    const uint32_t ring_u = smem_u32(my_ring);

    pdl_trigger();
    pdl_wait();
    const int units = plan<R, F::kUnit, 0, kFewThreads>(a, blockIdx.x, gridDim.x, plan_smem, reinterpret_cast<long long*>(ring));
    const Share& sh = plan_smem.share;
    if (threadIdx.x == 0) put_record(a, blockIdx.x, 0, 0, 0, 0, 0);
    const int n = units;
    if (n == 0) return;

    Walk<R, F::kUnit, 0> in, at;  // of the loads and of the arithmetic
    at.start(a, sh);
    in = at;
    int in_keys = in.r.template keys<R>(a, in.t), ids_b = -1, ids_k = 0, ids = 0;
    uint32_t good = 0;  // bit s: stage s holds a block that the table names

    const auto issue = [&](int i) {  // unit i of the share into stage i % S
        if (i < n) {
            // lane l keeps the table entry of this warp's sub-block in unit ids_k + l
            if (ids_b != in.b || in.k < ids_k || in.k >= ids_k + 32) {
                ids_b = in.b;
                ids_k = in.k;
                const long long page = ((long long)(in.k + lane) * F::kUnit + warp * KS) >> a.shift;
                ids = page < (a.cap >> a.shift) && (page << a.shift) < in.r.len
                          ? __ldcg(a.table + in.b * a.table_stride + page)
                          : -1;
            }
            const int id = __shfl_sync(0xffffffffu, ids, in.k - ids_k);
            const int key0 = in.k * F::kUnit + warp * KS, s = i % S;
            const bool ok = (unsigned)id < (unsigned)a.c.blocks;
            good = (good & ~(1u << s)) | (uint32_t(ok) << s);
            const long long block = ok ? id : 0, tok = key0 & ((1 << a.shift) - 1);
            const T* k = static_cast<const T*>(a.c.k) + block * a.c.k_block_stride + tok * a.c.k_token_stride +
                         in.h * a.c.k_head_stride;
            const T* v = static_cast<const T*>(a.c.v) + block * a.c.v_block_stride + tok * a.c.v_token_stride +
                         in.h * a.c.v_head_stride;
            const uint32_t dst = ring_u + s * (2 * F::kHalf);
            constexpr int kPer = KS * F::kChunks / 32;  // chunks of K per lane
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int x = j * 32 + lane, row = x / F::kChunks, ch = x % F::kChunks;
                const int bytes = ok && key0 + row < in_keys ? 16 : 0;
                const long long r = bytes ? row : 0;  // what is not read is not addressed either
                cp16(dst + row * (F::kChunks * 16) + (Math::kSwizzled ? swz_k<T>(row, ch) : ch) * 16, k + r * a.c.k_token_stride + ch * (16 / sizeof(T)), bytes);
                cp16(dst + F::kHalf + row * (F::kChunks * 16) + (Math::kSwizzled ? swz_v<T>(row, ch) : ch) * 16,
                     v + r * a.c.v_token_stride + ch * (16 / sizeof(T)), bytes);
            }
            in.advance(a, 1);
            if (in.k == 0) {
                in_keys = in.r.template keys<R>(a, in.t);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    Math math;
    int rows = 0, first = 0;
    int stretch = 0, folds = 0;         // units of this stretch of the item, stretches before it
    bool fresh = false, begun = false;  // begun: the item's first unit is this share's
    const auto begin = [&] {            // the item that the arithmetic has come to, or its next stretch
        if (folds == 0) begun = at.k == 0;
        stretch = 0;
        first = at.t * R;
        rows = min(R, at.r.rows - first);
        math.begin(
            [&](int r) {
                const int tok = over_group(a, first + r), hd = first + r - tok * a.group;
                return r < rows ? static_cast<const T*>(a.q) + (long long)(at.r.start + tok) * a.q_row +
                                      (long long)(at.h * a.group + hd) * a.q_head
                                : nullptr;
            },
            [&](int r) { return r < rows ? min(max(at.r.pos(a, first + r) + 1, 0), a.cap) : 0; }, a.sign, lane);
    };
    begin();  // its loads are on their way before the table entries are
    for (int i = 0; i < S - 1; ++i) issue(i);

    for (int i = 0; i < n; ++i) {
        if (fresh) begin();
        fresh = false;
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();
        const int s = i % S, key0 = at.k * F::kUnit + warp * KS;
        const bool named = (good >> s) & 1;
        issue(i + S - 1);  // into the stage consumed one unit ago

        math.unit(my_ring + s * (2 * F::kHalf), ring_u + s * (2 * F::kHalf), key0, named, a.scale2, lane);

        const bool last = at.k + 1 == at.nk || i + 1 == n;
        if (__builtin_expect(!last && ++stretch < kFewStretch, 1)) {
            at.advance(a, 1);
            continue;
        }

        // The item's keys end here, or this share or a stretch does: the warps' sums meet.
        // Each warp's output goes to the stage it has just consumed.
        float* mine = reinterpret_cast<float*>(my_ring + s * (2 * F::kHalf));
        __syncwarp();
        math.end(mine, ml[warp], rows, lane);
        __syncthreads();
        const bool whole = last && begun && at.k + 1 == at.nk;
        float* slot = part_slot<R, D>(a, blockIdx.x, begun ? 1 : 0);
        for (int x = threadIdx.x; x < rows * (D / 4); x += kFewThreads) {
            const int r = x / (D / 4), d4 = x % (D / 4);
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, ml[w][r].x);
            float2 old = make_float2(-INFINITY, 0.f);
            if (__builtin_expect(folds > 0, 0)) M = fmaxf(M, (old = kept[folds & 1][r]).x);
            const float rf = M == -INFINITY ? 0.f : M;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float f = ex2(ml[w][r].x - rf);
                const float4 v = *reinterpret_cast<const float4*>(
                    reinterpret_cast<const float*>(ring + w * kRingBytes + s * (2 * F::kHalf)) + r * D + ((4 * d4) ^ ((r & 7) << 2)));
                L += ml[w][r].y * f;
                y = make_float4(y.x + v.x * f, y.y + v.y * f, y.z + v.z * f, y.w + v.w * f);
            }
            if (__builtin_expect(folds > 0, 0)) {  // written by this thread at the stretch before
                const float f = ex2(old.x - rf);
                const float4 v = *reinterpret_cast<const float4*>(slot + r * D + 4 * d4);
                L += old.y * f;
                y = make_float4(y.x + v.x * f, y.y + v.y * f, y.z + v.z * f, y.w + v.w * f);
            }
            if (whole) {
                store4<T>(out_row<T>(a, at.r.start, first, r, at.h) + 4 * d4, normalised(y, L));
            } else {
                *reinterpret_cast<float4*>(slot + r * D + 4 * d4) = y;
                if (d4 == 0) (last ? reinterpret_cast<float2*>(slot + R * D) : kept[(folds + 1) & 1])[r] = make_float2(M, L);
            }
        }
        if (last && !whole && begun && threadIdx.x == 0) {  // it goes on: in how many shares
            const int end = cta_of(sh, sh.u0 + i + (at.nk - at.k) - 1);
            put_record(a, blockIdx.x, end - int(blockIdx.x) + 1, at.h, rows, at.r.start, first);
        }
        __syncthreads();
        at.advance(a, 1);
        fresh = true;
        folds = last ? 0 : folds + 1;
    }
}

template <class T, int D, int R>
cudaError_t launch(const Attn& a, long long rows, cudaStream_t s) {
    cudaError_t e = allow_smem<k_attn_few<T, D, R>>(kFewSmem);
    if (e != cudaSuccess) return e;
    const int ctas = 2 * 148;
    if ((e = launch_pdl(k_attn_few<T, D, R>, ctas, kFewThreads, kFewSmem, s, a)) != cudaSuccess) return e;
    return launch_pdl(k_join<T, R, D>, dim3(ctas, unsigned(std::min<long long>(rows, R))), kJoinThreads, 0, s, a);
}

// The smallest R that holds `rows`; more take several tiles.
template <int D>
cudaError_t launch32(const Attn& a, long long rows, cudaStream_t s) {
    if (rows <= 1) return launch<float, D, 1>(a, rows, s);
    if (rows <= 2) return launch<float, D, 2>(a, rows, s);
    if (rows <= 4) return launch<float, D, 4>(a, rows, s);
    if (rows <= kSimtMost) return launch<float, D, 8>(a, rows, s);
    return launch<float, D, kMmaRows>(a, rows, s);
}

}  // namespace

size_t few_workspace_floats(int head_dim) {
    return 2 * 2 * 148 * (head_dim == 64 ? part_floats<kMmaRows, 64>() : part_floats<kMmaRows, 128>());
}

// rows: of a request and kv head, as far as the host knows.
cudaError_t launch_few(const Attn& a, long long rows, cudaStream_t s) {
    const bool wide = a.c.head_dim == 128;
    constexpr int R = kMmaRows;
    switch (a.c.type) {
        case ITTS_PAGED_F16: return wide ? launch<__half, 128, R>(a, rows, s) : launch<__half, 64, R>(a, rows, s);
        case ITTS_PAGED_BF16: return wide ? launch<__nv_bfloat16, 128, R>(a, rows, s) : launch<__nv_bfloat16, 64, R>(a, rows, s);
        default: return wide ? launch32<128>(a, rows, s) : launch32<64>(a, rows, s);
    }
}

}  // namespace paged
}  // namespace itts
