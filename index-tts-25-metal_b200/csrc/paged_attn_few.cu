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
// The rows of an item (up to 16: the query heads of the group, times tokens)
// are one operand tile of mma.sync: with so few rows the tensor cores of either
// kind are idle most of the time, and the register operands of mma.sync need
// no descriptors, barriers or tensor memory.  Scores S = Q K^T come out with a
// row's keys in one quad of lanes, in the layout that the second product wants
// its left operand in.
//
// 16 bits: m16n8k16.  p is split into a 16-bit head and a 16-bit rest (two
// products), so that rounding p adds nothing to the rounding of the output.
// 32 bits: m16n8k8 on TF32 with every operand split x = hi + lo and three
// products hi hi + hi lo + lo hi, as in gemm_tma.cu; scores are summed in four
// accumulators.  The dimensions (keys, for the second product) are dealt to the
// operand's index in an order that lets a lane read four of them at once.
//
// A masked key gets p = 0; keys behind the length and keys of bad table entries
// are not read at all (cp.async fills zeros), so nothing that lies there can
// reach the sums.
#include "paged_attn.cuh"

namespace itts {
namespace paged {
namespace {

constexpr int kFewRows = 16;
constexpr int kFewWarps = 4;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kRingBytes = 24 * 1024;  // per warp

template <class T, int D>
struct Few {
    static constexpr int kKeys = sizeof(T) == 4 ? 8 : 16;      // of a sub-block
    static constexpr int kUnit = kKeys * kFewWarps;
    static constexpr int kHalf = kKeys * D * int(sizeof(T));   // bytes of K (and of V) in a stage
    static constexpr int kStages = kRingBytes / (2 * kHalf);
    static constexpr int kChunks = D * int(sizeof(T)) / 16;    // 16-byte chunks of a key row
    static_assert(2 * kHalf >= kFewRows * D * 4, "a stage holds a warp's output");
};
constexpr size_t kFewSmem = size_t(kRingBytes) * kFewWarps;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

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

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// Two values in 16 bits, and what the rounding left.
template <class T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
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

template <class T, int D>
__global__ void __launch_bounds__(kFewThreads, 2) k_attn_few(const __grid_constant__ Attn a) {
    using F = Few<T, D>;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ PlanSmem<kFewThreads> plan_smem;
    __shared__ float2 ml[kFewWarps][kFewRows];
    constexpr int S = F::kStages, KS = F::kKeys;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    unsigned char* my_ring = ring + warp * kRingBytes;
    const uint32_t ring_u = smem_u32(my_ring);

    pdl_trigger();
    pdl_wait();
    const Share sh = plan<kFewRows, F::kUnit, kFewThreads>(a, blockIdx.x, gridDim.x, plan_smem);
    if (threadIdx.x == 0) put_record(a, blockIdx.x, 0, 0, 0, 0, 0);
    const int n = int(sh.u1 - sh.u0);
    if (n == 0) return;

    Walk<kFewRows, F::kUnit> in, at;  // of the loads and of the arithmetic
    at.start(a, sh);
    in = at;
    int in_keys = in.r.template keys<kFewRows>(a, in.t), ids_b = -1, ids_k = 0, ids = 0;
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
                cp16(dst + row * (F::kChunks * 16) + swz_k<T>(row, ch) * 16, k + r * a.c.k_token_stride + ch * (16 / sizeof(T)), bytes);
                cp16(dst + F::kHalf + row * (F::kChunks * 16) + swz_v<T>(row, ch) * 16,
                     v + r * a.c.v_token_stride + ch * (16 / sizeof(T)), bytes);
            }
            if (++in.k == in.nk && i + 1 < n) {
                in.next(a);
                in_keys = in.r.template keys<kFewRows>(a, in.t);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    for (int i = 0; i < S - 1; ++i) issue(i);

    Query<T, D> q;
    float m[2], l[2], o[D / 8][4];
    int lim[2], rows = 0, first = 0;  // keys that the lane's two rows see; the item's rows
    bool fresh = true, begun = false; // an item's first unit here; begun: it is the item's first unit at all
    for (int i = 0; i < n; ++i) {
        if (fresh) {
            fresh = false;
            begun = at.k == 0;
            first = at.t * kFewRows;
            rows = min(kFewRows, at.r.rows - first);
            const T* row[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = g + 8 * j;
                lim[j] = r < rows ? min(max(at.r.pos(a, first + r) + 1, 0), a.cap) : 0;
                const int tok = (first + r) / a.group, hd = (first + r) - tok * a.group;
                row[j] = r < rows ? static_cast<const T*>(a.q) + (long long)(at.r.start + tok) * a.q_row +
                                        (long long)(at.h * a.group + hd) * a.q_head
                                  : nullptr;
                m[j] = -INFINITY;
                l[j] = 0.f;
            }
            q.load(row[0], row[1], c, a.sign);
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();
        const int s = i % S, key0 = at.k * F::kUnit + warp * KS;
        const bool named = (good >> s) & 1;
        issue(i + S - 1);  // into the stage consumed one unit ago

        const uint32_t kb = ring_u + s * (2 * F::kHalf), vb = kb + F::kHalf;
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
                const float4 kx = *reinterpret_cast<const float4*>(my_ring + (kb - ring_u) + g * (F::kChunks * 16) +
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
            const float mn = fmaxf(m[j], mx[j] * a.scale2);
            moved |= mn > m[j];
            ref[j] = mn == -INFINITY ? 0.f : mn;
            cor[j] = ex2(m[j] - ref[j]);
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
            for (int e = 0; e < 4; ++e) {
                sc[t][e] = ex2(fmaf(sc[t][e], a.scale2, -ref[e >> 1]));
                l[e >> 1] += sc[t][e];
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
                mma16<T>(o[2 * d], pl, f[0], f[1]);
                mma16<T>(o[2 * d + 1], pl, f[2], f[3]);
                mma16<T>(o[2 * d], ph, f[0], f[1]);
                mma16<T>(o[2 * d + 1], ph, f[2], f[3]);
            }
        } else {
            // operand index c is key 2c, c + 4 is key 2c + 1; column n of tile 4 q + t is dimension 32 q + 4 n + t
            float h[4], lo[4];
            split4({sc[0][0], sc[0][2], sc[0][1], sc[0][3]}, h, lo);
#pragma unroll
            for (int qd = 0; qd < D / 32; ++qd) {
                const unsigned char* base = my_ring + (vb - ring_u);
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

        if (++at.k < at.nk && i + 1 < n) continue;

        // The item's keys end here, or this share does: the warps' sums meet.
        // Each warp's output goes to the stage it has just consumed.
        float* mine = reinterpret_cast<float*>(my_ring + s * (2 * F::kHalf));
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
            l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
            const int r = g + 8 * j;
            if (r < rows) {
                if (c == 0) ml[warp][r] = make_float2(m[j], l[j]);
                float* dst = mine + r * D;
                const int x = (r & 7) << 2;  // floats of a row are kept in chunks of four at chunk ^ (r & 7)
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int d = 0; d < D / 8; ++d)
                        *reinterpret_cast<float2*>(dst + ((8 * d + 2 * c) ^ x)) = make_float2(o[d][2 * j], o[d][2 * j + 1]);
                } else {
#pragma unroll
                    for (int qd = 0; qd < D / 32; ++qd)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *reinterpret_cast<float4*>(dst + ((32 * qd + 8 * c + 4 * e) ^ x)) =
                                make_float4(o[4 * qd][2 * j + e], o[4 * qd + 1][2 * j + e], o[4 * qd + 2][2 * j + e],
                                            o[4 * qd + 3][2 * j + e]);
                }
            }
        }
        __syncthreads();
        const bool whole = begun && at.k == at.nk;
        float* slot = whole ? nullptr : part_slot<kFewRows, D>(a, blockIdx.x, begun ? 1 : 0);
        for (int x = threadIdx.x; x < rows * (D / 4); x += kFewThreads) {
            const int r = x / (D / 4), d4 = x % (D / 4);
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, ml[w][r].x);
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
            if (whole) {
                store4<T>(out_row<T>(a, at.r.start, first, r, at.h) + 4 * d4, normalised(y, L));
            } else {
                *reinterpret_cast<float4*>(slot + r * D + 4 * d4) = y;
                if (d4 == 0) reinterpret_cast<float2*>(slot + kFewRows * D)[r] = make_float2(M, L);
            }
        }
        if (!whole && begun && threadIdx.x == 0) {  // it goes on: in how many shares
            const int last = cta_of(sh, sh.u0 + i + (at.nk - at.k));
            put_record(a, blockIdx.x, last - int(blockIdx.x) + 1, at.h, rows, at.r.start, first);
        }
        __syncthreads();
        if (i + 1 < n) at.next(a);
        fresh = true;
    }
}

template <class T, int D>
cudaError_t launch(const Attn& a, cudaStream_t s) {
    cudaError_t e = allow_smem<k_attn_few<T, D>>(kFewSmem);
    if (e != cudaSuccess) return e;
    const int ctas = 2 * 148;
    if ((e = launch_pdl(k_attn_few<T, D>, ctas, kFewThreads, kFewSmem, s, a)) != cudaSuccess) return e;
    return launch_pdl(k_join<T, kFewRows, D>, ctas, kJoinThreads, kJoinThreads * sizeof(float4), s, a);
}

}  // namespace

size_t few_workspace_floats(int head_dim) {
    return 2 * 2 * 148 * (head_dim == 64 ? part_floats<kFewRows, 64>() : part_floats<kFewRows, 128>());
}

cudaError_t launch_few(const Attn& a, cudaStream_t s) {
    const bool wide = a.c.head_dim == 128;
    switch (a.c.type) {
        case ITTS_PAGED_F16: return wide ? launch<__half, 128>(a, s) : launch<__half, 64>(a, s);
        case ITTS_PAGED_BF16: return wide ? launch<__nv_bfloat16, 128>(a, s) : launch<__nv_bfloat16, 64>(a, s);
        default: return wide ? launch<float, 128>(a, s) : launch<float, 64>(a, s);
    }
}

}  // namespace paged
}  // namespace itts
