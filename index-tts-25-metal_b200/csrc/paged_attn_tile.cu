// Paged attention of many rows per request (prompt chunks), 16-bit types, on
// the 5th-generation tensor cores.
//
// S = Q K^T and O += P V are 128 x 128 (x head_dim) tcgen05 products; bound by
// them and, as closely, by the exponentials: a 128 x 128 tile of scores takes
// 1024 clocks of the tensor core (both products, head_dim 128) and 1024 clocks of
// the SM's exponential units.  So the two must run at once.  A CTA works on an
// item of 256 rows as two tiles of 128 with a softmax warpgroup each: while
// one tile's scores go through the exponentials, the tensor core runs the other
// tile's P V and next Q K^T.
//
// 384 threads in five roles:
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread per row (no shuffles).  Loads
//                   its 128 scores from tensor memory, keeps the running maximum
//                   and sum, writes P in 16 bits over the scores.  The output is
//                   rescaled only when the maximum has grown by 2^8 or more
//                   since the last time (P then stays below 2^8, far from
//                   the 16-bit types' limits, and the division at the end
//                   takes the same maximum out again).  Half of the exponentials
//                   are computed on the FMA units (exp2_fit).  Writes the
//                   output, or the partial sums, at an item's end.
//   warp 8          issues the products (one lane): per unit and tile P V of this
//                   unit, then Q K^T of the next, in that order into the same
//                   queue, so a tile's P (which lies over its S) is consumed
//                   before S is overwritten without a wait in between.
//   warp 9          TMA producer: K and V blocks of a 128-key unit into a ring of
//                   160 KB, one box per block and 64 dimensions, found through
//                   the block table; a block outside the cache reads as zeros.
//   warps 10, 11    walk the items ahead of the others: Q of tile 0, 1 as soon as
//                   the last Q K^T on the one before is done (TMA where the
//                   query heads of a group divide a tile, plain loads otherwise);
//                   warp 10 also publishes the items' extents in shared memory.
// Tensor memory (512 columns): S / P of the tiles, O of the tiles.
//
// P is rounded to the 16-bit type once (V's type: the products take one type);
// the sum is taken over the unrounded values.  That rounding is of the size of
// the output's own, and averages over the keys.
//
// Masks are applied only in units that hold a masked key for some row of the
// warp.  V rows behind the item's last key are zeroed in shared memory before
// the product, so that what lies in the cache there cannot reach it (0 * NaN).
//
// Every wait is bounded; a CTA that gives up waits (bounded) for its own loads
// and products, frees its tensor memory, writes NaN to the rows of its share and
// returns.
#include <mutex>

#include "paged_tc.cuh"

namespace itts {
namespace paged {
namespace {

constexpr int kTileRows = 256, kUnitKeys = 128;
constexpr int kTileThreads = 384;  // three warpgroups: 168 registers a thread at launch ...
constexpr int kSoftmaxRegs = 208;  // ... 208 + 208 + 88 = 3 x 168 after the split
constexpr int kOtherRegs = 88;
constexpr int kTileCtas = 148;
constexpr int kTileItem = 3;  // what an item costs besides its units, in units
constexpr float kGrow = 8.f;  // log2 of the growth of the maximum that is let pass

// A part of an item in this share: units [k0, k0 + n) of the item.
struct Segment {
    int first, rows, k0, n, keys;  // first row of the item in its request, its rows (<= 256), its keys
    int start, pos, kvh;           // first row of the request, position of its row 0, kv head
    int tu[2];                     // units of the segment that tile t (128 rows) has keys in
    int parts;                     // 0: begins and ends here; 1: goes on from another share; n > 1: begins here, n shares
};
constexpr int kSegments = 4;

template <int D>
struct alignas(1024) TileSmem {
    static constexpr int kHalves = D / 64;
    static constexpr int kTileBytes = kUnitKeys * D * 2;  // a K or V tile
    static constexpr int kStages = 160 * 1024 / kTileBytes;
    unsigned char q[2][kTileBytes];
    unsigned char kv[kStages][kTileBytes];
    unsigned long long full[kStages], empty[kStages], q_full[2], q_free[2], s_ready[2], p_ready[2], o_done[2], done;
    unsigned long long seg_full[kSegments], seg_empty[kSegments];
    PlanSmem<kTileThreads> plan;
    Segment seg[kSegments];
    unsigned bad[8];  // per unit (mod 8): blocks that the table does not name
    uint32_t tmem;
    int abort;
};

template <class T>
constexpr uint32_t kKind = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
// Instruction descriptor: D f32, A and B of type T, M = 128, N = n, B K-major or (mn) MN-major.
template <class T>
constexpr uint32_t idesc16(int n, bool mn) {
    return (1u << 4) | (kKind<T> << 7) | (kKind<T> << 10) | (uint32_t(mn) << 16) | (uint32_t(n >> 3) << 17) |
           (uint32_t(128 >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
        : "memory");
}

template <class T>
__device__ __forceinline__ uint32_t pack16(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 2^x of two values on the FMA units: x = n + f with n the nearest whole number
// (read off the low bits of x + 1.5 2^23), 2^f by a polynomial fitted to the
// least largest relative error on [-1/2, 1/2], n added to the exponent.  Degree
// 3 is off by 2^-13 (bf16 rounds to 2^-9), degree 4 by 2^-18 (f16: 2^-12).
// Below -126 the result stays at 2^-126: not for masked keys.
template <class T>
__device__ __forceinline__ float2 exp2_fit(float2 x) {
    const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);
    const float2 neg = make_float2(-1.f, -1.f);
    x = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
    const float2 t = add2(x, magic), f = fma2(add2(t, minus), neg, x);
    const auto both = [](float c) { return make_float2(c, c); };
    float2 p;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        p = fma2(both(0.0551714934f), f, both(0.242610931f));
        p = fma2(p, f, both(0.693260968f));
        p = fma2(p, f, both(0.999928057f));
    } else {
        p = fma2(both(0.00957008637f), f, both(0.0559178516f));
        p = fma2(p, f, both(0.240247443f));
        p = fma2(p, f, both(0.693121791f));
        p = fma2(p, f, both(0.999999285f));
    }
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}
// Of every kFitOf pairs of weights kFit are computed so, the rest by the exponential unit.
constexpr int kFit = 2, kFitOf = 4;

using TileWalk = Walk<kTileRows, kUnitKeys, kTileItem>;
// The segment that begins at the walk's unit.
__device__ __forceinline__ Segment segment(const Attn& a, const TileWalk& w, const Share& sh) {
    Segment s;
    s.first = w.t * kTileRows;
    s.rows = min(kTileRows, w.r.rows - s.first);
    s.k0 = w.k - kTileItem;
    s.n = w.run();
    s.keys = w.r.keys<kTileRows>(a, w.t);
    s.start = w.r.start;
    s.pos = w.r.len - w.r.tokens;
    s.kvh = w.h;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int last = min(s.rows, 128 * (t + 1)) - 1;
        const int seen = min(max(w.r.pos(a, s.first + last) + 1, 0), a.cap);
        s.tu[t] = last < 128 * t ? 0 : min(max(max(1, (seen + kUnitKeys - 1) / kUnitKeys) - s.k0, 0), s.n);
    }
    s.parts = w.parts(sh);
    return s;
}

// NaN for every row of the share: what the CTA leaves when a wait has run out.
template <class T, int D>
__device__ __noinline__ void poison(const Attn& a, const Share& sh) {
    TileWalk w;
    w.start(a, sh);
    const float nan = __int_as_float(0x7fffffff);
    while (w.work()) {
        const Segment g = segment(a, w, sh);
        for (int x = threadIdx.x; x < g.rows * (D / 4); x += kTileThreads) {
            const int row = x / (D / 4), d4 = x % (D / 4);
            if (g.parts == 0)
                store4<T>(out_row<T>(a, g.start, g.first, row, g.kvh) + 4 * d4, make_float4(nan, nan, nan, nan));
            else if (d4 == 0)
                reinterpret_cast<float2*>(part_slot<kTileRows, D>(a, blockIdx.x, g.parts > 1 ? 1 : 0) + kTileRows * D)[row] =
                    make_float2(0.f, nan);
        }
        if (threadIdx.x == 0 && g.parts > 1) put_record(a, blockIdx.x, g.parts, g.kvh, g.rows, g.start, g.first);
        w.advance(a, g.n);
    }
}

template <class T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_attn_tile(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ CUtensorMap map_q, const __grid_constant__ Attn a, int q_tokens) {
    extern __shared__ unsigned char smem_raw[];
    using Smem = TileSmem<D>;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    constexpr int NS = Smem::kStages, kHalves = Smem::kHalves;
    constexpr uint32_t kTileBytes = Smem::kTileBytes, kHalfBytes = kTileBytes / kHalves;
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sm.q_full[t], 1);
            mbar_init(&sm.q_free[t], 1);
            mbar_init(&sm.s_ready[t], 1);
            mbar_init(&sm.p_ready[t], 4);
            mbar_init(&sm.o_done[t], 1);
        }
        for (int x = 0; x < kSegments; ++x) {
            mbar_init(&sm.seg_full[x], 1);
            mbar_init(&sm.seg_empty[x], 10);  // softmax warps, products, Q of tile 1
        }
        mbar_init(&sm.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sm.abort = 0;
    }
    pdl_wait();
    const int units = plan<kTileRows, kUnitKeys, kTileItem, kTileThreads>(a, blockIdx.x, gridDim.x, sm.plan, reinterpret_cast<int*>(sm.kv));
    const Share& sh = sm.plan.share;
    if (threadIdx.x == 0) put_record(a, blockIdx.x, 0, 0, 0, 0, 0);
    if (units == 0) return;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the plan's scratch lies where TMA writes next
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(sm.tmem);
    // columns: S / P of tile t at 128 t, O of tile t at 256 + 128 t

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
        // ---- TMA producer: lane = (block of the unit, 64 dimensions)
        TileWalk w;
        w.start(a, sh);
        const int blocks = kUnitKeys >> a.shift, bl = lane / kHalves, half = lane % kHalves;
        const bool mine = bl < blocks;
        const uint32_t dst = half * kHalfBytes + bl * (128u << a.shift);
        int issued = 0;
        bool ok = true;
        const auto table_id = [&] {  // of this lane's block in the walk's unit
            const long long page = (long long)(w.k - kTileItem) * blocks + bl;
            const bool there = mine && page < (a.cap >> a.shift) && (page << a.shift) < w.r.len;
            return there ? __ldcg(a.table + w.b * a.table_stride + page) : -1;
        };
        bool more = w.work();
        int id = table_id();
        for (int i = 0; more && ok; ++i) {
            const bool named = (unsigned)id < (unsigned)a.c.blocks;
            const unsigned bad = __ballot_sync(0xffffffffu, mine && half == 0 && !named);
            const int block = named ? id : a.c.blocks, head = w.h;
            w.advance(a, 1);
            more = w.work();
            if (more) id = table_id();  // under way while this unit's loads are issued
            if (lane == 0) *reinterpret_cast<volatile unsigned*>(&sm.bad[i & 7]) = bad;
            for (int v = 0; v < 2; ++v) {
                const int x = 2 * i + v, s = x % NS;
                if (x >= NS && !mbar_wait(&sm.empty[s], uint32_t(x / NS + 1) & 1u, &sm.abort)) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_expect(&sm.full[s], kTileBytes);
                __syncwarp();
                if (mine) tma_block(smem_u32(sm.kv[s]) + dst, v ? &map_v : &map_k, 64 * half, head, block, &sm.full[s]);
                issued = x + 1;
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        // loads still in flight land before the CTA may exit
        for (int x = max(0, issued - NS); x < issued; ++x) mbar_wait(&sm.full[x % NS], uint32_t(x / NS) & 1u, nullptr);
    } else if (warp == 8) {
        // ---- products
        uint32_t ph_q[2] = {0, 0}, ph_p[2] = {0, 0};
        bool ok = true;
        const auto scores = [&](int t, int x) {  // S of tile t from the K tile that is x-th in the ring
            const uint32_t q = desc_low(smem_u32(sm.q[t]), 16), k = desc_low(smem_u32(sm.kv[x % NS]), 16);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                const uint32_t o = ((d / 4) * kHalfBytes + (d % 4) * 32u) >> 4;
                mma_ss(tmem + 128u * t, q + o, k + o, idesc16<T>(kUnitKeys, false), d > 0);
            }
        };
        for (int i = 0, x = 0; ok; ++x) {
            ok = uniform(mbar_wait(&sm.seg_full[x % kSegments], uint32_t(x / kSegments) & 1u, &sm.abort));
            if (!ok) break;
            const Segment& sg = sm.seg[x % kSegments];
            const int gn = uniform(sg.n), live0 = uniform(sg.keys - sg.k0 * kUnitKeys);
            const int tu[2] = {uniform(sg.tu[0]), uniform(sg.tu[1])};
            __syncwarp();
            if (elect()) mbar_arrive(&sm.seg_empty[x % kSegments]);
            if (gn == 0) break;
#pragma unroll
            for (int t = 0; t < 2 && ok; ++t)
                if (tu[t] > 0) {
                    ok = uniform(mbar_wait(&sm.q_full[t], ph_q[t], &sm.abort));
                    ph_q[t] ^= 1u;
                }
            ok = ok && uniform(mbar_wait(&sm.full[(2 * i) % NS], uint32_t((2 * i) / NS) & 1u, &sm.abort));
            if (!ok) break;
            tc_after();
            if (elect()) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (tu[t] > 0) {
                        scores(t, 2 * i);
                        tc_commit(&sm.s_ready[t]);
                        if (tu[t] == 1) tc_commit(&sm.q_free[t]);
                    }
                tc_commit(&sm.empty[(2 * i) % NS]);
            }
            __syncwarp();
            for (int j = 0; j < gn && ok; ++j) {
                const int xv = 2 * (i + j) + 1, xk = xv + 1;
                ok = uniform(mbar_wait(&sm.full[xv % NS], uint32_t(xv / NS) & 1u, &sm.abort));
                if (!ok) break;
                const uint32_t v = desc_low(smem_u32(sm.kv[xv % NS]), kHalfBytes);
                const int live = live0 - j * kUnitKeys;
                if (live < kUnitKeys) {  // rows behind the item's last key: zeros, whatever the cache holds
                    for (int x = max(live, 0) * 8 + lane; x < kUnitKeys * 8; x += 32)
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            *reinterpret_cast<uint4*>(sm.kv[xv % NS] + hf * kHalfBytes + x * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                bool have_k = false;
#pragma unroll
                for (int t = 0; t < 2 && ok; ++t) {
                    if (j < tu[t]) {
                        ok = uniform(mbar_wait(&sm.p_ready[t], ph_p[t], &sm.abort));
                        ph_p[t] ^= 1u;
                        if (!ok) break;
                        tc_after();
                        if (elect()) {
#pragma unroll
                            for (int k = 0; k < kUnitKeys / 16; ++k)
                                mma_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * k,
                                       v + k * (2048u >> 4), idesc16<T>(D, true), j > 0 || k > 0);
                            if (j + 1 == tu[t]) tc_commit(&sm.o_done[t]);
                        }
                        __syncwarp();
                    }
                    if (j + 1 < tu[t]) {
                        if (!have_k) {
                            have_k = true;
                            ok = uniform(mbar_wait(&sm.full[xk % NS], uint32_t(xk / NS) & 1u, &sm.abort));
                            if (!ok) break;
                            tc_after();
                        }
                        if (elect()) {
                            scores(t, xk);
                            tc_commit(&sm.s_ready[t]);
                            if (j + 2 == tu[t]) tc_commit(&sm.q_free[t]);
                        }
                        __syncwarp();
                    }
                }
                if (ok && elect()) {
                    tc_commit(&sm.empty[xv % NS]);
                    if (j + 1 < gn) tc_commit(&sm.empty[xk % NS]);
                }
                __syncwarp();
            }
            i += gn;
        }
        if (elect()) {
            tc_commit(&sm.done);  // completes when every product issued above has
            mbar_wait(&sm.done, 0u, nullptr);
        }
        __syncwarp();
    } else {
        // ---- segments and Q: warp 10 + t for tile t
        const int t = warp - 10;
        TileWalk w;
        w.start(a, sh);
        bool ok = true;
        int loads = 0;  // of Q tile t so far
        for (int x = 0; ok; ++x) {
            Segment g;
            if (t == 0) {
                if (x >= kSegments) ok = uniform(mbar_wait(&sm.seg_empty[x % kSegments], uint32_t(x / kSegments + 1) & 1u, &sm.abort));
                if (!ok) break;
                if (w.work())
                    g = segment(a, w, sh);
                else
                    g.n = 0;  // the end
                if (lane == 0) {
                    sm.seg[x % kSegments] = g;
                    mbar_arrive(&sm.seg_full[x % kSegments]);
                    if (g.n > 0 && g.parts > 1) put_record(a, blockIdx.x, g.parts, g.kvh, g.rows, g.start, g.first);
                }
            } else {
                ok = uniform(mbar_wait(&sm.seg_full[x % kSegments], uint32_t(x / kSegments) & 1u, &sm.abort));
                if (!ok) break;
                g = sm.seg[x % kSegments];
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.seg_empty[x % kSegments]);
            }
            if (g.n == 0) break;
            if (g.tu[t] > 0) {
                if (loads > 0) ok = uniform(mbar_wait(&sm.q_free[t], uint32_t(loads - 1) & 1u, &sm.abort));
                if (!ok) break;
                ++loads;
                const int row0 = g.first + 128 * t;
                if (q_tokens > 0) {  // a box of q_tokens tokens and the group's heads is the tile
                    if (lane == 0) {
                        mbar_expect(&sm.q_full[t], kTileBytes);
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            tma_rows(smem_u32(sm.q[t]) + hf * kHalfBytes, &map_q, 64 * hf, g.kvh * a.group,
                                     g.start + over_group(a, row0), &sm.q_full[t]);
                    }
                } else {
                    const uint32_t flip = a.sign < 0.f ? 0x80008000u : 0u;
                    constexpr int kChunks = D / 8;
#pragma unroll 4
                    for (int y = lane; y < 128 * kChunks; y += 32) {
                        const int r = y / kChunks, ch = y % kChunks;
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (128 * t + r < g.rows) {
                            const int tok = over_group(a, row0 + r), hd = (row0 + r) - tok * a.group;
                            v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                                     (long long)(g.start + tok) * a.q_row +
                                                                     (long long)(g.kvh * a.group + hd) * a.q_head) + ch);
                            v = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
                        }
                        *reinterpret_cast<uint4*>(sm.q[t] + (ch / 8) * kHalfBytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.q_full[t]);
                }
            }
            if (t == 0) w.advance(a, g.n);
        }
        // the last load lands before the CTA may exit
        if (loads > 0 && q_tokens > 0) mbar_wait(&sm.q_full[t], uint32_t(loads - 1) & 1u, nullptr);
    }
    } else {
        // ---- softmax: tile t, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = warp >> 2, row = threadIdx.x;
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
        const uint32_t s_col = tmem + lanes + 128u * t, o_col = tmem + lanes + 256u + 128u * t;
        uint32_t ph_s = 0, ph_o = 0;
        bool ok = true;
        for (int i = 0, x = 0;; ++x) {
            if (ok) ok = mbar_wait(&sm.seg_full[x % kSegments], uint32_t(x / kSegments) & 1u, &sm.abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const Segment& g = sm.seg[x % kSegments];
            if (g.n == 0) break;
            const int units = g.tu[t];
            int seen = 0;  // keys of the unit that the row sees
            if (row < g.rows) seen = min(max(g.pos + over_group(a, g.first + row) + 1, 0), a.cap) - g.k0 * kUnitKeys;
            else seen = -g.k0 * kUnitKeys;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < units; ++j, seen -= kUnitKeys) {
                if (ok) ok = mbar_wait(&sm.s_ready[t], ph_s, &sm.abort);
                ok = __all_sync(0xffffffffu, ok);
                ph_s ^= 1u;
                if (!ok) break;
                tc_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_col + 32u * c, s[c]);
                const unsigned bad = *reinterpret_cast<volatile unsigned*>(&sm.bad[(i + j) & 7]);
                const bool masked = __any_sync(0xffffffffu, seen < kUnitKeys) || bad;
                const auto mask = [&](int c, uint32_t (&s)[32]) {  // a bit per key of the chunk: a block is 16 keys or more
                    const int left = seen - 32 * c;
                    uint32_t see = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                    if (bad >> (((32 * c) >> a.shift) * kHalves) & 1u) see &= 0xffff0000u;
                    if (bad >> (((32 * c + 16) >> a.shift) * kHalves) & 1u) see &= 0x0000ffffu;
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (!(see >> x & 1u)) s[x] = 0xff800000u;
                };
                tc_wait_ld(s[0]);
#pragma unroll
                for (int c = 1; c < 4; ++c) tc_wait_ld(s[c]);
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) mask(c, s[c]);
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < 32; x += 2)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        mx[c] = max3(mx[c], __uint_as_float(s[c][x]), __uint_as_float(s[c][x + 1]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
                const bool grow = top > m + kGrow || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : ex2(m - mn);
                    m = mn;
                    l *= f;
                    if (j > 0) {  // the products of the units before are done: this unit's scores came after them
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(o_col + 16u * c, o);
                            tc_wait_ld(o);
#pragma unroll
                            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                            tmem_st16(o_col + 16u * c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : -m;
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 sc = make_float2(a.scale2, a.scale2), rf = make_float2(ref, ref);
                const auto weights = [&](auto fit) {  // P of the unit over its scores, and its sum
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t p[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            float2 y = fma2(make_float2(__uint_as_float(s[c][2 * x]), __uint_as_float(s[c][2 * x + 1])), sc, rf);
                            if (decltype(fit)::value && x % kFitOf < kFit)
                                y = exp2_fit<T>(y);
                            else
                                y = make_float2(ex2(y.x), ex2(y.y));
                            sum[x & 1] = add2(sum[x & 1], y);
                            p[x] = pack16<T>(y.x, y.y);
                        }
                        tmem_st16(s_col + 16u * c, p);  // over scores that this warp has read
                    }
                };
                if (masked)
                    weights(std::false_type());  // a masked weight has to be 0
                else
                    weights(std::true_type());
                l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_ready[t]);
            }
            // the segment's output
            if (units > 0 && ok) {
                ok = mbar_wait(&sm.o_done[t], ph_o, &sm.abort);
                ok = __all_sync(0xffffffffu, ok);
                tc_after();
            }
            if (units > 0) ph_o ^= 1u;
            const bool live = row < g.rows, whole = g.parts == 0;
            float* slot = whole ? nullptr : part_slot<kTileRows, D>(a, blockIdx.x, g.parts > 1 ? 1 : 0);
            T* dst = live && whole ? out_row<T>(a, g.start, g.first, row, g.kvh) : nullptr;
            if (!ok) break;
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (ok && units > 0) {
                    tmem_ld32(o_col + 32u * c, o);
                    tc_wait_ld(o);
                } else {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
                if (!live) continue;
#pragma unroll
                for (int x = 0; x < 32; x += 8) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[x + e]);
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = l == 0.f ? 0.f : y[e] * inv;
                        *reinterpret_cast<uint4*>(dst + 32 * c + x) = make_uint4(
                            pack16<T>(y[0], y[1]), pack16<T>(y[2], y[3]), pack16<T>(y[4], y[5]), pack16<T>(y[6], y[7]));
                    } else {
                        float4* to = reinterpret_cast<float4*>(slot + (size_t)row * D + 32 * c + x);
                        to[0] = make_float4(y[0], y[1], y[2], y[3]);
                        to[1] = make_float4(y[4], y[5], y[6], y[7]);
                    }
                }
            }
            if (!whole && live) reinterpret_cast<float2*>(slot + kTileRows * D)[row] = make_float2(m, l);
            i += g.n;
            tc_before();  // the output has been read out of tensor memory
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.seg_empty[x % kSegments]);
        }
    }
    tc_before();
    __syncthreads();
    if (warp == 8) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (sm.abort) poison<T, D>(a, sh);
}

PFN_cuTensorMapEncodeTiled_v12000 encode() {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

template <class T, int D>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, int q_tokens, const Attn& a,
                   cudaStream_t s) {
    constexpr size_t smem = sizeof(TileSmem<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    cudaError_t e = allow_smem<k_attn_tile<T, D>>(smem);
    if (e != cudaSuccess) return e;
    if ((e = launch_pdl(k_attn_tile<T, D>, kTileCtas, kTileThreads, smem, s, mk, mv, mq, a, q_tokens)) != cudaSuccess) return e;
    return launch_pdl(k_join_rows<T, kTileRows, D>, dim3(kTileCtas, kTileRows / join_rows(D)), kJoinThreads, 0, s, a);
}

}  // namespace

cudaError_t make_block_map(CUtensorMap* map, const itts_paged_cache& c, bool v) {
    const auto fn = encode();
    if (!fn) return cudaErrorNotSupported;
    const int size = c.type == ITTS_PAGED_F32 ? 4 : 2;
    // the stride of a dimension of one is never used, but has to be a legal one
    const auto bytes = [&](long long stride, int n) { return n == 1 ? 16ull : (unsigned long long)(stride * size); };
    const cuuint64_t dims[4] = {cuuint64_t(c.head_dim), cuuint64_t(c.block_size), cuuint64_t(c.heads), cuuint64_t(c.blocks)};
    const cuuint64_t strides[3] = {bytes(v ? c.v_token_stride : c.k_token_stride, c.block_size),
                                   bytes(v ? c.v_head_stride : c.k_head_stride, c.heads),
                                   bytes(v ? c.v_block_stride : c.k_block_stride, c.blocks)};
    const cuuint32_t box[4] = {cuuint32_t(128 / size), cuuint32_t(c.block_size), 1, 1}, one[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = c.type == ITTS_PAGED_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : c.type == ITTS_PAGED_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = fn(map, type, 4, v ? c.v : c.k, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

namespace {
// Tensor map of the query rows: [rows][q_heads][head_dim] at their strides, boxes of `tokens` rows by one group of
// heads x 128 bytes.
cudaError_t make_row_map(CUtensorMap* map, const Attn& a, int tokens) {
    const auto fn = encode();
    if (!fn) return cudaErrorNotSupported;
    const int heads = a.group * a.c.heads;
    const cuuint64_t dims[3] = {cuuint64_t(a.c.head_dim), cuuint64_t(heads), cuuint64_t(a.rows)};
    const cuuint64_t strides[2] = {heads == 1 ? 16ull : cuuint64_t(a.q_head * 2), a.rows == 1 ? 16ull : cuuint64_t(a.q_row * 2)};
    const cuuint32_t box[3] = {64, cuuint32_t(a.group), cuuint32_t(tokens)}, one[3] = {1, 1, 1};
    const CUresult r = fn(map, a.c.type == ITTS_PAGED_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          3, const_cast<void*>(a.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
}  // namespace

size_t tile_workspace_floats(int head_dim) {
    return size_t(2) * kTileCtas * (head_dim == 64 ? part_floats<kTileRows, 64>() : part_floats<kTileRows, 128>());
}

// cudaErrorNotSupported: the cache's strides have no tensor map.
cudaError_t launch_tile(const Attn& a, cudaStream_t s) {
    CUtensorMap mk, mv;
    if (make_block_map(&mk, a.c, false) != cudaSuccess || make_block_map(&mv, a.c, true) != cudaSuccess)
        return cudaErrorNotSupported;
    // Q by TMA: rows are numbered token-major, so a tile is a box of 128 / group tokens by the group's heads
    CUtensorMap mq = mk;
    const int q_tokens = 128 % a.group == 0 && a.sign > 0.f && make_row_map(&mq, a, 128 / a.group) == cudaSuccess
                             ? 128 / a.group
                             : 0;
    const bool wide = a.c.head_dim == 128;
    if (a.c.type == ITTS_PAGED_F16)
        return wide ? launch<__half, 128>(mk, mv, mq, q_tokens, a, s) : launch<__half, 64>(mk, mv, mq, q_tokens, a, s);
    return wide ? launch<__nv_bfloat16, 128>(mk, mv, mq, q_tokens, a, s)
                : launch<__nv_bfloat16, 64>(mk, mv, mq, q_tokens, a, s);
}

}  // namespace paged
}  // namespace itts
