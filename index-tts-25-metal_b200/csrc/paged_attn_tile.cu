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
// 320 threads in four roles:
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread per row (no shuffles).  Loads
//                   its 128 scores from tensor memory, keeps the running maximum
//                   and sum, writes P in 16 bits over the scores.  The output is
//                   rescaled only when the maximum has grown by 2^8 or more
//                   since the last time (P then stays below 2^8, far from
//                   the 16-bit types' limits, and the division at the end
//                   takes the same maximum out again).  Also loads Q into shared
//                   memory at an item's start and writes the output at its end.
//   warp 8          issues the products (one lane): per unit and tile P V of this
//                   unit, then Q K^T of the next, in that order into the same
//                   queue, so a tile's P (which lies over its S) is consumed
//                   before S is overwritten without a wait in between.
//   warp 9          TMA producer: K and V blocks of a 128-key unit into a ring of
//                   160 KB, one box per block and 64 dimensions, found through
//                   the block table; a block outside the cache reads as zeros.
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
// Every wait is bounded; a CTA that gives up writes NaN to the rows that it did
// not finish, waits (bounded) for its own loads and products, frees its tensor
// memory and returns.
#include <mutex>

#include "paged_tc.cuh"

namespace itts {
namespace paged {
namespace {

constexpr int kTileRows = 256, kUnitKeys = 128;
constexpr int kTileThreads = 320;
constexpr int kTileCtas = 148;
constexpr float kGrow = 8.f;  // log2 of the growth of the maximum that is let pass

template <int D>
struct alignas(1024) TileSmem {
    static constexpr int kHalves = D / 64;
    static constexpr int kTileBytes = kUnitKeys * D * 2;  // a K or V tile
    static constexpr int kStages = 160 * 1024 / kTileBytes;
    unsigned char q[2][kTileBytes];
    unsigned char kv[kStages][kTileBytes];
    unsigned long long full[kStages], empty[kStages], q_full[2], s_ready[2], p_ready[2], o_done[2], done;
    PlanSmem<kTileThreads> plan;
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

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(acc)
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

// A part of an item in this share: units [k0, k0 + n) of the item.
struct Segment {
    int first, rows, k0, n, keys;  // first row of the item in its request, its rows (<= 256), its keys
    bool begun, whole;             // begins here; begins and ends here
    // Units of the segment that tile t (128 rows) has keys in.
    __device__ __forceinline__ int tile_units(const Attn& a, const Request& r, int t) const {
        const int last = min(rows, 128 * (t + 1)) - 1;
        if (last < 128 * t) return 0;
        const int seen = min(max(r.pos(a, first + last) + 1, 0), a.cap);
        return min(max(max(1, (seen + kUnitKeys - 1) / kUnitKeys) - k0, 0), n);
    }
};
using TileWalk = Walk<kTileRows, kUnitKeys>;
__device__ __forceinline__ Segment segment(const Attn& a, const TileWalk& w, long long left) {
    Segment s;
    s.first = w.t * kTileRows;
    s.rows = min(kTileRows, w.r.rows - s.first);
    s.k0 = w.k;
    s.n = int(min((long long)(w.nk - w.k), left));
    s.keys = w.r.keys<kTileRows>(a, w.t);
    s.begun = w.k == 0;
    s.whole = s.begun && s.n == w.nk;
    return s;
}

template <class T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_attn_tile(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ Attn a) {
    extern __shared__ unsigned char smem_raw[];
    using Smem = TileSmem<D>;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    constexpr int NS = Smem::kStages, kHalves = Smem::kHalves;
    constexpr uint32_t kTileBytes = Smem::kTileBytes, kHalfBytes = kTileBytes / kHalves;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sm.q_full[t], 4);
            mbar_init(&sm.s_ready[t], 1);
            mbar_init(&sm.p_ready[t], 4);
            mbar_init(&sm.o_done[t], 1);
        }
        mbar_init(&sm.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sm.abort = 0;
    }
    pdl_wait();
    const Share sh = plan<kTileRows, kUnitKeys, kTileThreads>(a, blockIdx.x, gridDim.x, sm.plan);
    if (threadIdx.x == 0) put_record(a, blockIdx.x, 0, 0, 0, 0, 0);
    const int n = int(sh.u1 - sh.u0);
    if (n == 0) return;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = sm.tmem;
    // columns: S / P of tile t at 128 t, O of tile t at 256 + 128 t

    TileWalk w;
    w.start(a, sh);

    if (warp == 9) {
        // ---- TMA producer: lane = (block of the unit, 64 dimensions)
        const int blocks = kUnitKeys >> a.shift, bl = lane / kHalves, half = lane % kHalves;
        const bool mine = bl < blocks;
        const uint32_t dst = half * kHalfBytes + bl * (128u << a.shift);
        int issued = 0;
        bool ok = true;
        const auto table_id = [&] {  // of this lane's block in the walk's unit
            const long long page = (long long)w.k * blocks + bl;
            const bool there = mine && page < (a.cap >> a.shift) && (page << a.shift) < w.r.len;
            return there ? __ldcg(a.table + w.b * a.table_stride + page) : -1;
        };
        int id = table_id();
        for (int i = 0; i < n && ok; ++i) {
            const bool named = (unsigned)id < (unsigned)a.c.blocks;
            const unsigned bad = __ballot_sync(0xffffffffu, mine && half == 0 && !named);
            const int block = named ? id : a.c.blocks, head = w.h;
            if (i + 1 < n) {  // the next unit's entry is under way while this one's loads are issued
                if (++w.k == w.nk) w.next(a);
                id = table_id();
            }
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
            const uint32_t q = smem_u32(sm.q[t]), k = smem_u32(sm.kv[x % NS]);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                const uint32_t o = (d / 4) * kHalfBytes + (d % 4) * 32u;
                mma_ss(tmem + 128u * t, desc_sw128(q + o, 16), desc_sw128(k + o, 16), idesc16<T>(kUnitKeys, false), d > 0);
            }
        };
        for (int i = 0; i < n && ok;) {
            const Segment g = segment(a, w, n - i);
            int tu[2];
            for (int t = 0; t < 2; ++t) tu[t] = g.tile_units(a, w.r, t);
            for (int t = 0; t < 2 && ok; ++t)
                if (tu[t] > 0) {
                    ok = mbar_wait(&sm.q_full[t], ph_q[t], &sm.abort);
                    ph_q[t] ^= 1u;
                }
            ok = ok && mbar_wait(&sm.full[(2 * i) % NS], uint32_t((2 * i) / NS) & 1u, &sm.abort);
            if (!ok) break;
            tc_after();
            if (lane == 0) {
                for (int t = 0; t < 2; ++t)
                    if (tu[t] > 0) {
                        scores(t, 2 * i);
                        tc_commit(&sm.s_ready[t]);
                    }
                tc_commit(&sm.empty[(2 * i) % NS]);
            }
            __syncwarp();
            for (int j = 0; j < g.n && ok; ++j) {
                const int xv = 2 * (i + j) + 1, xk = xv + 1;
                ok = mbar_wait(&sm.full[xv % NS], uint32_t(xv / NS) & 1u, &sm.abort);
                if (!ok) break;
                const uint32_t v = smem_u32(sm.kv[xv % NS]);
                const int live = g.keys - (g.k0 + j) * kUnitKeys;
                if (live < kUnitKeys) {  // rows behind the item's last key: zeros, whatever the cache holds
                    for (int x = max(live, 0) * 8 + lane; x < kUnitKeys * 8; x += 32)
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            *reinterpret_cast<uint4*>(sm.kv[xv % NS] + hf * kHalfBytes + x * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                bool have_k = false;
                for (int t = 0; t < 2 && ok; ++t) {
                    if (j < tu[t]) {
                        ok = mbar_wait(&sm.p_ready[t], ph_p[t], &sm.abort);
                        ph_p[t] ^= 1u;
                        if (!ok) break;
                        tc_after();
                        if (lane == 0) {
#pragma unroll
                            for (int k = 0; k < kUnitKeys / 16; ++k)
                                mma_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * k,
                                       desc_sw128(v + k * 2048u, kHalfBytes), idesc16<T>(D, true), j > 0 || k > 0);
                            if (j + 1 == tu[t]) tc_commit(&sm.o_done[t]);
                        }
                        __syncwarp();
                    }
                    if (j + 1 < tu[t]) {
                        if (!have_k) {
                            have_k = true;
                            ok = mbar_wait(&sm.full[xk % NS], uint32_t(xk / NS) & 1u, &sm.abort);
                            if (!ok) break;
                            tc_after();
                        }
                        if (lane == 0) {
                            scores(t, xk);
                            tc_commit(&sm.s_ready[t]);
                        }
                        __syncwarp();
                    }
                }
                if (ok && lane == 0) {
                    tc_commit(&sm.empty[xv % NS]);
                    if (j + 1 < g.n) tc_commit(&sm.empty[xk % NS]);
                }
                __syncwarp();
            }
            i += g.n;
            if (i < n) {
                w.k += g.n - 1;  // to the item's last unit, and over it
                w.next(a);
            }
        }
        if (lane == 0) {
            tc_commit(&sm.done);  // completes when every product issued above has
            mbar_wait(&sm.done, 0u, nullptr);
        }
        __syncwarp();
    } else {
        // ---- softmax: tile t, a thread per row
        const int t = warp >> 2, row = 128 * t + (threadIdx.x & 127), wl = threadIdx.x & 127;
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
        const uint32_t s_col = tmem + lanes + 128u * t, o_col = tmem + lanes + 256u + 128u * t;
        uint32_t ph_s = 0, ph_o = 0;
        bool ok = true;
        for (int i = 0; i < n;) {
            const Segment g = segment(a, w, n - i);
            const int units = g.tile_units(a, w.r, t);
            const int lim = row < g.rows ? min(max(w.r.pos(a, g.first + row) + 1, 0), a.cap) : 0;
            if (units > 0) {
                // Q: four warps, 16-byte chunks of consecutive rows' head_dim
                const uint32_t flip = a.sign < 0.f ? 0x80008000u : 0u;
                constexpr int kChunks = D / 8;
#pragma unroll 4
                for (int x = wl; x < 128 * kChunks; x += 128) {
                    const int r = x / kChunks, ch = x % kChunks, rr = 128 * t + r;
                    uint4 y = make_uint4(0, 0, 0, 0);
                    if (rr < g.rows) {
                        const int tok = (g.first + rr) / a.group, hd = (g.first + rr) - tok * a.group;
                        y = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                                 (long long)(w.r.start + tok) * a.q_row +
                                                                 (long long)(w.h * a.group + hd) * a.q_head) + ch);
                        y = make_uint4(y.x ^ flip, y.y ^ flip, y.z ^ flip, y.w ^ flip);
                    }
                    *reinterpret_cast<uint4*>(sm.q[t] + (ch / 8) * kHalfBytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = y;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_before();  // the last item's output has been read out of tensor memory
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.q_full[t]);
            }
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < units; ++j) {
                if (ok) ok = mbar_wait(&sm.s_ready[t], ph_s, &sm.abort);
                ok = __all_sync(0xffffffffu, ok);
                ph_s ^= 1u;
                if (!ok) break;
                tc_after();
                uint32_t s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_col + 32u * c, s, 32 * c);
                tc_wait_ld();
                const int seen = lim - (g.k0 + j) * kUnitKeys;
                const unsigned bad = *reinterpret_cast<volatile unsigned*>(&sm.bad[(i + j) & 7]);
                if (__any_sync(0xffffffffu, seen < kUnitKeys) || bad) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        if (c >= seen || (bad >> ((c >> a.shift) * kHalves) & 1u)) s[c] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
                const bool first = j == 0;
                const bool grow = top > m + kGrow || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : ex2(m - mn);
                    m = mn;
                    l *= f;
                    if (!first) {  // the products of the units before are done: this unit's scores came after them
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(o_col + 32u * c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                            tmem_st32(o_col + 32u * c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : -m;
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 sc = make_float2(a.scale2, a.scale2), rf = make_float2(ref, ref);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t p[32];
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        const int e = 64 * c + 2 * x;
                        float2 y = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sc, rf);
                        y = make_float2(ex2(y.x), ex2(y.y));
                        sum[x & 1] = make_float2(sum[x & 1].x + y.x, sum[x & 1].y + y.y);
                        p[x] = pack16<T>(y.x, y.y);
                    }
                    tmem_st32(s_col + 32u * c, p);
                }
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
            const bool live = row < g.rows;
            float* slot = g.whole ? nullptr : part_slot<kTileRows, D>(a, blockIdx.x, g.begun ? 1 : 0);
            T* dst = live && g.whole ? out_row<T>(a, w.r.start, g.first, row, w.h) : nullptr;
            if (!ok) l = __int_as_float(0x7fffffff);
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (ok && units > 0) {
                    tmem_ld32(o_col + 32u * c, o);
                    tc_wait_ld();
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
                    if (g.whole) {
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
            if (!g.whole) {
                if (live) reinterpret_cast<float2*>(slot + kTileRows * D)[row] = make_float2(m, l);
                if (g.begun && threadIdx.x == 0)
                    put_record(a, blockIdx.x, cta_of(sh, sh.u0 + i + w.nk - 1) - int(blockIdx.x) + 1, w.h, g.rows, w.r.start,
                               g.first);
            }
            i += g.n;
            if (i < n) {
                w.k += g.n - 1;
                w.next(a);
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == 8) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
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
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mv, const Attn& a, cudaStream_t s) {
    constexpr size_t smem = sizeof(TileSmem<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    cudaError_t e = cudaFuncSetAttribute(k_attn_tile<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    if ((e = launch_pdl(k_attn_tile<T, D>, kTileCtas, kTileThreads, smem, s, mk, mv, a)) != cudaSuccess) return e;
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

size_t tile_workspace_floats(int head_dim) {
    return size_t(2) * kTileCtas * (head_dim == 64 ? part_floats<kTileRows, 64>() : part_floats<kTileRows, 128>());
}

// cudaErrorNotSupported: the cache's strides have no tensor map.
cudaError_t launch_tile(const Attn& a, cudaStream_t s) {
    CUtensorMap mk, mv;
    if (make_block_map(&mk, a.c, false) != cudaSuccess || make_block_map(&mv, a.c, true) != cudaSuccess)
        return cudaErrorNotSupported;
    const bool wide = a.c.head_dim == 128;
    if (a.c.type == ITTS_PAGED_F16) return wide ? launch<__half, 128>(mk, mv, a, s) : launch<__half, 64>(mk, mv, a, s);
    return wide ? launch<__nv_bfloat16, 128>(mk, mv, a, s) : launch<__nv_bfloat16, 64>(mk, mv, a, s);
}

}  // namespace paged
}  // namespace itts
