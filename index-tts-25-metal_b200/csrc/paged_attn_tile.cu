// Paged attention of many rows per request (prompt chunks), 16-bit types, on
// the 5th-generation tensor cores.
//
// S = Q K^T and O += P V are tcgen05 products; bound by them and, as closely, by
// the exponentials: 128 rows x 128 keys take 1024 clocks of the tensor core (both
// products, head_dim 128) and 1024 clocks of the SM's exponential units.  A CTA
// works on an item of 256 rows as two tiles of 128 with a softmax warpgroup each.
// P has columns of its own, so the next unit's scores are computed as soon as this
// unit's are read, and the softmax's chain (read the scores, maximum, exponentials,
// write P) does not wait for the products.  To find room in the 512 columns of tensor
// memory a unit is 64 keys with head_dim 128, 128 keys with 64.  Measured per 64 keys
// and both tiles (head_dim 128): 1900 clocks; the exponential unit works 1024 of them,
// the tensor core 1500 (a product of 64 keys takes it as long as one of 128, since
// Q is read again from shared memory), the chain of a tile takes the rest of the
// way.  With P over the scores, units of 128 keys: 3850 for 128.
// The output is rescaled only when the maximum has grown by more than 2^8 (fp16: 2^4)
// since the last time: P stays below that, within the 16-bit types' limits, and the
// division at the end takes the same maximum out again.
// Tried and left, as none was faster: a part of the exponentials by a polynomial on
// the FMA units; weights with the last unit's maximum beside this unit's; two threads
// a row (four softmax warpgroups); the tiles' exponentials in turns or out of step;
// the next scores fetched before P is written.
//
// 384 threads in five roles:
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread per row (no shuffles); writes
//                   the output, or the partial sums, at an item's end.
//   warps 8, 11     issue the products of tile 0, 1: the next unit's scores when this
//                   unit's are read, P V when P is written.  (A wait that is over
//                   and an issue cost a warp 100 clocks and more: one warp for both
//                   tiles was the bound, 2480 clocks for a unit of 64 keys.)
//   warp 9          TMA producer: K and V blocks of a unit into a ring of ten 16 KB
//                   stages, one box per block and 64 dimensions, found through
//                   the block table; a block outside the cache reads as zeros.
//   warp 10         walks the items ahead of the others, publishes their extents in
//                   shared memory and loads Q of the tiles as soon as the last
//                   scores with the one before are done (TMA where the query
//                   heads of a group divide a tile, cp.async otherwise).
// Tensor memory: S of the tiles, P of the tiles, O of the tiles.
//
// P is rounded to the 16-bit type once (V's type: the products take one type);
// the sum is taken over the unrounded values.  That rounding is of the size of the
// output's own at most, and less where the keys' roundings differ.
//
// Masks are applied only in units that hold a masked key for some row of the
// warp.  V rows behind the item's last key are zeroed in shared memory before
// the product, so that what lies in the cache there cannot reach it (0 * NaN).
//
// Every wait is bounded; a CTA that gives up waits (bounded) for its own loads
// and products, frees its tensor memory, writes NaN to the rows of its share and
// returns.
#include <algorithm>
#include <mutex>

#include "paged_tc.cuh"

namespace itts {
namespace paged {
namespace {

constexpr int kTileRows = 256;
// Keys of a unit: 2 S + 2 P + 2 O columns are 3 keys + 2 head_dim <= 512.
template <int D>
constexpr int kUnitOf = D == 128 ? 64 : 128;
constexpr int kTileThreads = 384;
// Registers a thread: 168 at launch (65536 / 384, rounded down to a multiple of 8), then by role.
constexpr int kRegsLaunch = 168, kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + kOtherRegs == 3 * kRegsLaunch && kSoftmaxRegs >= kRegsLaunch && kOtherRegs <= kRegsLaunch,
              "more would wait for ever; inc does not lower, dec does not raise");
constexpr int kTileCtas = 148;
constexpr int kTileItem = 1;  // what an item costs besides its units, in units
// log2 of the growth of the maximum that is let pass.  fp16 has 15 octaves above 1 to share out between it and the
// lift of the weights, which keeps small ones: 2^-25 2^-11 of the maximum is where they end (chunks of 512..1024 rows
// over 1024..8192 keys: 2^8 and no lift 291 us, 2^4 and 2^11 292).
template <class T>
constexpr int kGrow = std::is_same<T, __half>::value ? 4 : 8;
// Keys over which tensor memory sums up an item's output.  The tensor core's accumulation does not round to nearest:
// with 2^20 keys at a stretch the result came out 6e-3 short, with 2^14 1e-4.  Then the sums so far go to the item's
// slot of the workspace, where they are added up in fp32 (148 items of 2^17 keys 2.12 ms at a stretch, 2.18 ms so).
constexpr int kStretch = 1 << 14;

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
    static constexpr int kTileBytes = kUnitOf<D> * D * 2;  // a K or V tile
    static constexpr int kStages = 10;
    static constexpr int kQBytes = 128 * D * 2;
    unsigned char q[2][kQBytes];
    unsigned char kv[kStages][kTileBytes];
    unsigned long long full[kStages], empty[kStages], q_full[2], q_free[2], s_ready[2], s_read[2], p_ready[2], o_done[2], done[2];
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

template <int D>
using TileWalk = Walk<kTileRows, kUnitOf<D>, kTileItem>;
// The segment that begins at the walk's unit.
template <int D>
__device__ __forceinline__ Segment segment(const Attn& a, const TileWalk<D>& w, const Share& sh) {
    constexpr int KU = kUnitOf<D>;
    Segment s;
    s.first = w.t * kTileRows;
    s.rows = min(kTileRows, w.r.rows - s.first);
    s.k0 = w.k - kTileItem;
    s.n = w.run();
    s.keys = w.r.template keys<kTileRows>(a, w.t);
    s.start = w.r.start;
    s.pos = w.r.len - w.r.tokens;
    s.kvh = w.h;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int last = min(s.rows, 128 * (t + 1)) - 1;
        const int seen = min(max(w.r.pos(a, s.first + last) + 1, 0), a.cap);
        s.tu[t] = last < 128 * t ? 0 : min(max(max(1, (seen + KU - 1) / KU) - s.k0, 0), s.n);
    }
    s.parts = w.parts(sh);
    return s;
}

// NaN for every row of the share: what the CTA leaves when a wait has run out.
template <class T, int D>
__device__ __noinline__ void poison(const Attn& a, const Share& sh) {
    TileWalk<D> w;
    w.start(a, sh);
    const float nan = __int_as_float(0x7fffffff);
    while (w.work()) {
        const Segment g = segment<D>(a, w, sh);
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
    constexpr int NS = Smem::kStages, kHalves = Smem::kHalves, KU = kUnitOf<D>, NC = KU / 32;
    constexpr int kFold = kStretch / KU;  // units
    constexpr uint32_t kTileBytes = Smem::kTileBytes, kHalfBytes = kTileBytes / kHalves;
    constexpr uint32_t kQHalf = Smem::kQBytes / kHalves;
    constexpr uint32_t kP = 2 * KU, kO = 3 * KU;  // columns of tensor memory: S of tile t at KU t, P at kP + KU / 2 t, O at kO + D t
    static_assert(kO + 2 * D <= 512, "tensor memory");
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    pdl_trigger();
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (threadIdx.x == 320) {
        prefetch_map(&map_k);
        prefetch_map(&map_v);
        if (q_tokens > 0) prefetch_map(&map_q);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 2);  // both tiles are done with the stage
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sm.q_full[t], 1);
            mbar_init(&sm.q_free[t], 1);
            mbar_init(&sm.s_ready[t], 1);
            mbar_init(&sm.s_read[t], 4);
            mbar_init(&sm.p_ready[t], 4);
            mbar_init(&sm.o_done[t], 1);
        }
        for (int x = 0; x < kSegments; ++x) {
            mbar_init(&sm.seg_full[x], 1);
            mbar_init(&sm.seg_empty[x], 10);  // softmax warps, products of each tile
        }
        mbar_init(&sm.done[0], 1);
        mbar_init(&sm.done[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sm.abort = 0;
    }
    pdl_wait();
    const int units = plan<kTileRows, KU, kTileItem, kTileThreads>(a, blockIdx.x, gridDim.x, sm.plan, reinterpret_cast<long long*>(sm.kv));
    const Share& sh = sm.plan.share;
    if (threadIdx.x == 0) put_record(a, blockIdx.x, 0, 0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the plan's scratch lies where TMA writes next
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(sm.tmem);
    if (units == 0) {
        if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        return;
    }

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
        // ---- TMA producer: lane = (block of the unit, 64 dimensions)
        TileWalk<D> w;
        w.start(a, sh);
        const int shift = min(a.shift, KU == 64 ? 6 : 7);  // tokens of a box: a block, or the unit's part of one
        const int blocks = KU >> shift, bl = lane / kHalves, half = lane % kHalves;
        const bool mine = bl < blocks;
        const uint32_t dst = half * kHalfBytes + bl * (128u << shift);
        int issued = 0;
        bool ok = true;
        const auto table_id = [&] {  // of this lane's block in the walk's unit
            const long long key = (long long)(w.k - kTileItem) * KU + (bl << shift);
            const bool there = mine && key < a.cap && key < w.r.len;
            return there ? __ldcg(a.table + w.b * a.table_stride + (key >> a.shift)) : -1;
        };
        bool more = w.work();
        int id = table_id();
        for (int i = 0; more && ok; ++i) {
            const bool named = (unsigned)id < (unsigned)a.c.blocks;
            const unsigned bad = __ballot_sync(0xffffffffu, mine && half == 0 && !named);
            const int block = named ? id : a.c.blocks, head = w.h;
            const int token = ((w.k - kTileItem) * KU) & ((1 << a.shift) - 1);  // 0 but in blocks of more than a unit
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
                if (mine) tma_block(smem_u32(sm.kv[s]) + dst, v ? &map_v : &map_k, 64 * half, token, head, block, &sm.full[s]);
                issued = x + 1;
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        // loads still in flight land before the CTA may exit
        for (int x = max(0, issued - NS); x < issued; ++x) mbar_wait(&sm.full[x % NS], uint32_t(x / NS) & 1u, nullptr);
    } else if (warp != 10) {
        // ---- products of tile t
        const int t = warp == 8 ? 0 : 1;
        uint32_t ph_q = 0, ph_p = 0;
        bool ok = true;
        const uint32_t s_col = tmem + KU * t, p_col = tmem + kP + KU / 2 * t, o_col = tmem + kO + D * t;
        const auto scores = [&](int x) {  // S from the K tile that is x-th in the ring
            const uint32_t q = desc_low(smem_u32(sm.q[t]), 16), k = desc_low(smem_u32(sm.kv[x % NS]), 16);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
                mma_ss(s_col, q + (((d / 4) * kQHalf + (d % 4) * 32u) >> 4), k + (((d / 4) * kHalfBytes + (d % 4) * 32u) >> 4),
                       idesc16<T>(KU, false), d > 0);
            tc_commit(&sm.s_ready[t]);
            tc_commit(&sm.empty[x % NS]);
        };
        const auto output = [&](int x, bool add) {  // O += P V
            const uint32_t v = desc_low(smem_u32(sm.kv[x % NS]), kHalfBytes);
#pragma unroll
            for (int k = 0; k < KU / 16; ++k)
                mma_ts(o_col, p_col + 8u * k, v + k * (2048u >> 4), idesc16<T>(D, true), add || k > 0);
            tc_commit(&sm.o_done[t]);
            tc_commit(&sm.empty[x % NS]);
        };
        const auto wait = [&](unsigned long long* bar, uint32_t parity) {
            ok = ok && uniform(mbar_wait(bar, parity, &sm.abort));
            return ok;
        };
        const auto full = [&](int x) { return wait(&sm.full[x % NS], uint32_t(x / NS) & 1u); };
        for (int i = 0, x = 0; ok; ++x) {
            if (!wait(&sm.seg_full[x % kSegments], uint32_t(x / kSegments) & 1u)) break;
            const Segment& sg = sm.seg[x % kSegments];
            const int gn = uniform(sg.n), live0 = uniform(sg.keys - sg.k0 * KU), units = uniform(sg.tu[t]);
            __syncwarp();
            if (elect()) mbar_arrive(&sm.seg_empty[x % kSegments]);
            __syncwarp();
            if (gn == 0) break;
            if (units > 0) {
                if (!full(2 * i) || !wait(&sm.q_full[t], ph_q)) break;
                ph_q ^= 1u;
                tc_after();
                if (elect()) {
                    scores(2 * i);
                    if (units == 1) tc_commit(&sm.q_free[t]);
                }
                __syncwarp();
            }
            for (int j = 0; j < units; ++j) {
                const int xv = 2 * (i + j) + 1, xk = xv + 1;
                if (j + 1 < units) {
                    if (!full(xk) || !wait(&sm.s_read[t], ph_p)) break;
                    tc_after();
                    if (elect()) {
                        scores(xk);
                        if (j + 2 == units) tc_commit(&sm.q_free[t]);
                    }
                    __syncwarp();
                }
                if (!full(xv)) break;
                const int live = live0 - j * KU;
                if (live < KU) {  // rows behind the item's last key: zeros (from both tiles), whatever the cache holds
                    for (int y = max(live, 0) * 8 + lane; y < KU * 8; y += 32)
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            *reinterpret_cast<uint4*>(sm.kv[xv % NS] + hf * kHalfBytes + y * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (!wait(&sm.p_ready[t], ph_p)) break;  // after which the unit's scores are read, too
                ph_p ^= 1u;
                tc_after();
                if (elect()) output(xv, (j & (kFold - 1)) != 0);
                __syncwarp();
            }
            for (int j = units; j < gn && ok; ++j) {  // units that none of the tile's rows sees
                const int xk = 2 * (i + j);
                if (!full(xk) || !full(xk + 1)) break;
                if (elect()) {
                    mbar_arrive(&sm.empty[xk % NS]);
                    mbar_arrive(&sm.empty[(xk + 1) % NS]);
                }
                __syncwarp();
            }
            i += gn;
        }
        if (elect()) {
            tc_commit(&sm.done[t]);  // completes when every product issued above has
            mbar_wait(&sm.done[t], 0u, nullptr);
        }
        __syncwarp();
    } else {
        // ---- segments and Q
        TileWalk<D> w;
        w.start(a, sh);
        bool ok = true;
        int loads[2] = {0, 0};  // of Q of tile t so far
        for (int x = 0; ok; ++x) {
            if (x >= kSegments) ok = uniform(mbar_wait(&sm.seg_empty[x % kSegments], uint32_t(x / kSegments + 1) & 1u, &sm.abort, kItemLimitNs));
            if (!ok) break;
            Segment g;
            g.n = 0;  // the end
            if (w.work()) g = segment<D>(a, w, sh);
            if (lane == 0) {
                sm.seg[x % kSegments] = g;
                mbar_arrive(&sm.seg_full[x % kSegments]);
                if (g.n > 0 && g.parts > 1) put_record(a, blockIdx.x, g.parts, g.kvh, g.rows, g.start, g.first);
            }
            if (g.n == 0) break;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (g.tu[t] == 0) continue;
                if (loads[t] > 0) ok = uniform(mbar_wait(&sm.q_free[t], uint32_t(loads[t] - 1) & 1u, &sm.abort, kItemLimitNs));
                if (!ok) break;
                ++loads[t];
                const int row0 = g.first + 128 * t;
                if (q_tokens > 0) {  // a box of q_tokens tokens and the group's heads is the tile
                    if (lane == 0) {
                        mbar_expect(&sm.q_full[t], Smem::kQBytes);
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            tma_rows(smem_u32(sm.q[t]) + hf * kQHalf, &map_q, 64 * hf, g.kvh * a.group,
                                     g.start + over_group(a, row0), &sm.q_full[t]);
                    }
                } else {
                    constexpr int kChunks = D / 8;
                    const auto chunk = [&](int r, int ch) {
                        return sm.q[t] + (ch / 8) * kQHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                    };
#pragma unroll 4
                    for (int y = lane; y < 128 * kChunks; y += 32) {  // all in flight at once: four at a time took 6 us a tile
                        const int r = y / kChunks, ch = y % kChunks;
                        const bool live = 128 * t + r < g.rows;
                        const int tok = over_group(a, row0 + (live ? r : 0)), hd = row0 + (live ? r : 0) - tok * a.group;
                        cp16(smem_u32(chunk(r, ch)), static_cast<const T*>(a.q) + (long long)(g.start + tok) * a.q_row +
                                                         (long long)(g.kvh * a.group + hd) * a.q_head + 8 * ch, live ? 16 : 0);
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    if (a.sign < 0.f)
                        for (int y = lane; y < 128 * kChunks; y += 32) {  // this lane's own
                            uint4& v = *reinterpret_cast<uint4*>(chunk(y / kChunks, y % kChunks));
                            v = make_uint4(v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u);
                        }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.q_full[t]);
                }
            }
            w.advance(a, g.n);
        }
        // the last loads land before the CTA may exit
        if (q_tokens > 0) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (loads[t] > 0) mbar_wait(&sm.q_full[t], uint32_t(loads[t] - 1) & 1u, nullptr);
        }
    }
    } else {
        // ---- softmax: tile t, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = warp >> 2, row = threadIdx.x;
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16;
        const uint32_t s_col = tmem + lanes + KU * t, p_col = tmem + lanes + kP + KU / 2 * t, o_col = tmem + lanes + kO + D * t;
        uint32_t ph_s = 0, ph_o = 0;
        bool ok = true;
        for (int i = 0, x = 0;; ++x) {
            // where its rows have no units in an item, this tile waits for the next one's while the other works on it
            if (ok) ok = mbar_wait(&sm.seg_full[x % kSegments], uint32_t(x / kSegments) & 1u, &sm.abort, kItemLimitNs);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const Segment& g = sm.seg[x % kSegments];
            if (g.n == 0) break;
            const int units = g.tu[t];
            int seen = 0;  // keys of the unit that the row sees
            if (row < g.rows) seen = min(max(g.pos + over_group(a, g.first + row) + 1, 0), a.cap) - g.k0 * KU;
            else seen = -g.k0 * KU;
            float m = -INFINITY, l = 0.f;
            // The item's slot (where it lies in this share alone: the one that a later item may take): earlier sums.
            const auto kept = [&] { return part_slot<kTileRows, D>(a, blockIdx.x, g.parts == 1 ? 0 : 1) + (size_t)row * D; };
            const auto kept_ml = [&] {
                return reinterpret_cast<float2*>(part_slot<kTileRows, D>(a, blockIdx.x, g.parts == 1 ? 0 : 1) + kTileRows * D) + row;
            };
            const auto since = [&](float then) { return then == m ? 1.f : ex2(then - m); };  // both may be -inf
            for (int j = 0; j < units; ++j, seen -= KU) {
                ok = mbar_wait(&sm.s_ready[t], ph_s, &sm.abort, j == 0 ? kItemLimitNs : kWaitLimitNs);
                ok = __all_sync(0xffffffffu, ok);
                ph_s ^= 1u;
                if (!ok) break;
                tc_after();
                // chunks of 32 keys that some row of the warp sees: the others' weights are 0
                const int chunks = min(max((__reduce_max_sync(0xffffffffu, seen) + 31) >> 5, 0), NC);
                uint32_t s[NC][32];
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    if (c < chunks) tmem_ld32(s_col + 32u * c, s[c]);
#pragma unroll
                for (int c = 0; c < NC; ++c) tc_wait_ld(s[c]);
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.s_read[t]);
                const unsigned bad = *reinterpret_cast<volatile unsigned*>(&sm.bad[(i + j) & 7]);
                bool any = true;  // the row sees a key of the unit
                if (__any_sync(0xffffffffu, seen < KU) || bad) {
                    any = false;
                    const int box = min(a.shift, KU == 64 ? 6 : 7);
#pragma unroll
                    for (int c = 0; c < NC; ++c) {  // a bit per key of the chunk: a block is 16 keys or more
                        const int left = seen - 32 * c;
                        uint32_t see = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                        if (bad >> (((32 * c) >> box) * kHalves) & 1u) see &= 0xffff0000u;
                        if (bad >> (((32 * c + 16) >> box) * kHalves) & 1u) see &= 0x0000ffffu;
                        any |= see != 0u;
                        if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(see >> e & 1u)) s[c][e] = 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    if (c < chunks) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                            mx[e / 2 & 3] = max3(mx[e / 2 & 3], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
                    }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2;
                // P V of the unit before is done: P may be overwritten, O rescaled
                if (j > 0) {
                    ok = mbar_wait(&sm.o_done[t], ph_o, &sm.abort);
                    ok = __all_sync(0xffffffffu, ok);
                    ph_o ^= 1u;
                    if (!ok) break;
                    tc_after();
                    if (__builtin_expect((j & (kFold - 1)) == 0, 0)) {
                        const float2 old = j == kFold ? make_float2(m, 0.f) : *kept_ml();
                        const float f = since(old.x);
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(o_col + 16u * c, o);
                            tc_wait_ld(o);
                            float4* to = reinterpret_cast<float4*>(kept() + 16 * c);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float4 y = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                                       __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                                if (j > kFold) {
                                    const float4 z = to[e];
                                    y = make_float4(fmaf(z.x, f, y.x), fmaf(z.y, f, y.y), fmaf(z.z, f, y.z), fmaf(z.w, f, y.w));
                                }
                                to[e] = y;
                            }
                        }
                        *kept_ml() = make_float2(m, fmaf(old.y, f, l));
                        l = 0.f;
                    }
                }
                const bool grow = top > m + float(kGrow<T>) || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : ex2(m - mn);
                    m = mn;
                    l *= f;
                    if (j & (kFold - 1)) {
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(o_col + 16u * c, o);
                            tc_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(o_col + 16u * c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : lift<T>(kGrow<T>) - m;
                const float2 sc = make_float2(a.scale2, a.scale2), rf = make_float2(ref, ref);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    uint32_t p[16];
                    if (c < chunks) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 y = fma2(make_float2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), sc, rf);
                            y = make_float2(ex2(y.x), ex2(y.y));
                            sum[e & 1] = add2(sum[e & 1], y);
                            p[e] = pack2<T>(y.x, y.y);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) p[e] = 0u;
                    }
                    tmem_st16(p_col + 16u * c, p);
                }
                if (any) l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
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
            if (__builtin_expect(units > kFold, 0)) {  // the earlier sums join
                const float2 old = *kept_ml();
                const float f = since(old.x);
                l = fmaf(old.y, f, l);
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16(o_col + 16u * c, o);
                    tc_wait_ld(o);
                    const float* z = kept() + 16 * c;
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(fmaf(z[e], f, __uint_as_float(o[e])));
                    tmem_st16(o_col + 16u * c, o);
                }
                tc_wait_st();
            }
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
                            pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
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
    cudaError_t e = allow_smem<k_attn_tile<T, D>>(smem, kRegsLaunch);
    if (e != cudaSuccess) return e;
    if ((e = launch_pdl(k_attn_tile<T, D>, kTileCtas, kTileThreads, smem, s, mk, mv, mq, a, q_tokens)) != cudaSuccess) return e;
    return launch_pdl(k_join_rows<T, kTileRows, D>, dim3(kTileCtas, kTileRows / join_rows(D)), kJoinThreads, 0, s, a);
}

}  // namespace

cudaError_t make_block_map(CUtensorMap* map, const itts_paged_cache& c, bool v, int tokens) {
    const auto fn = encode();
    if (!fn) return cudaErrorNotSupported;
    const int size = c.type == ITTS_PAGED_F32 ? 4 : 2;
    // the stride of a dimension of one is never used, but has to be a legal one
    const auto bytes = [&](long long stride, int n) { return n == 1 ? 16ull : (unsigned long long)(stride * size); };
    // a map does not repeat a dimension
    const auto repeats = [](long long stride, int n) { return n > 1 && stride == 0; };
    if (repeats(v ? c.v_token_stride : c.k_token_stride, c.block_size) ||
        repeats(v ? c.v_head_stride : c.k_head_stride, c.heads) || repeats(v ? c.v_block_stride : c.k_block_stride, c.blocks))
        return cudaErrorNotSupported;
    const cuuint64_t dims[4] = {cuuint64_t(c.head_dim), cuuint64_t(c.block_size), cuuint64_t(c.heads), cuuint64_t(c.blocks)};
    const cuuint64_t strides[3] = {bytes(v ? c.v_token_stride : c.k_token_stride, c.block_size),
                                   bytes(v ? c.v_head_stride : c.k_head_stride, c.heads),
                                   bytes(v ? c.v_block_stride : c.k_block_stride, c.blocks)};
    const cuuint32_t box[4] = {cuuint32_t(128 / size), cuuint32_t(std::min(c.block_size, tokens)), 1, 1}, one[4] = {1, 1, 1, 1};
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
    if ((heads > 1 && a.q_head == 0) || (a.rows > 1 && a.q_row == 0)) return cudaErrorNotSupported;
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
    const int unit = a.c.head_dim == 128 ? kUnitOf<128> : kUnitOf<64>;
    if (make_block_map(&mk, a.c, false, unit) != cudaSuccess || make_block_map(&mv, a.c, true, unit) != cudaSuccess)
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
