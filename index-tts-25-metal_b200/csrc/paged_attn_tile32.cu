// Paged attention of many rows per request (prompt chunks), fp32, on the
// 5th-generation tensor cores.
//
// Every fp32 operand x is taken as three bf16 words, x = h + m + l with h =
// rn(x), m = rn(x - h), l = rn(x - h - m): 8 bits each, so the rest is below
// 2^-26 |x| and the fp32 exponent range is kept.  A product is the six bf16
// products hh + hm + mh + hl + mm + lh (what is dropped is below 2^-26 |x y|),
// the small ones first, so that the tensor core's accumulation rounds at their
// scale until the last.  Six bf16 products cost what three TF32 products cost
// and need no other layout than the 16-bit kernel's: V is read as it lies
// (keys by dimensions), which 32-bit operands are not.  CUDA cores would need
// five times as long.
//
// Bound by the products: a unit of 128 rows x 64 keys (head_dim 128) takes 3072
// clocks.  640 threads in five warpgroups:
//   0     softmax: a thread per row.  Puts Q's three words into tensor memory at an
//         item's start; per unit reads the scores, updates maximum and sum, writes
//         P's three words over them.
//   1     output: a thread per row, head_dim fp32 registers.  Adds every
//         unit's P V (drained from tensor memory, rounded to nearest) to the running
//         output, rescaled; divides and writes it at the item's end.
//   2, 3  K and V: load blocks (found through the block table) into registers a
//         unit ahead, split them and write the words to shared memory, two stages
//         of 48 KB each for K and V.  What is behind the item's keys or in a bad
//         block is not read: zeros.
//   4     warp 16 issues the products; warps 17 and 18 walk the items and publish
//         in shared memory their extents and where their units' keys lie.
// Tensor memory: Q (three words), two buffers of scores / P, O.  With two score
// buffers Q K^T of unit j + 2 follows P V of unit j in the queue, so the tensor
// core has work while the softmax of j + 1 runs, and O is drained meanwhile.
//
// Every wait is bounded; a CTA that gives up waits (bounded) for its own
// products, frees its tensor memory, writes NaN to the rows of its share and
// returns.
#include "paged_tc.cuh"

namespace itts {
namespace paged {
namespace {

constexpr int kRows32 = 128, kUnit32 = 64;
constexpr int kThreads32 = 640;
constexpr int kCtas32 = 148;
constexpr int kItem32 = 3;  // what an item costs besides its units, in units
// Registers a thread: 96 at launch (65536 / 640, rounded down to a multiple of 8), then by role.  K and V with 80 and
// the softmax with 112 was 8% slower.
constexpr int kRegsLaunch = 96, kRegsSoftmax = 104, kRegsOut = 160, kRegsSplit = 88, kRegsIssue = 40;
static_assert(kRegsSoftmax + kRegsOut + 2 * kRegsSplit + kRegsIssue == 5 * kRegsLaunch, "more would wait for ever");
static_assert(kRegsSoftmax >= kRegsLaunch && kRegsOut >= kRegsLaunch, "setmaxnreg.inc does not lower");
static_assert(kRegsSplit <= kRegsLaunch && kRegsIssue <= kRegsLaunch, "setmaxnreg.dec does not raise");
constexpr int kSegments32 = 4;
// Units of a segment at most: a stretch over which a row's sums run on.  Every addition is off by up to 2^-24 of the
// sum, one way if the addends are alike: over 2^19 keys, one of them 17 nats ahead, the others' share came out 2.5e-4
// wrong (1.1e-5 so).  A longer part of an item is several segments, whose sums meet in the item's slot of the workspace;
// each loads Q again (20 requests of 60 rows over 20000 keys 1.23 ms either way).
constexpr int kStretch32 = 256;

struct Segment32 {
    int first, rows, k0, n;  // first row of the item in its request, its rows (<= 128), first unit, units
    int start, pos, kvh;     // first row of the request, position of its row 0, kv head
    int parts;               // 0: begins and ends here; 1: goes on from another share; n > 1: begins here, n shares
    bool later, more;        // segments of the item in this share come before, come after it
};

// Where the keys of a unit lie.
struct Unit32 {
    int ids[kUnit32 / 16];  // block of 16 keys, -1: none that the table names
    int keys, tok, kvh;     // keys left in the item, token of the first in its block, kv head (-1: no unit, the end)
};
constexpr int kUnits32 = 8;

template <int D>
struct alignas(1024) Smem32 {
    static constexpr int kWord = kUnit32 * D * 2;  // one word of a K or V tile
    unsigned char k[2][3][kWord];
    unsigned char v[2][3][kWord];
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], s_ready[2], p_ready[2], f_ready[4];
    unsigned long long q_full, o_done, o_free, done;
    unsigned long long seg_full[kSegments32], seg_empty[kSegments32], unit_full[kUnits32], unit_empty[kUnits32];
    Unit32 unit[kUnits32];
    float2 ml[4][kRows32];  // of unit j at j % 4: running maximum and sum,
    float f[4][kRows32];    // and what they rescale the output by
    float4 turn[4][32 * 8];  // per softmax warp: 32 dimensions of its 32 rows of Q, on their way from lanes along a row
                             // to a lane per row
    Segment32 seg[kSegments32];
    unsigned bad[4][kUnit32 / 16];  // per unit (mod 4) and 16 keys: a block that the table does not name
    PlanSmem<kThreads32> plan;
    uint32_t tmem;
    int abort;
};

using Walk32 = Walk<kRows32, kUnit32, kItem32>;

__device__ __forceinline__ Segment32 segment32(const Attn& a, const Walk32& w, const Share& sh) {
    Segment32 s;
    s.first = w.t * kRows32;
    s.rows = min(kRows32, w.r.rows - s.first);
    s.k0 = w.k - kItem32;
    s.n = w.run();
    s.start = w.r.start;
    s.pos = w.r.len - w.r.tokens;
    s.kvh = w.h;
    s.parts = w.parts(sh);
    s.later = s.more = false;
    return s;
}

// Instruction descriptor: D f32, A and B bf16, M = 128, N = n, B K-major or (mn) MN-major.
constexpr uint32_t idesc32(int n, bool mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ts32(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "r"(kDescHigh)
        : "memory");
}
// The products of a pair of operands, small ones first: words (of A, of B).
__host__ __device__ constexpr int word_a(int p) { return p == 0 ? 2 : p == 2 || p == 3 ? 1 : 0; }
__host__ __device__ constexpr int word_b(int p) { return p == 1 ? 2 : p == 2 || p == 4 ? 1 : 0; }

// Two values as three bf16 words each, packed.
__device__ __forceinline__ void split3(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
    const auto pack = [](float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    };
    const float2 minus = make_float2(-1.f, -1.f);
    h = pack(x, y);
    float2 r = fma2(make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)), minus, make_float2(x, y));
    m = pack(r.x, r.y);
    r = fma2(make_float2(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)), minus, r);
    l = pack(r.x, r.y);
}

template <int D>
__device__ __noinline__ void poison32(const Attn& a, const Share& sh) {
    Walk32 w;
    w.start(a, sh);
    const float nan = __int_as_float(0x7fffffff);
    while (w.work()) {
        const Segment32 g = segment32(a, w, sh);
        for (int x = threadIdx.x; x < g.rows * (D / 4); x += kThreads32) {
            const int row = x / (D / 4), d4 = x % (D / 4);
            if (g.parts == 0)
                store4<float>(out_row<float>(a, g.start, g.first, row, g.kvh) + 4 * d4, make_float4(nan, nan, nan, nan));
            else if (d4 == 0)
                reinterpret_cast<float2*>(part_slot<kRows32, D>(a, blockIdx.x, g.parts > 1 ? 1 : 0) + kRows32 * D)[row] =
                    make_float2(0.f, nan);
        }
        if (threadIdx.x == 0 && g.parts > 1) put_record(a, blockIdx.x, g.parts, g.kvh, g.rows, g.start, g.first);
        w.advance(a, g.n);
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads32, 1) k_attn_tile32(const __grid_constant__ Attn a) {
    extern __shared__ unsigned char smem_raw[];
    using Smem = Smem32<D>;
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023));
    constexpr uint32_t kWord = Smem::kWord, kHalf = kUnit32 * 128;  // bytes of 64 dimensions of a word's tile
    // tensor memory columns
    constexpr uint32_t kQ = 0, kQWord = D / 2, kS = 3 * kQWord, kSBuf = 96, kPWord = 32, kO = kS + 2 * kSBuf;
    static_assert(kO + D <= 512, "tensor memory");
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, wg = warp >> 2;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.k_full[s], 8);
            mbar_init(&sm.k_empty[s], 1);
            mbar_init(&sm.v_full[s], 8);
            mbar_init(&sm.v_empty[s], 1);
            mbar_init(&sm.s_ready[s], 1);
            mbar_init(&sm.p_ready[s], 4);
        }
        for (int s = 0; s < 4; ++s) mbar_init(&sm.f_ready[s], 4);
        for (int s = 0; s < kSegments32; ++s) {
            mbar_init(&sm.seg_full[s], 1);
            mbar_init(&sm.seg_empty[s], 9);  // softmax and output warps, products
        }
        for (int s = 0; s < kUnits32; ++s) {
            mbar_init(&sm.unit_full[s], 1);
            mbar_init(&sm.unit_empty[s], 8);
        }
        mbar_init(&sm.q_full, 4);
        mbar_init(&sm.o_done, 1);
        mbar_init(&sm.o_free, 4);
        mbar_init(&sm.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sm.abort = 0;
    }
    pdl_wait();
    const int units = plan<kRows32, kUnit32, kItem32, kThreads32>(a, blockIdx.x, gridDim.x, sm.plan, reinterpret_cast<long long*>(sm.k));
    const Share& sh = sm.plan.share;
    if (threadIdx.x == 0) put_record(a, blockIdx.x, 0, 0, 0, 0, 0);
    if (units == 0) return;
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = uniform(sm.tmem);
    const uint32_t lanes = tmem + (uint32_t(32 * (warp & 3)) << 16);  // this warp's lanes of tensor memory

    if (wg == 0) {
        // ---- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int row = threadIdx.x;
        bool ok = true;
        for (int i = 0, x = 0;; ++x) {
            ok = __all_sync(0xffffffffu, mbar_wait(&sm.seg_full[x % kSegments32], uint32_t(x / kSegments32) & 1u, &sm.abort));
            if (!ok) break;
            const Segment32& g = sm.seg[x % kSegments32];
            if (g.n == 0) break;
            int seen = -g.k0 * kUnit32;  // keys of the unit that the row sees
            const bool live = row < g.rows;
            {
                if (live) seen += min(max(g.pos + over_group(a, g.first + row) + 1, 0), a.cap);
                // Q, every product with the one before being done (the last unit's scores were read).  Eight lanes
                // load 128 bytes of a row (a lane per row would fetch every sector twice: with 200 KB of it shared
                // memory leaves no cache to speak of), and the rows turn in shared memory.
                const int r8 = lane >> 3, c8 = lane & 7;
                const float* base[8];  // of rows r8, r8 + 4, ..
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int rr = 32 * warp + 4 * e + r8, at = g.first + rr, tk = over_group(a, at);
                    base[e] = rr < g.rows ? static_cast<const float*>(a.q) + (long long)(g.start + tk) * a.q_row +
                                                (long long)(g.kvh * a.group + at - tk * a.group) * a.q_head
                                          : nullptr;
                }
                float4 y[8];
                const auto load = [&](int c) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[e] = base[e] ? __ldg(reinterpret_cast<const float4*>(base[e]) + 8 * c + c8) : make_float4(0.f, 0.f, 0.f, 0.f);
                };
                load(0);
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) sm.turn[warp][(4 * e + r8) * 8 + (c8 ^ ((4 * e + r8) & 7))] = y[e];
                    __syncwarp();
                    if (c + 1 < D / 32) load(c + 1);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t h[8], m[8], l[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float4 z = sm.turn[warp][lane * 8 + ((4 * k + e) ^ (lane & 7))];
                            split3(z.x * a.sign, z.y * a.sign, h[2 * e], m[2 * e], l[2 * e]);
                            split3(z.z * a.sign, z.w * a.sign, h[2 * e + 1], m[2 * e + 1], l[2 * e + 1]);
                        }
                        const uint32_t col = lanes + kQ + 16u * c + 8u * k;
                        tmem_st8(col, h);
                        tmem_st8(col + kQWord, m);
                        tmem_st8(col + 2 * kQWord, l);
                    }
                }
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.q_full);
            }
            float m = -INFINITY, l = 0.f;
            const int units = g.n;
            for (int j = 0; j < units; ++j, seen -= kUnit32) {
                const int u = i + j;
                ok = __all_sync(0xffffffffu, mbar_wait(&sm.s_ready[u & 1], uint32_t(u >> 1) & 1u, &sm.abort));
                if (!ok) break;
                tc_after();
                const uint32_t buf = lanes + kS + kSBuf * (u & 1);
                uint32_t s[2][32];
                tmem_ld32(buf, s[0]);
                tmem_ld32(buf + 32u, s[1]);
                tc_wait_ld(s[0]);
                tc_wait_ld(s[1]);
                const volatile unsigned* b = sm.bad[u & 3];
                const uint4 bad = make_uint4(b[0], b[1], b[2], b[3]);
                if (__any_sync(0xffffffffu, seen < kUnit32) || (bad.x | bad.y | bad.z | bad.w)) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int left = seen - 32 * c;
                        uint32_t see = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                        if (c ? bad.z : bad.x) see &= 0xffff0000u;
                        if (c ? bad.w : bad.y) see &= 0x0000ffffu;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(see >> e & 1u)) s[c][e] = 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; ++e)
#pragma unroll
                    for (int c = 0; c < 2; ++c) mx[2 * c + (e & 1)] = fmaxf(mx[2 * c + (e & 1)], __uint_as_float(s[c][e]));
                const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2);
                const float ref = mn == -INFINITY ? 0.f : mn, f = ex2(m - ref);
                m = mn;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t ph[16], pm[16], pl[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float y0 = ex2(fmaf(__uint_as_float(s[c][2 * e]), a.scale2, -ref));
                        const float y1 = ex2(fmaf(__uint_as_float(s[c][2 * e + 1]), a.scale2, -ref));
                        sum[2 * (e & 1)] += y0;
                        sum[2 * (e & 1) + 1] += y1;
                        split3(y0, y1, ph[e], pm[e], pl[e]);
                    }
                    tmem_st16(buf + 16u * c, ph);
                    tmem_st16(buf + kPWord + 16u * c, pm);
                    tmem_st16(buf + 2 * kPWord + 16u * c, pl);
                }
                l = l * f + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                sm.f[u & 3][row] = f;
                sm.ml[u & 3][row] = make_float2(m, l);
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.p_ready[u & 1]);
                    mbar_arrive(&sm.f_ready[u & 3]);
                }
            }
            if (!ok) break;
            i += units;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.seg_empty[x % kSegments32]);
        }
    } else if (wg == 1) {
        // ---- output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsOut));
        const int row = threadIdx.x - 128;
        bool ok = true;
        for (int i = 0, x = 0;; ++x) {
            ok = __all_sync(0xffffffffu, mbar_wait(&sm.seg_full[x % kSegments32], uint32_t(x / kSegments32) & 1u, &sm.abort));
            if (!ok) break;
            const Segment32& g = sm.seg[x % kSegments32];
            if (g.n == 0) break;
            float o[D];
#pragma unroll
            for (int c = 0; c < D; ++c) o[c] = 0.f;
            const int units = g.n;
            float2 ml = make_float2(-INFINITY, 0.f);
            for (int j = 0; j < units; ++j) {
                const int u = i + j;
                ok = mbar_wait(&sm.f_ready[u & 3], uint32_t(u >> 2) & 1u, &sm.abort);
                const float f = ok ? sm.f[u & 3][row] : 0.f;
                if (ok) ml = sm.ml[u & 3][row];
                ok = ok && mbar_wait(&sm.o_done, uint32_t(u) & 1u, &sm.abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_after();
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    uint32_t v[8];
                    tmem_ld8(lanes + kO + 8u * c, v);
                    tc_wait_ld(v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[8 * c + e] = fmaf(o[8 * c + e], f, __uint_as_float(v[e]));
                }
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.o_free);
            }
            if (!ok) break;
            if (row < g.rows) {
                // the item's slot (where it lies in this share alone: the one that a later item may take)
                float* slot = part_slot<kRows32, D>(a, blockIdx.x, g.parts == 1 ? 0 : 1);
                if (g.later) {
                    const float2 old = reinterpret_cast<const float2*>(slot + kRows32 * D)[row];
                    const float m = fmaxf(old.x, ml.x), f = old.x == m ? 1.f : ex2(old.x - m), e = ml.x == m ? 1.f : ex2(ml.x - m);
                    ml = make_float2(m, fmaf(old.y, f, ml.y * e));
#pragma unroll
                    for (int c = 0; c < D; c += 4) {
                        const float4 z = *reinterpret_cast<const float4*>(slot + (size_t)row * D + c);
                        o[c] = fmaf(z.x, f, o[c] * e);
                        o[c + 1] = fmaf(z.y, f, o[c + 1] * e);
                        o[c + 2] = fmaf(z.z, f, o[c + 2] * e);
                        o[c + 3] = fmaf(z.w, f, o[c + 3] * e);
                    }
                }
                if (g.parts == 0 && !g.more) {
                    float* dst = out_row<float>(a, g.start, g.first, row, g.kvh);
                    const float inv = ml.y == 0.f ? 0.f : 1.0f / ml.y;
#pragma unroll
                    for (int c = 0; c < D; c += 4)
                        *reinterpret_cast<float4*>(dst + c) =
                            ml.y == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                        : make_float4(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv);
                } else {
#pragma unroll
                    for (int c = 0; c < D; c += 4)
                        *reinterpret_cast<float4*>(slot + (size_t)row * D + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                    reinterpret_cast<float2*>(slot + kRows32 * D)[row] = ml;
                }
            }
            i += units;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.seg_empty[x % kSegments32]);
        }
    } else if (wg < 4) {
        // ---- K and V: warp c of 8 takes keys 8 c .. 8 c + 7 of a unit
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsSplit));
        constexpr int kLanes = D / 4, kPer = 32 / kLanes, kLoads = 8 / kPer;  // lanes of a key, keys at once, loads
        const int c = warp - 8, key = 8 * c + lane / kLanes, d4 = lane % kLanes;
        float4 kr[kLoads], vr[kLoads];
        const auto load = [&](float4 (&y)[kLoads], const Unit32& w, const void* base, long long bs, long long ts, long long hs) {
            const int id = w.ids[c >> 1], keys = id < 0 ? 0 : w.keys - key,  // of this lane's first on
                       tok = (w.tok + key) & ((1 << a.shift) - 1);
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + max(id, 0) * bs + tok * ts +
                                                              w.kvh * hs) + d4;
            const long long step = kPer * (ts / 4);
            if (keys >= 8) {
#pragma unroll
                for (int e = 0; e < kLoads; ++e) y[e] = __ldg(p + e * step);
            } else {
#pragma unroll
                for (int e = 0; e < kLoads; ++e) y[e] = e * kPer < keys ? __ldg(p + e * step) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        };
        const auto store = [&](const float4 (&y)[kLoads], unsigned char (*tile)[Smem::kWord]) {
#pragma unroll
            for (int e = 0; e < kLoads; ++e) {
                const int r = key + e * kPer;
                uint2 h, m, l;
                split3(y[e].x, y[e].y, h.x, m.x, l.x);
                split3(y[e].z, y[e].w, h.y, m.y, l.y);
                const uint32_t at = (d4 / 16) * kHalf + r * 128 + ((((d4 % 16) / 2) ^ (r & 7)) << 4) + (d4 & 1) * 8;
                *reinterpret_cast<uint2*>(tile[0] + at) = h;
                *reinterpret_cast<uint2*>(tile[1] + at) = m;
                *reinterpret_cast<uint2*>(tile[2] + at) = l;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        // the unit's K and V are in registers when its turn comes, the next unit's loads follow them
        bool ok = uniform(mbar_wait(&sm.unit_full[0], 0u, &sm.abort));
        if (ok) ok = sm.unit[0].kvh >= 0;
        if (ok) {
            load(kr, sm.unit[0], a.c.k, a.c.k_block_stride, a.c.k_token_stride, a.c.k_head_stride);
            load(vr, sm.unit[0], a.c.v, a.c.v_block_stride, a.c.v_token_stride, a.c.v_head_stride);
        }
        bool more = true;
        for (int i = 0; more && ok; ++i) {
            const int s = i & 1;
            const Unit32& next = sm.unit[(i + 1) % kUnits32];
            if (i >= 2) ok = uniform(mbar_wait(&sm.k_empty[s], uint32_t((i >> 1) + 1) & 1u, &sm.abort));
            if (!ok) break;
            if (lane == 0 && (c & 1) == 0)
                *reinterpret_cast<volatile unsigned*>(&sm.bad[i & 3][c >> 1]) = sm.unit[i % kUnits32].ids[c >> 1] < 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.unit_empty[i % kUnits32]);
            store(kr, sm.k[s]);
            if (lane == 0) mbar_arrive(&sm.k_full[s]);
            ok = uniform(mbar_wait(&sm.unit_full[(i + 1) % kUnits32], uint32_t((i + 1) / kUnits32) & 1u, &sm.abort));
            if (!ok) break;
            more = uniform(next.kvh) >= 0;
            if (more) load(kr, next, a.c.k, a.c.k_block_stride, a.c.k_token_stride, a.c.k_head_stride);
            if (i >= 2) ok = uniform(mbar_wait(&sm.v_empty[s], uint32_t((i >> 1) + 1) & 1u, &sm.abort));
            if (!ok) break;
            store(vr, sm.v[s]);
            if (lane == 0) mbar_arrive(&sm.v_full[s]);
            if (more) load(vr, next, a.c.v, a.c.v_block_stride, a.c.v_token_stride, a.c.v_head_stride);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        if (warp == 16) {
            // ---- products
            bool ok = true;
            const auto scores = [&](int u) {
                const uint32_t d = tmem + kS + kSBuf * (u & 1), k = desc_low(smem_u32(sm.k[u & 1][0]), 16);
#pragma unroll
                for (int p = 0; p < 6; ++p)
#pragma unroll
                    for (int e = 0; e < D / 16; ++e)
                        mma_ts32(d, tmem + kQ + kQWord * word_a(p) + 8u * e,
                                 k + ((kWord * word_b(p) + (e / 4) * kHalf + (e % 4) * 32u) >> 4), idesc32(kUnit32, false),
                                 p > 0 || e > 0);
                tc_commit(&sm.s_ready[u & 1]);
                tc_commit(&sm.k_empty[u & 1]);
            };
            for (int i = 0, x = 0; ok; ++x) {
                ok = uniform(mbar_wait(&sm.seg_full[x % kSegments32], uint32_t(x / kSegments32) & 1u, &sm.abort));
                if (!ok) break;
                const int units = uniform(sm.seg[x % kSegments32].n);
                __syncwarp();
                if (elect()) mbar_arrive(&sm.seg_empty[x % kSegments32]);
                if (units == 0) break;
                ok = uniform(mbar_wait(&sm.q_full, uint32_t(x) & 1u, &sm.abort));
                for (int j = -2; j < units && ok; ++j) {  // P V of unit j, then Q K^T of unit j + 2
                    const int u = i + j;
                    if (j >= 0) {
                        ok = uniform(mbar_wait(&sm.v_full[u & 1], uint32_t(u >> 1) & 1u, &sm.abort));
                        if (ok && u > 0) ok = uniform(mbar_wait(&sm.o_free, uint32_t(u - 1) & 1u, &sm.abort));
                        ok = ok && uniform(mbar_wait(&sm.p_ready[u & 1], uint32_t(u >> 1) & 1u, &sm.abort));
                        if (!ok) break;
                        tc_after();
                        if (elect()) {
                            const uint32_t p = tmem + kS + kSBuf * (u & 1), v = desc_low(smem_u32(sm.v[u & 1][0]), kHalf);
#pragma unroll
                            for (int y = 0; y < 6; ++y)
#pragma unroll
                                for (int e = 0; e < kUnit32 / 16; ++e)
                                    mma_ts32(tmem + kO, p + kPWord * word_a(y) + 8u * e,
                                             v + ((kWord * word_b(y) + e * 2048u) >> 4), idesc32(D, true), y > 0 || e > 0);
                            tc_commit(&sm.o_done);
                            tc_commit(&sm.v_empty[u & 1]);
                        }
                        __syncwarp();
                    }
                    if (j + 2 < units) {
                        ok = uniform(mbar_wait(&sm.k_full[u & 1], uint32_t((u + 2) >> 1) & 1u, &sm.abort));
                        if (!ok) break;
                        tc_after();
                        if (elect()) scores(u + 2);
                        __syncwarp();
                    }
                }
                i += units;
            }
            if (elect()) {
                tc_commit(&sm.done);  // completes when every product issued above has
                mbar_wait(&sm.done, 0u, nullptr);
            }
            __syncwarp();
        } else if (warp == 17) {
            // ---- items
            Walk32 w;
            w.start(a, sh);
            bool ok = true, later = false;
            int parts = 0;  // of the item, as its first segment has it
            for (int x = 0;; ++x) {
                if (x >= kSegments32)
                    ok = uniform(mbar_wait(&sm.seg_empty[x % kSegments32], uint32_t(x / kSegments32 + 1) & 1u, &sm.abort, kItemLimitNs));
                if (!ok) break;
                Segment32 g;
                g.n = 0;  // the end
                if (w.work()) {
                    g = segment32(a, w, sh);
                    if (later) g.parts = parts;
                    parts = g.parts;
                    g.later = later;
                    g.more = later = g.n > kStretch32;
                    g.n = min(g.n, kStretch32);
                }
                if (lane == 0) {
                    sm.seg[x % kSegments32] = g;
                    mbar_arrive(&sm.seg_full[x % kSegments32]);
                    if (g.n > 0 && g.parts > 1) put_record(a, blockIdx.x, g.parts, g.kvh, g.rows, g.start, g.first);
                }
                if (g.n == 0) break;
                w.advance(a, g.n);
            }
        } else if (warp == 18) {
            // ---- units: lane = 16 keys
            Walk32 w;
            w.start(a, sh);
            int keys = w.r.keys<kRows32>(a, w.t);
            bool ok = true;
            for (int i = 0;; ++i) {
                const int x = i % kUnits32;
                const bool more = w.work();
                const int first = (w.k - kItem32) * kUnit32, key0 = first + 16 * lane;
                int id = -1;
                if (more && lane < kUnit32 / 16 && key0 < keys) id = __ldcg(a.table + w.b * a.table_stride + (key0 >> a.shift));
                if (i >= kUnits32) ok = uniform(mbar_wait(&sm.unit_empty[x], uint32_t(i / kUnits32 + 1) & 1u, &sm.abort));
                if (!ok) break;
                if (lane < kUnit32 / 16) sm.unit[x].ids[lane] = (unsigned)id < (unsigned)a.c.blocks ? id : -1;
                if (lane == 0) {
                    sm.unit[x].keys = keys - first;
                    sm.unit[x].tok = first & ((1 << a.shift) - 1);
                    sm.unit[x].kvh = more ? w.h : -1;  // -1: the end
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.unit_full[x]);
                if (!more) break;
                w.advance(a, 1);
                if (w.k == 0 && w.left > 0) keys = w.r.keys<kRows32>(a, w.t);
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == 16) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (sm.abort) poison32<D>(a, sh);
}

template <int D>
cudaError_t launch(const Attn& a, cudaStream_t s) {
    constexpr size_t smem = sizeof(Smem32<D>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    cudaError_t e = allow_smem<k_attn_tile32<D>>(smem, kRegsLaunch);
    if (e != cudaSuccess) return e;
    if ((e = launch_pdl(k_attn_tile32<D>, kCtas32, kThreads32, smem, s, a)) != cudaSuccess) return e;
    return launch_pdl(k_join_rows<float, kRows32, D>, dim3(kCtas32, kRows32 / join_rows(D)), kJoinThreads, 0, s, a);
}

}  // namespace

size_t tile32_workspace_floats(int head_dim) {
    return size_t(2) * kCtas32 * (head_dim == 64 ? part_floats<kRows32, 64>() : part_floats<kRows32, 128>());
}

cudaError_t launch_tile32(const Attn& a, cudaStream_t s) {
    return a.c.head_dim == 128 ? launch<128>(a, s) : launch<64>(a, s);
}

}  // namespace paged
}  // namespace itts
