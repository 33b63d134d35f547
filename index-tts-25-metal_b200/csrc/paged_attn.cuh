// What the paged attention kernels share: the geometry of a request, the
// sharing-out of the work among CTAs, and the partial results of items that
// several CTAs work on.
//
// An item is (request, row tile, key / value head): the rows of a request that
// read one key / value head, G = q_heads / heads of them per token, are
// numbered token-major (row r = token r / G, query head h * G + r % G) and cut
// into tiles of RT rows, so that the query heads of a group share the keys they
// load.  An item's keys (those that its last row sees) are cut into units of KU
// keys; an item without keys has one unit, which writes its zeros.  The lengths
// are on the device, so the sharing-out is too: every CTA adds up the units of
// all requests and takes an equal share [i U / n, (i + 1) U / n) of them, which
// keeps all SMs busy whether there are many short requests or one long one.  What
// an item costs besides its units (its queries, its output) counts as kItem units
// before its first one, which are shared out like the others but not worked on.
// An item that ends up with several CTAs leaves partial sums in the workspace,
// two slots a CTA (slot 0: the item its share begins inside of; slot 1: the
// item that begins in it and goes on in the next); k_join adds them up in CTA
// order, so results do not depend on timing.  Within a share sums of long items
// meet there, too, stretch by stretch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "paged.hpp"

namespace itts {
namespace paged {

constexpr int kMaxCtas = 592;  // of one attention launch: 148 SMs, up to four CTAs each
constexpr float kLog2e = 1.4426950408889634f;
// Units of one CTA beyond which a launch does nothing: minutes of work, which only lengths out of their senses ask for.
// It keeps the counts of a share in 32 bits.
constexpr long long kMostUnits = 1 << 29;
// A request's units are not counted on from here: it alone is more than all CTAs take, and so is the sum over
// 2^13 requests and 2^10 heads, which stays in 64 bits.
constexpr long long kEnoughUnits = 1ll << 39;
static_assert(kEnoughUnits > kMostUnits * kMaxCtas, "");

// The part of the arguments that the kernels read.
struct Attn {
    itts_paged_cache c;
    const void* q;
    void* out;
    long long q_row, q_head, o_row, o_head;
    const int *q_start, *lens, *table;
    long long table_stride;
    int rows, requests, group, shift;  // group = q_heads / heads, shift = log2(block_size)
    int cap;                           // keys that the table's columns can name
    uint32_t group_mul;                // r / group = r * group_mul >> group_shift for r < 2^30
    int group_shift;
    float scale2;                      // |scale| log2(e), at least 1e-30: a masked -inf stays -inf
    float sign;                        // of the scale, taken into q
    float* part;                       // partial sums
    int4* rec;                         // per CTA: {CTAs of the item that begins here, first row, kv head, rows}
};

__device__ __forceinline__ int over_group(const Attn& a, int r) {
    return int((unsigned long long)(unsigned)r * a.group_mul >> a.group_shift);
}

// A request's rows and keys.
struct Request {
    int start, tokens, rows, len;
    __device__ __forceinline__ void load(const Attn& a, int b) {
        const int s = __ldcg(a.q_start + b), e = __ldcg(a.q_start + b + 1);
        len = max(__ldcg(a.lens + b), 0);
        start = min(max(s, 0), a.rows);
        tokens = max(min(max(e, 0), a.rows) - start, 0);
        rows = tokens * a.group;  // the host has checked that a.rows * group <= 2^30
    }
    // Position of the token of row r.
    __device__ __forceinline__ int pos(const Attn& a, int r) const { return len - tokens + over_group(a, r); }
    // Keys that some row of tile t sees.
    template <int RT>
    __device__ __forceinline__ int keys(const Attn& a, int t) const {
        const int last = pos(a, min((t + 1) * RT, rows) - 1);
        return min(max(last + 1, 0), a.cap);
    }
    template <int RT, int KU>
    __device__ __forceinline__ int units(const Attn& a, int t) const {
        return max(1, (keys<RT>(a, t) + KU - 1) / KU);
    }
    // Units of one key / value head over all tiles.
    template <int RT, int KU, int kItem>
    __device__ __forceinline__ long long total(const Attn& a) const {
        long long n = 0;
        for (int t = 0; t * RT < rows && n < kEnoughUnits; ++t) n += kItem + units<RT, KU>(a, t);
        return n;
    }
};

// a b / c for b, c < 1024, in 32 bits where they do.
__device__ __forceinline__ long long share_of(long long a, int b, int c) {
    return a < (1 << 22) ? (long long)(unsigned(a) * unsigned(b) / unsigned(c)) : a * b / c;
}

// The units of a launch and where this CTA's share begins.
struct Share {
    long long units, u0, u1;  // of all items; this CTA's
    int ctas;                 // that have a share: every one of them at least one unit
    int b;                    // request of u0
    long long base;           // units before that request
    Request r;                // that request
};

template <int kThreadsT>
struct PlanSmem {
    long long warp_sum[kThreadsT / 32];
    Share share;
};

// Called by all threads of the CTA.  Returns the units of its share (0: none),
// which is then in sm.share.  `scratch`: a count per request in shared memory,
// used where there are more requests than threads.
template <int RT, int KU, int kItem, int kThreadsT>
__device__ int plan(const Attn& a, int cta, int ctas, PlanSmem<kThreadsT>& sm, long long* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.requests + kThreadsT - 1) / kThreadsT, b0 = tid * per, b1 = min(a.requests, b0 + per);
    long long mine = 0;
    Request r{};
    if (per == 1) {
        if (b0 < b1) {
            r.load(a, b0);
            mine = r.total<RT, KU, kItem>(a);
        }
    } else {  // coalesced loads, several in flight; then each thread adds up its requests in a row
#pragma unroll 4
        for (int b = tid; b < a.requests; b += kThreadsT) {
            Request x;
            x.load(a, b);
            scratch[b] = x.total<RT, KU, kItem>(a);
        }
        __syncthreads();
        for (int b = b0; b < b1; ++b) mine += scratch[b];
    }
    mine *= a.c.heads;
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sm.warp_sum[warp] = inc;
    __syncthreads();
    long long before = inc - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kThreadsT / 32; ++w) {
        if (w < warp) before += sm.warp_sum[w];
        all += sm.warp_sum[w];
    }
    if (all >= kMostUnits * ctas) all = 0;
    Share s{};
    s.units = all;
    s.ctas = int(min((long long)ctas, all));
    s.u0 = cta < s.ctas ? share_of(all, cta, s.ctas) : all;
    s.u1 = cta < s.ctas ? share_of(all, cta + 1, s.ctas) : all;
    if (before <= s.u0 && s.u0 < before + mine) {  // one thread holds the request of u0
        s.base = before;
        s.b = b0;
        if (per > 1) {
            while (s.u0 >= s.base + scratch[s.b] * a.c.heads) s.base += scratch[s.b++] * a.c.heads;
            r.load(a, s.b);
        }
        s.r = r;
        sm.share = s;
    }
    __syncthreads();
    return int(s.u1 - s.u0);
}

// The CTA whose share holds unit u: the guess is at most off by its rounding.
__device__ __forceinline__ int cta_of(const Share& s, long long u) {
    int i = min(s.ctas - 1, int(float(u) * float(s.ctas) / float(s.units)));
    const long long behind = (u + 1) * s.ctas;  // share i begins at or before u: units i < behind
    while (i > 0 && s.units * i >= behind) --i;
    while (i + 1 < s.ctas && s.units * (i + 1) < behind) ++i;
    return i;
}

// Walks the items of a share, unit by unit.
template <int RT, int KU, int kItem>
struct Walk {
    Request r;
    int b, t, h;  // item: request, tile, kv head
    int k, nk;    // unit of the item, units of the item, the kItem first ones among them
    int left;     // units of the share from this one on
    __device__ __forceinline__ void start(const Attn& a, const Share& s) {
        b = s.b;
        r = s.r;
        t = 0;
        left = int(s.u1 - s.u0);
        long long before = s.u0 - s.base;
        for (;; ++t) {
            nk = kItem + r.units<RT, KU>(a, t);
            if (before < (long long)nk * a.c.heads) break;
            before -= (long long)nk * a.c.heads;
        }
        h = before < (1ll << 31) ? int(unsigned(before) / unsigned(nk)) : int(before / nk);
        k = int(before - (long long)h * nk);
    }
    // To a unit that is worked on, this one if it is; false: the share has none left.
    __device__ __forceinline__ bool work() {
        if (kItem && k < kItem) {
            left -= kItem - k;
            k = kItem;
        }
        return left > 0;
    }
    // n units on, within the item; behind its last one to the next item.
    __device__ __forceinline__ void advance(const Attn& a, int n) {
        k += n;
        left -= n;
        if (k < nk || left <= 0) return;
        k = 0;
        if (++h < a.c.heads) return;
        h = 0;
        ++t;
        if (t * RT >= r.rows) {
            t = 0;
            do r.load(a, ++b);
            while (r.rows == 0);
        }
        nk = kItem + r.units<RT, KU>(a, t);
    }
    // At a unit that is worked on: the units of the item from here on in this share, and in how many shares
    // the item is worked on if it begins here (0: all in this one; 1: it began in another).
    __device__ __forceinline__ int run() const { return min(nk - k, left); }
    __device__ __forceinline__ int parts(const Share& s) const {
        if (k > kItem) return 1;
        return run() == nk - k ? 0 : cta_of(s, s.u1 - left + (nk - k) - 1) - int(blockIdx.x) + 1;
    }
};

// Partial sums of an item: RT rows of D unnormalised outputs, then RT pairs
// (maximum in units of log2, sum); slots are multiples of 128 bytes, so that the
// rows keep the alignment of their 16-byte accesses whatever RT is.
template <int RT, int D>
__host__ __device__ constexpr size_t part_floats() {
    return (size_t(RT) * (D + 2) + 31) / 32 * 32;
}
template <int RT, int D>
__device__ __forceinline__ float* part_slot(const Attn& a, int cta, int which) {
    return a.part + (size_t)(2 * cta + which) * part_floats<RT, D>();
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes to shared memory; the first `bytes` of them are read, the rest is zeros.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Two values in 16 bits.
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

// Weights p = 2^(s - m) of fp16 products are lifted by a power of two, 2^lift p,
// whose greatest value is the 2^15 that fp16 still holds: the type ends at 2^-24
// below, not at 2^-126 as fp32 and bf16 do, and unlifted a key 17 nats behind the
// largest lost all of its weight in the products but none in the sum (over 2^20 such
// keys 3% of the output).  The sum is taken over lifted weights too, in the partial
// sums as well, so the division takes the lift out.  above: log2 of the greatest p.
template <class T>
__device__ constexpr float lift(int above) {
    return std::is_same<T, __half>::value ? float(15 - above) : 0.f;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class T>
__device__ __forceinline__ void store4(T* p, float4 v);
template <>
__device__ __forceinline__ void store4<float>(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <>
__device__ __forceinline__ void store4<__half>(__half* p, float4 v) {
    const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, float4 v) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// Where row `row` of the item whose first row is `first` (counted over a
// request that starts at `start`) goes.
template <class T>
__device__ __forceinline__ T* out_row(const Attn& a, int start, int first, int row, int kvh) {
    const int r = first + row, tok = over_group(a, r), g = r - tok * a.group;
    return static_cast<T*>(a.out) + (long long)(start + tok) * a.o_row + (long long)(kvh * a.group + g) * a.o_head;
}

__device__ __forceinline__ float4 normalised(float4 o, float l) {
    if (l == 0.f) return make_float4(0.f, 0.f, 0.f, 0.f);  // no key: a NaN sum is not 0
    const float i = 1.0f / l;
    return make_float4(o.x * i, o.y * i, o.z * i, o.w * i);
}

// Adds up the partial sums of the items that several CTAs worked on: CTA (i, r)
// takes rows r, r + gridDim.y, .. of the item that begins in share i, if it goes on
// in other shares.  Groups of D / 4 threads take every gth part each.
constexpr int kJoinThreads = 256;
template <class T, int RT, int D>
__global__ void __launch_bounds__(kJoinThreads) k_join(Attn a) {
    pdl_wait();
    pdl_trigger();
    constexpr int kCols = D / 4, kGroups = kJoinThreads / kCols;
    __shared__ float4 joined[kJoinThreads];
    __shared__ float2 ml_of[kGroups];
    const int cta = blockIdx.x, col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
    const int4 rec = __ldcg(a.rec + 2 * cta), where = __ldcg(a.rec + 2 * cta + 1);
    const int parts = rec.x;
    if (parts < 2) return;
    for (int row = blockIdx.y; row < rec.w; row += gridDim.y) {
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int i = grp; i < parts; i += kGroups) {
            const float* p = part_slot<RT, D>(a, cta + i, i == 0 ? 1 : 0);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + RT * D) + row);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + row * D) + col);
            const float mn = fmaxf(m, ml.x), ref = mn == -INFINITY ? 0.f : mn;
            const float f = ex2(m - ref), g = ex2(ml.x - ref);
            l = l * f + ml.y * g;
            o = make_float4(o.x * f + v.x * g, o.y * f + v.y * g, o.z * f + v.z * g, o.w * f + v.w * g);
            m = mn;
        }
        joined[threadIdx.x] = o;
        if (col == 0) ml_of[grp] = make_float2(m, l);
        __syncthreads();
        if (grp == 0) {
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int i = 0; i < kGroups; ++i) M = fmaxf(M, ml_of[i].x);
            const float ref = M == -INFINITY ? 0.f : M;
            o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const float g = ex2(ml_of[i].x - ref);
                const float4 v = joined[i * kCols + col];
                L += ml_of[i].y * g;
                o = make_float4(o.x + v.x * g, o.y + v.y * g, o.z + v.z * g, o.w + v.w * g);
            }
            store4<T>(out_row<T>(a, where.x, where.y, row, rec.z) + 4 * col, normalised(o, L));
        }
        __syncthreads();
    }
}

// The same for items of many rows, which few CTAs share: a thread per four
// columns of kJoinEach rows, blockIdx.y over the rows (us, 319 rows of 16 heads on 8 over
// 325 keys, 1 / 2 / 4 / 8 of them: 24.1 / 22.8 / 23.4 / 24.2).
constexpr int kJoinEach = 2;
__host__ __device__ constexpr int join_rows(int D) { return kJoinEach * kJoinThreads * 4 / D; }
template <class T, int RT, int D>
__global__ void __launch_bounds__(kJoinThreads) k_join_rows(Attn a) {
    pdl_wait();
    pdl_trigger();
    const int cta = blockIdx.x;
    const int4 rec = __ldcg(a.rec + 2 * cta);
    constexpr int kStep = join_rows(D) / kJoinEach;  // between a thread's rows
    const int col = threadIdx.x % (D / 4), row0 = blockIdx.y * join_rows(D) + threadIdx.x / (D / 4);
    if (rec.x < 2 || row0 >= rec.w) return;
    const int4 where = __ldcg(a.rec + 2 * cta + 1);
    float m[kJoinEach], l[kJoinEach];
    float4 o[kJoinEach];
#pragma unroll
    for (int e = 0; e < kJoinEach; ++e) {
        m[e] = -INFINITY;
        l[e] = 0.f;
        o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 2
    for (int i = 0; i < rec.x; ++i) {
        const float* p = part_slot<RT, D>(a, cta + i, i == 0 ? 1 : 0);
        float2 ml[kJoinEach];
        float4 v[kJoinEach];
#pragma unroll
        for (int e = 0; e < kJoinEach; ++e)
            if (row0 + e * kStep < rec.w) {
                ml[e] = __ldcg(reinterpret_cast<const float2*>(p + RT * D) + row0 + e * kStep);
                v[e] = __ldcg(reinterpret_cast<const float4*>(p + (row0 + e * kStep) * D) + col);
            }
#pragma unroll
        for (int e = 0; e < kJoinEach; ++e) {
            const float mn = fmaxf(m[e], ml[e].x), ref = mn == -INFINITY ? 0.f : mn;
            const float f = ex2(m[e] - ref), g = ex2(ml[e].x - ref);
            l[e] = l[e] * f + ml[e].y * g;
            o[e] = make_float4(o[e].x * f + v[e].x * g, o[e].y * f + v[e].y * g, o[e].z * f + v[e].z * g, o[e].w * f + v[e].w * g);
            m[e] = mn;
        }
    }
#pragma unroll
    for (int e = 0; e < kJoinEach; ++e)
        if (row0 + e * kStep < rec.w)
            store4<T>(out_row<T>(a, where.x, where.y, row0 + e * kStep, rec.z) + 4 * col, normalised(o[e], l[e]));
}

// Records the item that begins in this share and goes on (or none), for k_join.
__device__ __forceinline__ void put_record(const Attn& a, int cta, int parts, int kvh, int rows, int start, int first) {
    a.rec[2 * cta] = make_int4(parts, 0, kvh, rows);
    a.rec[2 * cta + 1] = make_int4(start, first, 0, 0);
}

}  // namespace paged
}  // namespace itts
