// Block tables and slot maps of a paged K/V cache from request lengths
// (itts_paged_tables).
//
// Per request: have = ceil(cached / bs) blocks held, need = blocks beyond
// those after the step (0 if released), give = have if released.  Three
// exclusive sums over the requests place everything: fresh rows (q_start),
// new blocks (off the free stack) and released blocks (onto it).
//
// The work is a few hundred bytes to a few megabytes, so launch and dependent
// loads bound it.  One cluster does the bookkeeping: every CTA computes the
// sums redundantly in shared memory (a read of 8 bytes per request from L2)
// and then takes its share of the releases and of the new table entries.  The
// one cluster barrier between them orders all reads of the state (lengths,
// count, free list) before its updates, so lens may be cached and free_out may
// be free_in, and makes the released ids visible to the requests that take them.
// Row maps of up to kFusedRows rows are filled by the same launch; longer
// ones by a second grid (k_slots) that finds each row's request by bisection
// of q_start.
#include <climits>

#include "common.cuh"
#include "paged.hpp"

namespace itts {
namespace paged {
namespace {

constexpr int kTabThreads = 512;
constexpr int kTabWarps = kTabThreads / 32;
// Rows that one launch maps; more take the second grid.  Measured (us, 64 requests, one launch / two): 8 k rows 5.8 /
// 6.6, 16 k rows 7.0 / 7.3, 32 k rows 9.8 / 7.7.
constexpr int kFusedRows = 16384;
// Requests, mapped rows and new blocks that one CTA handles; more take a cluster of eight.  Measured (us, one / eight):
// 545 of them 4.2 / 5.2, 1.1 k 4.6 / 4.7 to 5.5, 2.1 k 5.8 / 4.8 and 7.0 / 6.2.
constexpr int kSmallWork = 1280;
constexpr int kClusterCtas = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int ld_cluster(const int* local, uint32_t rank) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return int(v);
}

// Largest b with off(b) <= x, for off(0) = 0 <= x < off(n): the request that
// owns item x (requests without items share their successor's offset).
template <class Off>
__device__ __forceinline__ int owner(Off off, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off(mid) <= x)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int clamp_int(long long v) { return int(min(v, (long long)INT_MAX)); }

__global__ void __launch_bounds__(kTabThreads) k_tables(itts_paged_tables_args a, int ctas, int map_rows) {
    extern __shared__ int tab_smem[];
    const int B = a.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = ctas > 1 ? int(cluster_rank()) : 0, step = ctas * kTabThreads, me = rank * kTabThreads + tid;
    int* q_off = tab_smem;           // [B + 1] fresh rows before request b
    int* new_off = q_off + B + 1;    // [B + 1] new blocks before it
    int* give_off = new_off + B + 1; // [B + 1] released blocks before it
    int* held = give_off + B + 1;    // [B] cached tokens
    __shared__ long long part[3][kTabWarps + 1];
    __shared__ int bad, bad_block;
    pdl_trigger();
    if (tid == 0) bad = bad_block = 0;
    __syncthreads();

    const int bs = a.block_size, shift = 31 - __clz(bs);
    const long long capacity = (long long)a.max_blocks * bs;
    const int per = (B + kTabThreads - 1) / kTabThreads, b0 = min(B, tid * per), b1 = min(B, b0 + per);
    const int F = __ldcg(a.free_in);
    long long sum[3] = {0, 0, 0};
    int flags = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = __ldcg(a.cached + b), f = __ldcg(a.fresh + b);
        held[b] = c;
        // the sums so far, relative to this thread's first request; made absolute below
        q_off[b] = clamp_int(sum[0]);
        new_off[b] = clamp_int(sum[1]);
        give_off[b] = clamp_int(sum[2]);
        if (c < 0 || (long long)c + max(f, 0) > capacity) {
            flags |= ITTS_PAGED_BAD_LENGTH;
            continue;
        }
        const int have = (c + bs - 1) >> shift;
        if (f >= 0) {
            sum[0] += f;
            sum[1] += int(((long long)c + f + bs - 1) >> shift) - have;
        } else {
            sum[2] += have;
        }
    }
    if (flags) atomicOr(&bad, flags);
    long long inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        inc[k] = sum[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc[k], o);
            if (lane >= o) inc[k] += v;
        }
        if (lane == 31) part[k][warp] = inc[k];
    }
    __syncthreads();
    if (tid < 3) {
        long long t = 0;
        for (int w = 0; w < kTabWarps; ++w) {
            const long long v = part[tid][w];
            part[tid][w] = t;
            t += v;
        }
        part[tid][kTabWarps] = t;
    }
    __syncthreads();
    const long long rows = part[0][kTabWarps], fresh_blocks = part[1][kTabWarps], given = part[2][kTabWarps];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const long long base = part[k][warp] + inc[k] - sum[k];
        int* off = k == 0 ? q_off : k == 1 ? new_off : give_off;
        for (int b = b0; b < b1; ++b) off[b] = clamp_int(base + off[b]);
    }
    if (tid == 0) {
        q_off[B] = clamp_int(rows);
        new_off[B] = clamp_int(fresh_blocks);
        give_off[B] = clamp_int(given);
        int f = 0;
        if (rows > a.rows) f |= ITTS_PAGED_NO_ROWS;
        if (F < 0 || F > a.blocks || F + given > a.blocks)
            f |= ITTS_PAGED_BAD_FREE;
        else if (fresh_blocks > F + given)
            f |= ITTS_PAGED_NO_BLOCKS;
        bad |= f;
    }
    __syncthreads();

    // Every CTA has come to the same flags.  Without one, the counts fit: 0 <=
    // F <= top <= blocks and fresh_blocks <= top.
    const bool fits = bad == 0;
    const int top = fits ? F + int(given) : 0;
    if (fits) {
        // the check of what was on the stack already, and the releases (checked as they go on it)
        bool wrong = false;
        for (int i = top - int(fresh_blocks) + me; i < F; i += step)
            wrong |= (unsigned)__ldcg(a.free_list + i) >= (unsigned)a.blocks;
        for (int i = me; i < int(given); i += step) {
            const int b = owner([=](int b) { return give_off[b]; }, B, i);
            const int id = __ldcg(a.table + (long long)b * a.table_stride + (i - give_off[b]));
            wrong |= (unsigned)id >= (unsigned)a.blocks;
            a.free_list[F + i] = id;
        }
        if (wrong) bad_block = ITTS_PAGED_BAD_BLOCK;
    }
    int late = 0;
    if (ctas > 1) {
        cluster_arrive();
        cluster_wait();
        for (int r = 0; r < ctas; ++r) late |= ld_cluster(&bad_block, r);
        cluster_arrive();  // waited for at the end: no CTA leaves while another reads its flag
    } else {
        __syncthreads();
        late = bad_block;
    }
    const bool ok = fits && !late;
    if (rank == 0 && tid == 0) {
        *a.status = bad | late;
        *a.free_out = ok ? top - int(fresh_blocks) : F;
        a.q_start[B] = ok ? q_off[B] : 0;
    }
    for (int b = me; b < B; b += step) {
        const int grown = held[b] + q_off[b + 1] - q_off[b];
        a.q_start[b] = ok ? q_off[b] : 0;
        a.lens[b] = !ok ? held[b] : __ldcg(a.fresh + b) < 0 ? 0 : grown;
    }
    if (ok) {
        constexpr int kBatch = 4;  // loads in flight: a store to the table may, for all the compiler knows, change the list
        for (int i0 = me; i0 < int(fresh_blocks); i0 += kBatch * step) {
            int id[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (i0 + u * step < int(fresh_blocks)) id[u] = __ldcg(a.free_list + top - 1 - (i0 + u * step));
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * step;
                if (i >= int(fresh_blocks)) break;
                const int b = owner([=](int b) { return new_off[b]; }, B, i), have = (held[b] + bs - 1) >> shift;
                a.table[(long long)b * a.table_stride + have + (i - new_off[b])] = id[u];
            }
        }
    }
    for (int t = me; t < map_rows; t += step) {
        int pos = 0, slot = -1;
        if (ok && t < q_off[B]) {
            const int b = owner([=](int b) { return q_off[b]; }, B, t), have = (held[b] + bs - 1) >> shift;
            pos = held[b] + (t - q_off[b]);
            const int j = pos >> shift;
            // a block of this step comes straight from the stack: its table entry may be another thread's store
            const int id = j < have ? __ldcg(a.table + (long long)b * a.table_stride + j)
                                    : __ldcg(a.free_list + top - 1 - (new_off[b] + j - have));
            if ((unsigned)id < (unsigned)a.blocks) slot = (id << shift) + (pos & (bs - 1));
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    if (ctas > 1) cluster_wait();
}

// Row maps from the finished tables: four rows per thread, 1024 per block.  The
// block finds its first row's request in two loads (256 samples of q_start, then
// a window from the sampled request on), and its threads bisect the window in
// shared memory.
constexpr int kSlotThreads = 256, kWindow = 5 * kSlotThreads;
__global__ void __launch_bounds__(kSlotThreads) k_slots(itts_paged_tables_args a) {
    __shared__ int first[kWindow + 1], len[kWindow];
    pdl_wait();
    const int B = a.requests, shift = 31 - __clz(a.block_size), tid = threadIdx.x;
    const int block0 = blockIdx.x * kSlotThreads * 4, t0 = block0 + tid * 4;
    const int total = __ldcg(a.q_start + B);
    const int sample = int((long long)tid * B / kSlotThreads);
    const int low = __syncthreads_count(__ldcg(a.q_start + sample) <= block0) - 1;
    const int base = int((long long)low * B / kSlotThreads);  // its q_start is at or before the block
#pragma unroll
    for (int i = 0; i < kWindow; i += kSlotThreads) {
        const int b = base + i + tid;
        first[i + tid] = b < B ? __ldcg(a.q_start + b) : total;
        len[i + tid] = b < B ? __ldcg(a.lens + b) : 0;
    }
    if (tid == 0) first[kWindow] = base + kWindow < B ? __ldcg(a.q_start + base + kWindow) : total;
    __syncthreads();
    if (t0 >= a.rows) return;
    int pos[4] = {0, 0, 0, 0}, slot[4] = {-1, -1, -1, -1};
    if (t0 < total) {
        // requests without rows may push the row's request out of the window
        const bool near = t0 < first[kWindow];
        int b = near ? base + owner([&](int r) { return first[r]; }, kWindow, t0)
                     : owner([&](int r) { return __ldcg(a.q_start + r); }, B, t0);
        const auto end_of = [&](int r) {
            return r - base < kWindow ? first[r - base + 1] : __ldcg(a.q_start + r + 1);
        };
        const auto len_of = [&](int r) { return r - base < kWindow ? len[r - base] : __ldcg(a.lens + r); };
        int end = end_of(b), n = len_of(b);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int t = t0 + k;
            if (t >= total) break;
            while (t >= end) {
                ++b;
                end = end_of(b);
                n = len_of(b);
            }
            pos[k] = n - (end - t);
            const int id = __ldcg(a.table + (long long)b * a.table_stride + (pos[k] >> shift));
            if ((unsigned)id < (unsigned)a.blocks) slot[k] = (id << shift) + (pos[k] & (a.block_size - 1));
        }
    }
    if (t0 + 4 <= a.rows && (reinterpret_cast<uintptr_t>(a.positions) & 15) == 0 &&
        (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0) {
        *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (t0 + k < a.rows) {
                a.positions[t0 + k] = pos[k];
                a.slots[t0 + k] = slot[k];
            }
    }
}

}  // namespace

cudaError_t launch_tables(const itts_paged_tables_args& a, cudaStream_t s) {
    const bool fused = a.rows <= kFusedRows;
    const int map_rows = fused ? a.rows : 0;
    const int ctas = a.requests + map_rows + a.rows / a.block_size <= kSmallWork ? 1 : kClusterCtas;
    const size_t smem = (size_t(a.requests) * 4 + 3) * sizeof(int);
    // whatever the size: what a launch may use without leave is 48 KB less the kernel's static shared memory
    cudaError_t e = allow_smem<k_tables>((size_t(ITTS_PAGED_MAX_REQUESTS) * 4 + 3) * sizeof(int));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kTabThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((e = cudaLaunchKernelEx(&cfg, k_tables, a, ctas, map_rows)) != cudaSuccess || fused) return e;
    return launch_pdl(k_slots, (a.rows + 4 * kSlotThreads - 1) / (4 * kSlotThreads), kSlotThreads, 0, s, a);
}

}  // namespace paged
}  // namespace itts
