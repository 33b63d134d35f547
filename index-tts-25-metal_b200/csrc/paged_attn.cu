// Causal attention of a step's fresh rows over a paged K/V cache
// (itts_paged_attention): the choice of kernel and the workspace.
#include <algorithm>
#include <cmath>

#include "paged_attn.cuh"

namespace itts {
namespace paged {

size_t few_workspace_floats(int head_dim);
cudaError_t launch_few(const Attn& a, long long rows, cudaStream_t s);
size_t tile_workspace_floats(int head_dim);
cudaError_t launch_tile(const Attn& a, cudaStream_t s);
size_t tile32_workspace_floats(int head_dim);
cudaError_t launch_tile32(const Attn& a, cudaStream_t s);

namespace {
// Rows of a request and kv head up to which the streaming kernel is used.  Measured (us, 16 requests, streaming / tile
// kernel), bf16, 16 heads on 8 of 128: 200 keys, 16 rows 16.0 / 18.1, 18 rows 26.5 / 18.2; 4000 keys, 16 rows 55 / 65,
// 18 rows 96 / 65.  fp32: 16 rows 20 / 24 and 144 / 169, 18 rows 36 / 24 and 280 / 170.
constexpr int kFewMost = 16;
constexpr size_t kRecords = size_t(2) * kMaxCtas * sizeof(int4);
}

size_t attention_workspace(int head_dim) {
    return kRecords + std::max({few_workspace_floats(head_dim), tile_workspace_floats(head_dim),
                                tile32_workspace_floats(head_dim)}) * sizeof(float);
}

cudaError_t launch_attention(const itts_paged_attention_args& p, cudaStream_t s) {
    Attn a{};
    a.c = p.cache;
    a.q = p.q;
    a.out = p.out;
    a.q_row = p.q_row_stride;
    a.q_head = p.q_head_stride;
    a.o_row = p.out_row_stride;
    a.o_head = p.out_head_stride;
    a.q_start = p.q_start;
    a.lens = p.lens;
    a.table = p.table;
    a.table_stride = p.table_stride;
    a.rows = p.rows;
    a.requests = p.requests;
    a.group = p.q_heads / p.cache.heads;
    int bits = 0;
    while ((1 << bits) < a.group) ++bits;
    a.group_shift = 30 + bits;
    a.group_mul = uint32_t(((uint64_t(1) << a.group_shift) + a.group - 1) / a.group);
    while ((1 << a.shift) < p.cache.block_size) ++a.shift;
    a.cap = p.max_blocks << a.shift;
    a.scale2 = std::fmax(std::fabs(p.scale) * kLog2e, 1e-30f);
    a.sign = p.scale < 0.f ? -1.f : 1.f;
    a.rec = static_cast<int4*>(p.workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + kRecords);
    if ((long long)p.max_fresh * a.group > kFewMost) {
        if (p.cache.type == ITTS_PAGED_F32) return launch_tile32(a, s);
        const cudaError_t e = launch_tile(a, s);
        if (e != cudaErrorNotSupported) return e;
    }
    return launch_few(a, (long long)p.max_fresh * a.group, s);
}

}  // namespace paged
}  // namespace itts
