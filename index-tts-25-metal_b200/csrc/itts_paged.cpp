// Entry points of the paged K/V cache operators (include/itts_paged.h): the
// argument checks, the device switch and the launches.  No state is kept
// beyond the calling thread's message.
#include "itts_paged.h"

#include <cuda_runtime.h>

#include <cmath>
#include <new>
#include <string>

#include "paged.hpp"

namespace {

thread_local std::string g_paged_error;

struct PagedFailure {
    int code;
    std::string msg;
};
void check(bool ok, const char* msg) {
    if (!ok) throw PagedFailure{ITTS_ERR_INVALID_ARGUMENT, msg};
}
void ck(cudaError_t e, const char* what) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        throw PagedFailure{ITTS_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e)};
    }
}

// Makes `device` current for a scope.
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int device) {
        int cur = 0;
        ck(cudaGetDevice(&cur), "cudaGetDevice");
        if (cur != device) {
            ck(cudaSetDevice(device), "cudaSetDevice");
            prev = cur;
        }
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

template <class F>
int guard(F&& f) {
    try {
        g_paged_error.clear();
        f();
        return ITTS_OK;
    } catch (const PagedFailure& e) {
        g_paged_error = e.msg;
        return e.code;
    } catch (const std::bad_alloc&) {
        return ITTS_ERR_OUT_OF_MEMORY;
    } catch (const std::exception& e) {
        g_paged_error = e.what();
        return ITTS_ERR_RUNTIME;
    }
}

constexpr int64_t kInt32 = int64_t(1) << 31;
constexpr int32_t kMaxRows = 1 << 30;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t size_of(int type) { return type == ITTS_PAGED_F32 ? 4 : 2; }
bool known(int type) { return type == ITTS_PAGED_F32 || type == ITTS_PAGED_F16 || type == ITTS_PAGED_BF16; }
// Strides of up to 2^40 bytes that keep 16-byte alignment.
bool stride16(int64_t stride, int type) {
    const int64_t most = (int64_t(1) << 40) / size_of(type);
    return stride >= 0 && stride < most && stride * size_of(type) % 16 == 0;
}

void check_block(int32_t block_size, int32_t blocks) {
    check(block_size == 16 || block_size == 32 || block_size == 64 || block_size == 128,
          "paged cache block_size is 16, 32, 64 or 128");
    check(blocks >= 1 && int64_t(blocks) * block_size < kInt32, "paged cache size out of range");
}

void check_cache(const itts_paged_cache& c) {
    check(c.k && c.v, "paged cache is null");
    check(known(c.type), "paged cache type is f32, f16 or bf16");
    check_block(c.block_size, c.blocks);
    check(c.heads >= 1 && c.heads <= 1024, "paged cache heads out of range");
    check(c.head_dim == 64 || c.head_dim == 128, "paged cache head_dim is 64 or 128");
    check(c.reserved == 0, "paged cache reserved field is not 0");
    check(aligned(c.k, 16) && aligned(c.v, 16) && stride16(c.k_block_stride, c.type) &&
              stride16(c.k_token_stride, c.type) && stride16(c.k_head_stride, c.type) &&
              stride16(c.v_block_stride, c.type) && stride16(c.v_token_stride, c.type) &&
              stride16(c.v_head_stride, c.type),
          "paged cache addresses and strides must be multiples of 16 bytes");
}

void check_table(const int32_t* table, int64_t stride, int32_t requests, int32_t max_blocks, int32_t block_size) {
    check(table, "block table is null");
    check(requests >= 1 && requests <= ITTS_PAGED_MAX_REQUESTS, "requests out of range");
    check(max_blocks >= 1 && int64_t(max_blocks) * block_size <= kMaxRows, "block table width out of range");
    check(stride >= max_blocks && stride < kInt32, "block table stride out of range");
}

}  // namespace

extern "C" {

const char* itts_paged_last_error(void) { return g_paged_error.c_str(); }

int itts_paged_tables(int device, const itts_paged_tables_args* a, void* stream) {
    return guard([&] {
        check(a, "args is null");
        check_block(a->block_size, a->blocks);
        check_table(a->table, a->table_stride, a->requests, a->max_blocks, a->block_size);
        check(a->rows >= 0 && a->rows <= kMaxRows, "rows out of range");
        check(a->cached && a->fresh && a->free_list && a->free_in && a->free_out && a->lens && a->q_start && a->status,
              "null argument");
        check(a->rows == 0 || (a->positions && a->slots), "null argument");
        OnDevice on(device);
        ck(itts::paged::launch_tables(*a, static_cast<cudaStream_t>(stream)), "block tables");
    });
}

int itts_paged_append(int device, const itts_paged_append_args* a, void* stream) {
    return guard([&] {
        check(a, "args is null");
        check_cache(a->cache);
        check(a->source_type == a->cache.type || a->source_type == ITTS_PAGED_F32,
              "source type is the cache's type or f32");
        check(a->rows >= 0 && a->rows <= kMaxRows, "rows out of range");
        if (a->rows == 0) return;
        check(a->k && a->v && a->slots, "null argument");
        const int64_t size = size_of(a->source_type), most = (int64_t(1) << 40) / size;
        const itts_paged_cache& c = a->cache;
        check(c.k_token_stride && c.v_token_stride && (c.blocks == 1 || (c.k_block_stride && c.v_block_stride)) &&
                  (c.heads == 1 || (c.k_head_stride && c.v_head_stride)),
              "paged cache repeats a dimension that the append writes");
        check(aligned(a->k, size_t(size)) && aligned(a->v, size_t(size)), "key or value rows are misaligned");
        for (int64_t s : {a->k_row_stride, a->k_head_stride, a->v_row_stride, a->v_head_stride})
            check(s >= 0 && s < most, "key or value stride out of range");
        OnDevice on(device);
        ck(itts::paged::launch_append(*a, static_cast<cudaStream_t>(stream)), "paged append");
    });
}

size_t itts_paged_attention_workspace(int32_t head_dim) {
    return head_dim == 64 || head_dim == 128 ? itts::paged::attention_workspace(head_dim) : 0;
}

int itts_paged_attention(int device, const itts_paged_attention_args* a, void* stream) {
    return guard([&] {
        check(a, "args is null");
        check_cache(a->cache);
        check_table(a->table, a->table_stride, a->requests, a->max_blocks, a->cache.block_size);
        check(a->rows >= 0 && a->rows <= kMaxRows, "rows out of range");
        check(a->q_heads >= 1 && a->q_heads % a->cache.heads == 0 && a->q_heads / a->cache.heads <= 128,
              "q_heads must be a multiple (at most 128 times) of the cache's heads");
        check(int64_t(a->rows) * (a->q_heads / a->cache.heads) <= kMaxRows, "rows out of range");
        check(a->max_fresh >= 1, "max_fresh must be positive");
        check(std::isfinite(a->scale), "scale must be finite");
        check(a->workspace && aligned(a->workspace, 256) &&
                  a->workspace_bytes >= itts::paged::attention_workspace(a->cache.head_dim),
              "workspace is null, misaligned or too small");
        if (a->rows == 0) return;
        check(a->q && a->out && a->q_start && a->lens, "null argument");
        check(a->q != a->out, "out must not overlap q");
        check(aligned(a->q, 16) && aligned(a->out, 16) && stride16(a->q_row_stride, a->cache.type) &&
                  stride16(a->q_head_stride, a->cache.type) && stride16(a->out_row_stride, a->cache.type) &&
                  stride16(a->out_head_stride, a->cache.type),
              "q and out addresses and strides must be multiples of 16 bytes");
        check((a->rows == 1 || a->out_row_stride) && (a->q_heads == 1 || a->out_head_stride), "out repeats a dimension");
        OnDevice on(device);
        ck(itts::paged::launch_attention(*a, static_cast<cudaStream_t>(stream)), "paged attention");
    });
}

}  // extern "C"
