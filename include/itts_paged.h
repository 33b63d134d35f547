/* C-ABI of the paged K/V cache operators (B200, sm_100a): block tables and slot
 * maps built on the GPU from request lengths, the append of a step's key and
 * value rows, and the attention of a step's query rows over the cached keys.
 * itts_qwen_generate_batch (itts_qwen.h) runs on them; a server with its own
 * model calls them on its own device buffers.
 *
 * A cache holds `blocks` blocks of `block_size` tokens.  Slot s is token
 * s % block_size of block s / block_size.  Request b's token p (p counted from
 * 0 over its whole length) lies in slot
 *   table[b * table_stride + p / block_size] * block_size + p % block_size.
 * A step gives every request b some fresh rows (none, one, or a chunk of a
 * prompt).  The rows of all requests are packed in request order: request b
 * owns rows q_start[b] .. q_start[b + 1) of the step's tensors.
 *
 * Conventions
 *  - All pointers in the argument structs are device pointers of GPU `device`;
 *    the calls enqueue on `stream` (a cudaStream_t of that device) and return
 *    without waiting.  They allocate nothing, keep nothing from one call to
 *    the next and may be captured into a CUDA graph.  The caller's current
 *    device is left as it was.
 *  - Status codes as in itts_gpt.h.  Arguments that the host can check (null
 *    pointers, sizes, types, alignment, the workspace's size) are refused with
 *    ITTS_ERR_INVALID_ARGUMENT before anything is enqueued; the message of
 *    the last failure on the calling thread is itts_paged_last_error().
 *  - Lengths, tables and slots live on the device, where the host cannot check
 *    them.  The kernels do: an index outside its range is never followed (each
 *    call says what happens instead).
 *  - Calls on several threads and streams may run at once as long as they write
 *    neither the same outputs nor the same workspace. */
#ifndef ITTS_PAGED_H
#define ITTS_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "itts_gpt.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ITTS_PAGED_MAX_REQUESTS 8192 /* requests of one call */

typedef enum itts_paged_type { ITTS_PAGED_F32 = 0, ITTS_PAGED_F16 = 1, ITTS_PAGED_BF16 = 2 } itts_paged_type;

/* Bits of the status word that itts_paged_tables writes on the device. */
#define ITTS_PAGED_BAD_LENGTH 1 /* cached < 0, or a length beyond the table's columns */
#define ITTS_PAGED_NO_ROWS 2    /* more fresh rows than `rows` */
#define ITTS_PAGED_NO_BLOCKS 4  /* the free list is too short */
#define ITTS_PAGED_BAD_FREE 8   /* free count outside 0 .. blocks, before or after the releases */
#define ITTS_PAGED_BAD_BLOCK 16 /* a released or a handed-out block id outside 0 .. blocks - 1 */

/* Message of the last failure of an itts_paged_* call on this thread. */
const char* itts_paged_last_error(void);

/* One step's bookkeeping: from the tokens that each request has cached and the
 * fresh rows it gets (or its release), the blocks it needs, its new table
 * entries and length, and for every fresh row its position and its slot.
 *
 * Releases come first, then the growth: the blocks of every released request
 * (fresh < 0) go on top of the free list in request order and, within a
 * request, in column order; then the requests take their new blocks from the
 * top, one after the other in request order.  The result does not depend on
 * timing.  A block id that is handed out is not erased from the free list; the
 * entries at and above the count mean nothing.
 *
 * Entries of the table that a request keeps are not checked: a row whose entry
 * is outside 0 .. blocks - 1 gets the slot -1, which the append leaves out.
 *
 * If a status bit is set nothing is taken or given: lens = cached (q_start all
 * 0, slots all -1, positions all 0), free_out = free_in, and the table is as
 * it was; free_list entries above the count may have been written. */
typedef struct itts_paged_tables_args {
    int32_t requests;     /* 1 .. ITTS_PAGED_MAX_REQUESTS */
    int32_t block_size;   /* 16, 32, 64 or 128 */
    int32_t blocks;       /* blocks of the pool; blocks * block_size < 2^31 */
    int32_t max_blocks;   /* columns of the table; max_blocks * block_size <= 2^30 */
    int64_t table_stride; /* elements between the rows of the table, >= max_blocks */
    int32_t rows;         /* entries of positions and slots, 0 .. 2^30 */
    const int32_t* cached;  /* [requests] tokens cached before the step */
    const int32_t* fresh;   /* [requests] rows of this step; < 0 releases the request */
    int32_t* table;         /* [requests][max_blocks], new entries are written */
    int32_t* free_list;     /* [blocks], a stack: the next block is free_list[count - 1] */
    const int32_t* free_in; /* [1] count before */
    int32_t* free_out;      /* [1] count after; may be free_in */
    int32_t* lens;          /* [requests] tokens after the step (0 if released); may be cached */
    int32_t* q_start;       /* [requests + 1] first fresh row of each request */
    int32_t* positions;     /* [rows] position of each fresh row; 0 behind the last */
    int32_t* slots;         /* [rows] slot of each fresh row; -1 behind the last */
    int32_t* status;        /* [1] ITTS_PAGED_* bits, 0 = done */
} itts_paged_tables_args;
int itts_paged_tables(int device, const itts_paged_tables_args* args, void* stream);

/* A paged cache: K and V of [blocks][block_size][heads][head_dim] elements at
 * any strides (in elements; head_dim contiguous).  A stride of 0 repeats a
 * dimension, such as one head for all: the attention reads it, the append
 * refuses it. */
typedef struct itts_paged_cache {
    void* k;
    void* v;
    int32_t type;       /* itts_paged_type */
    int32_t blocks;     /* blocks * block_size < 2^31 */
    int32_t block_size; /* 16, 32, 64 or 128 */
    int32_t heads;      /* key / value heads */
    int32_t head_dim;   /* 64 or 128 */
    int32_t reserved;   /* 0 */
    int64_t k_block_stride, k_token_stride, k_head_stride;
    int64_t v_block_stride, v_token_stride, v_head_stride;
} itts_paged_cache;

/* Writes key and value rows into the cache: row t goes to slot slots[t],
 * rounded to nearest even where the cache's type is narrower.  source_type is
 * the cache's type or ITTS_PAGED_F32.  A row whose slot is outside
 * 0 .. blocks * block_size - 1 (the padding of a step) is left out.  Two rows
 * with the same slot are the caller's error: each element then comes from one
 * of them. */
typedef struct itts_paged_append_args {
    itts_paged_cache cache;
    const void* k; /* [rows][heads][head_dim], head_dim contiguous */
    const void* v;
    int32_t source_type;
    int32_t rows; /* 0 .. 2^30 */
    int64_t k_row_stride, k_head_stride; /* elements */
    int64_t v_row_stride, v_head_stride;
    const int32_t* slots; /* [rows] */
} itts_paged_append_args;
int itts_paged_append(int device, const itts_paged_append_args* args, void* stream);

/* Causal attention of the fresh rows over the cached keys, the rows' own keys
 * (appended before) among them: row i of request b's n = q_start[b + 1] -
 * q_start[b] rows stands at position lens[b] - n + i and sees the keys at
 * positions 0 .. that position.  Query head h reads key / value head
 * h / (q_heads / heads).
 *   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max)
 * A row that sees no key (position < 0) is written as zeros.  Rows before
 * q_start[0] and from q_start[requests] on are left as they were.
 *
 * Scores, maxima and sums are held in fp32 and a 16-bit output is rounded once.
 * Where max_fresh * q_heads / heads is more than 16, the 16-bit types' weights
 * p_j are rounded to the type too before they multiply v_j (not for their sum;
 * by half a step, up to the output's own rounding), and their products are added
 * up by the tensor core, which does not round to nearest (up to 2^-13 of a sum).
 *
 * What lies in the cache behind a request's length, or in blocks that its
 * table does not name, never reaches the output, NaN and infinities included.
 * A table entry outside 0 .. blocks - 1 is not followed: its keys count as not
 * seen, as do the keys behind the table's last column.  q_start values are
 * clamped to 0 .. rows.  (A NaN in a key makes every row that sees it NaN, one in
 * a value the row's output at its dimension.  An infinity may make such a row NaN or infinite; a key whose score it
 * makes -inf may count as not seen.  Either in the value row of a later row of
 * the same chunk may reach the chunk's earlier rows, too.)
 *
 * Work beyond all measure is not begun: if the lengths ask for more than 2^29
 * tiles (of 1 to 128 rows by 32 to 128 keys) per CTA, which is minutes, every
 * row is left as it was.
 *
 * max_fresh is a bound on the fresh rows of one request, known on the host
 * where the lengths are not.  The kernel is chosen by it; results are right
 * (to rounding) whatever it says. */
typedef struct itts_paged_attention_args {
    itts_paged_cache cache;
    const void* q;   /* [rows][q_heads][head_dim] of the cache's type, head_dim contiguous */
    void* out;       /* as q; must not overlap it */
    int32_t q_heads; /* a multiple of cache.heads, at most 128 times it */
    int32_t rows;    /* 0 .. 2^30, and so is rows * q_heads / heads */
    int64_t q_row_stride, q_head_stride; /* elements */
    int64_t out_row_stride, out_head_stride; /* not 0 */
    const int32_t* q_start; /* [requests + 1] */
    const int32_t* lens;    /* [requests] */
    const int32_t* table;   /* [requests][max_blocks] */
    int64_t table_stride;
    int32_t requests;  /* 1 .. ITTS_PAGED_MAX_REQUESTS */
    int32_t max_blocks; /* columns of the table; max_blocks * block_size <= 2^30 */
    int32_t max_fresh; /* >= 1 */
    float scale;       /* finite */
    void* workspace;   /* 256-byte aligned; its contents before the call do not matter */
    size_t workspace_bytes; /* >= itts_paged_attention_workspace(...) */
} itts_paged_attention_args;
int itts_paged_attention(int device, const itts_paged_attention_args* args, void* stream);

/* Bytes of workspace that every itts_paged_attention call with this head_dim
 * needs (64 or 128; 0 for another). */
size_t itts_paged_attention_workspace(int32_t head_dim);

#ifdef __cplusplus
}
#endif

#endif /* ITTS_PAGED_H */
