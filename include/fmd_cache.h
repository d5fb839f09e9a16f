/*
 * fmd_cache.h -- C ABI of the paged-cache operators (same library,
 * libfmd_decoder.so): appending rows to a paged key/value cache in 16 or 4
 * bits, attention over it with a sliding window and sinks, and forking,
 * copying and compacting its pages. The decoder handle of fmd_decoder.h uses
 * the same kernels for its 4-bit cache, its window and its forks.
 *
 * Conventions
 *  - No handle. Every buffer is the caller's: device memory of the current
 *    device unless an argument is marked "host". Host arrays are read before
 *    the call returns.
 *  - Work is queued on `stream` (a cudaStream_t; NULL = legacy default
 *    stream). No call synchronises, allocates or keeps anything, so every call
 *    can be captured into a CUDA graph; calls that run at the same time need
 *    workspaces of their own.
 *  - Return values are the FMD_* codes of fmd_decoder.h; what the host can see
 *    is checked before anything is launched. What only the device can see (slots,
 *    positions, page numbers) is checked by the kernels: a row or page out of
 *    range is skipped, never accessed, and `status` (2 x int32, may be NULL)
 *    receives FMD_EINVAL (slot or page number) or FMD_EOVERFLOW (position).
 *  - Row pointers are 16-byte aligned and row and head strides are multiples
 *    of 8 elements; the dims of a head are contiguous. Inputs may repeat a row or
 *    a head with a stride of 0, and overlap. No two heads of an output may share an
 *    element, nor an output and an input but where q_out is q itself, strides
 *    included (FMD_EINVAL). Outputs whose addresses lie among an input's have the
 *    input's row stride, as views of one buffer have; with another they are refused.
 */
#ifndef FMD_CACHE_H
#define FMD_CACHE_H

#include <stdint.h>

#include "fmd_decoder.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FMD_CACHE_PAGE 64 /* positions of a page */
#define FMD_CACHE_WORKSPACE_ZERO 65536

/* ---- storage formats ------------------------------------------------------ */
#define FMD_CACHE_F16 1  /* FMD_DT_F16  */
#define FMD_CACHE_BF16 2 /* FMD_DT_BF16 */
#define FMD_CACHE_Q4 4   /* 4-bit codes, one f16 scale per 32 dims: 4.5 bits a value */

/* A paged cache. The pool is [layer][page][k|v][kv head][block], a block being
 * the 64 positions of one head (fmd_cache_block_bytes):
 *  - 16 bits: [64][head_dim];
 *  - Q4: 64 rows of head_dim / 2 code bytes, then 64 rows of head_dim / 32 f16
 *    scales d. A value is (code - 8) x d of its 32 dims, with d = f16(m / -8) for
 *    the value m of largest magnitude (the first among equals) and
 *    code = floor(-8 x / m + 8.5), at most 15. A key row's code bytes are four
 *    chunks c of head_dim / 8 bytes; chunk c holds one little-endian 32-bit word
 *    per 32-dim block g with dims 32 g + 8 c + e (e = 0..7) at nibble
 *    (e >> 1) + 4 (e & 1). A value row's word w holds dims 8 w + e at nibble e.
 *    Magnitudes above 65504 saturate; a NaN or infinity makes its block NaN.
 * Entry [slot][i] of the page table is the page of positions 64 i .. 64 i + 63. */
typedef struct fmd_cache {
  void* pool;           /* 16-byte aligned, fmd_cache_pool_bytes() bytes           */
  int32_t* page_table;  /* [max_slots][max_pages_per_slot]                         */
  int32_t format;       /* FMD_CACHE_*                                             */
  int32_t layers;
  int32_t n_pages;
  int32_t kv_heads;
  int32_t head_dim;     /* 64 or 128                                               */
  int32_t max_slots;
  int32_t max_pages_per_slot;
  int32_t reserved;
} fmd_cache;

/* The rows of a call: sequence i owns rows [row0[i], row0[i + 1]) of the
 * caller's row buffers, at positions pos0[i], pos0[i] + 1, ... of slot[i]. With
 * row0 == NULL each sequence has one row, row i. A sequence with slot -1 is
 * padding: its rows are left as they were, like the rows behind the last
 * sequence. Sequences without rows are allowed. No (slot, position) may appear twice. */
typedef struct fmd_cache_rows {
  const int32_t* slot;  /* [n_seqs]                                                */
  const int32_t* pos0;  /* [n_seqs]                                                */
  const int32_t* row0;  /* [n_seqs + 1], ascending, or NULL                        */
  int32_t n_seqs;
  int32_t n_rows;       /* rows of the row buffers (>= row0[n_seqs])               */
  int32_t max_rows;     /* attention: rows of the longest sequence at most; >= 1
                         * without row0                                            */
  int32_t reserved;
} fmd_cache_rows;

/* Bytes of one block, of the whole pool (0 for a bad description). */
int64_t fmd_cache_block_bytes(int32_t format, int32_t head_dim);
int64_t fmd_cache_pool_bytes(const fmd_cache* c);

/* ---- append ---------------------------------------------------------------- */

/* What fmd_cache_append does to each row. Strides are in elements. */
typedef struct fmd_cache_append_args {
  const void *k, *v;          /* rows of [kv_heads][head_dim]                       */
  const void* q;              /* rows of [n_heads][head_dim], or NULL               */
  void* q_out;                /* normed and rotated queries (may be q itself)       */
  int64_t k_row, k_head, v_row, v_head, q_row, q_head, q_out_row, q_out_head;
  const void *q_norm, *k_norm; /* [head_dim] RMS norm weights, or NULL: no norm     */
  const float *cos_table, *sin_table; /* [table_rows][rot_dim / 2], or NULL         */
  float eps;
  int32_t dtype;              /* of q, k, v, q_out and the norm weights: F16 / BF16 */
  int32_t n_heads;
  int32_t rot_dim;            /* leading dims rotated: a multiple of 8, 0: none     */
  int32_t table_rows;
  int32_t interleaved;        /* pairs (2 i, 2 i + 1); else (i, i + rot_dim / 2)    */
} fmd_cache_append_args;

/* Norms the query and key heads of each row, x * rsqrt(mean(x^2) + eps) * w,
 * rotates their first rot_dim dims by the row's position, (a, b) ->
 * (a cos - b sin, b cos + a sin), stores keys and values in the cache and the
 * queries in q_out, in one pass. f32 arithmetic, one rounding per stored value.
 * q_out may be q; k and v must not overlap the pool. A cache of 16 bits has the
 * rows' dtype. */
int fmd_cache_append(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows,
                     const fmd_cache_append_args* args, int32_t* status, void* stream);

/* The cached values of the rows' positions as f32, [n_rows][kv_heads][head_dim];
 * k and v may not overlap (FMD_EINVAL). */
int fmd_cache_read(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows, float* k, float* v,
                   int32_t* status, void* stream);

/* ---- attention --------------------------------------------------------------- */

typedef struct fmd_cache_attend_args {
  const void* q;      /* rows of [n_heads][head_dim]                               */
  void* out;          /* the same shape; must not overlap q                        */
  int64_t q_row, q_head, out_row, out_head; /* strides in elements                 */
  float scale;        /* of q . k, finite and > 0                                  */
  int32_t dtype;      /* of q and out: F16 / BF16 (that of a 16-bit cache)         */
  int32_t n_heads;    /* kv_heads x 1, 2, 4, 8 or 16; head h reads kv head
                       * h / (n_heads / kv_heads)                                  */
  int32_t window;     /* 0: none; else the newest `window` positions are visible   */
  int32_t sinks;      /* and the first `sinks` ones (ignored without a window)     */
} fmd_cache_attend_args;

/* Bytes of workspace for calls of up to n_seqs sequences of up to max_rows
 * rows (0: none needed). */
int64_t fmd_cache_attend_workspace(const fmd_cache* c, int32_t n_heads, int32_t n_seqs, int32_t max_rows);

/* Attention of each row over its slot's cached positions j <= its own position p
 * with window == 0, j > p - window or j < sinks: softmax(scale q . k_j) weighted
 * sum of the values. The row's own key is in the cache (append first). Pages
 * outside every row's window and sinks are not looked up. Softmax statistics and
 * sums are f32. Probabilities meet the values as 16-bit numbers: as two terms each
 * in calls of up to 16 (row, query head) pairs per kv head and sequence over 16 bits
 * and for f16 rows over 4 bits, else as one. 4-bit values, and the queries that meet
 * 4-bit keys, are rounded to f16.
 * What a cached position that no row of the call sees holds, NaN
 * included, has no influence. `workspace` is 16-byte aligned; its first
 * FMD_CACHE_WORKSPACE_ZERO bytes are zero before its first use, and every call
 * leaves them zero, so calls of any shape and cache may take turns with it (after
 * a FMD_ETIMEDOUT in `status` they must be zeroed again). `out` may not be q. */
int fmd_cache_attend(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows,
                     const fmd_cache_attend_args* args, void* workspace, int64_t workspace_bytes, int32_t* status,
                     void* stream);

/* ---- pages --------------------------------------------------------------------- */

/* Copies pages src[i] -> dst[i] (host arrays) of every layer. No dst may occur
 * twice or as a src (FMD_EINVAL). */
int fmd_cache_copy_pages(const fmd_cache* c, int32_t n, const int32_t* src, const int32_t* dst, void* stream);

/* Forks slots (host arrays): dst_slot[i] gets the first len[i] positions of
 * src_slot[i]: its page table row names the same full pages, and the len[i] % 64
 * rows behind them are copied, in every layer, to page new_page[i] (ignored when
 * there are none). No dst_slot may occur twice or as a src_slot, no new_page
 * twice (FMD_EINVAL), and none in a src_slot's row. */
int fmd_cache_fork(const fmd_cache* c, int32_t n, const int32_t* src_slot, const int32_t* dst_slot,
                   const int32_t* len, const int32_t* new_page, int32_t* status, void* stream);

/* Makes the pages in use dense: with U pages named by the first n_entries[slot]
 * entries of the page table's rows (device array [max_slots]; entries of -1 are
 * skipped), the i-th used page >= U moves into the i-th free page < U, in every
 * layer, and the entries follow. *n_used (device) receives U. A page that
 * several entries name stays shared. */
int64_t fmd_cache_compact_workspace(const fmd_cache* c);
int fmd_cache_compact(const fmd_cache* c, const int32_t* n_entries, void* workspace, int64_t workspace_bytes,
                      int32_t* n_used, int32_t* status, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FMD_CACHE_H */
