// The paged cache as its kernels see it (include/fmd_cache.h), shared by the
// cache operators and the decoder runtime.
#pragma once

#include <cuda.h>

#include "../../include/fmd_cache.h"
#include "fmd_common.cuh"

namespace fmd {

struct CacheView {
  uint8_t* pool;
  const int* page_table;
  int format, n_pages, kv_heads, head_dim, max_slots, max_pages;
  __host__ __device__ size_t block_bytes() const {
    return format == FMD_CACHE_Q4 ? (size_t)kPageTokens * (head_dim / 2 + head_dim / 16)
                                  : (size_t)kPageTokens * head_dim * 2;
  }
  __host__ __device__ size_t page_bytes() const { return 2 * kv_heads * block_bytes(); }
  // block of (layer, page, k|v, head)
  __host__ __device__ uint8_t* block(int layer, int page, int kv, int head) const {
    return pool + ((((size_t)layer * n_pages + page) * 2 + kv) * kv_heads + head) * block_bytes();
  }
};

// The sequences of a launch. blk_n == nullptr: the public form (slot and pos0
// by sequence, row0 null or [n + 1]). Else the decoder's prefill blocks: block
// i has blk_n[i] rows from row row0[i], slot and pos0 are by row; an even block
// and the next one, if it goes on in the same slot, are one sequence.
struct CacheRows {
  const int* slot;
  const int* pos0;
  const int* row0;
  const int* blk_n;
  const int* n_ptr;  // device count of sequences, or nullptr: n_seqs
  int n_seqs;
  int n_rows;
  FMD_DEV int count() const { return n_ptr ? min(*n_ptr, n_seqs) : n_seqs; }
  // rows [r0, r0 + n) of sequence i, clipped to the row buffers
  FMD_DEV void get(int i, int& sl, int& p0, int& r0, int& n) const {
    if (blk_n) {
      r0 = row0[i];
      n = blk_n[i];
      sl = slot[r0];
      p0 = pos0[r0];
      if (i & 1) {
        if (slot[row0[i - 1]] == sl) n = 0;  // part of the block before
      } else if (i + 1 < count() && slot[row0[i + 1]] == sl) {
        n += blk_n[i + 1];
      }
    } else {
      r0 = row0 ? row0[i] : i;
      n = row0 ? row0[i + 1] - r0 : 1;
      sl = slot[i];
      p0 = pos0[i];
    }
    if (r0 < 0 || r0 > n_rows) n = 0;
    n = min(n, n_rows - r0);
  }
};

FMD_DEV void cache_report(int* status, int code) {
  if (status) atomicCAS(status, 0, code);
}
// The page of position p of a slot, or -1 (reported).
FMD_DEV int cache_page(const CacheView& c, int slot, int p, int* status) {
  if (p < 0 || p / kPageTokens >= c.max_pages) {
    cache_report(status, FMD_EOVERFLOW);
    return -1;
  }
  const int page = c.page_table[(size_t)slot * c.max_pages + p / kPageTokens];
  if (page < 0 || page >= c.n_pages) {
    cache_report(status, FMD_EINVAL);
    return -1;
  }
  return page;
}
// A slot that can be looked up; -1 is padding, anything else out of range is reported.
FMD_DEV bool cache_slot_ok(const CacheView& c, int slot, int* status) {
  if (slot >= 0 && slot < c.max_slots) return true;
  if (slot != -1) cache_report(status, FMD_EINVAL);
  return false;
}

// ---- launchers ------------------------------------------------------------------
struct CacheAppend {
  const void *q, *k, *v;
  void* q_out;
  long long q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head;
  const void *q_norm, *k_norm;
  const float *cos, *sin;
  float eps;
  int n_heads, rot_dim, table_rows, interleaved;
  // keys and values come from a 16-bit pool of one layer with the same page table
  // (k and v are not read)
  const uint8_t* staged;
};
cudaError_t launch_cache_append(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAppend& a,
                                int* status, cudaStream_t s);

// Copies the rows behind the full pages of `len` positions of a fork (fmd_cache_fork, one).
cudaError_t launch_cache_fork_one(const CacheView& c, int layers, int* table, int src, int dst, int len, int page,
                                  cudaStream_t s);
// fmd_cache_compact
size_t cache_compact_workspace(int n_pages);
cudaError_t launch_cache_compact(const CacheView& c, int layers, int* table, const int* n_entries, void* workspace,
                                 int* n_used, int* status, cudaStream_t s);

struct CacheAttend {
  const void* q;
  void* out;
  long long q_row, q_head, out_row, out_head;
  float scale;
  int n_heads, window, sinks, max_rows;
};
// Units of a sequence in either form at most (32 keys each, and what stands for its fixed cost);
// the units of all kv heads are numbered in 32 bits.
inline long long cache_units(const CacheView& c) { return 2LL * c.max_pages + 16; }
// fmd_cache_decode.cu: at most 16 (row, head) pairs per kv head and sequence
bool cache_decode_fits(const CacheView& c, int n_heads, int max_rows);
size_t cache_decode_workspace(const CacheView& c, int n_heads, int max_rows);
cudaError_t launch_cache_decode(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAttend& a,
                                void* workspace, int* status, cudaStream_t s);

// the TMA map of a 16-bit cache's layer as [rows][head_dim], 64 x 64 boxes, 128-byte swizzle
bool cache_tensor_map(CUtensorMap* m, const CacheView& c, int layer);
// fmd_cache_chunk.cu: the others
size_t cache_chunk_workspace(const CacheView& c);
cudaError_t launch_cache_chunk(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAttend& a,
                               void* workspace, int* status, cudaStream_t s);

}  // namespace fmd
