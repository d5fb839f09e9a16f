// The paged cache's row and page operators (include/fmd_cache.h): append, read,
// fork, copy and compact.
#include <algorithm>
#include <cstring>

#include "fmd_cache.cuh"

namespace fmd {

namespace {

// ---- append -------------------------------------------------------------------------
//
// One warp per (row, head); lane l holds dims V l .. V l + V - 1, V = D / 32.
template <typename T, int D, bool Q4>
__global__ void __launch_bounds__(256) k_cache_append(CacheView c, int layer, CacheRows r, CacheAppend a, int* status) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const int heads = a.n_heads + 2 * c.kv_heads;
  const int n_seqs = r.count();
  const int n_rows = r.row0 ? min(r.row0[n_seqs], r.n_rows) : min(n_seqs, r.n_rows);
  const long long works = (long long)n_rows * heads;
  for (long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); w < works; w += (long long)gridDim.x * 8) {
    const int row = (int)(w / heads);
    int head = (int)(w % heads);
    int lo = 0;
    if (r.row0) {
      int hi = n_seqs - 1;  // the last sequence that starts at or before the row
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (r.row0[mid] <= row) lo = mid;
        else hi = mid - 1;
      }
    } else {
      lo = row;
    }
    int slot, p0, r0, n;
    r.get(lo, slot, p0, r0, n);
    if (row < r0 || row >= r0 + n || !cache_slot_ok(c, slot, status)) continue;
    const int pos = p0 + row - r0;
    const int page = cache_page(c, slot, pos, status);
    if (page < 0) continue;
    if (a.rot_dim > 0 && pos >= a.table_rows) {
      cache_report(status, FMD_EOVERFLOW);
      continue;
    }
    const int part = head < a.n_heads ? 0 : head < a.n_heads + c.kv_heads ? 1 : 2;
    if (part) head = (head - a.n_heads) % c.kv_heads;
    const T* src = part == 0   ? (const T*)a.q + row * a.q_row + head * a.q_head
                   : part == 1 ? (const T*)a.k + row * a.k_row + head * a.k_head
                               : (const T*)a.v + row * a.v_row + head * a.v_head;
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = Act<T>::to_f(src[lane * V + i]);
    const T* nw = (const T*)(part == 0 ? a.q_norm : part == 1 ? a.k_norm : nullptr);
    if (nw) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
      const float rs = rsqrtf(warp_sum(ss) / D + a.eps);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = x[i] * rs * Act<T>::to_f(nw[lane * V + i]);
    }
    if (part < 2 && a.rot_dim > 0) {
      const float* cs = a.cos + (size_t)pos * (a.rot_dim / 2);
      const float* sn = a.sin + (size_t)pos * (a.rot_dim / 2);
      const int half = a.rot_dim / 2;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int d = lane * V + i;
        // the other half's element: rot_dim is a multiple of 8, so it sits at the same i
        const int other = a.interleaved ? lane : (d < half ? lane + half / V : lane - half / V);
        const float y = __shfl_sync(0xffffffffu, x[i], other & 31);
        if (d < a.rot_dim && !a.interleaved) {
          const int f = d < half ? d : d - half;
          x[i] = d < half ? x[i] * cs[f] - y * sn[f] : x[i] * cs[f] + y * sn[f];
        }
      }
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const int d = lane * V + i;
          if (d < a.rot_dim) {
            const float c0 = cs[d / 2], s0 = sn[d / 2], u = x[i], w0 = x[i + 1];
            x[i] = u * c0 - w0 * s0;
            x[i + 1] = w0 * c0 + u * s0;
          }
        }
      }
    }
    if (part == 0 || !Q4) {
      T* dst = part == 0 ? (T*)a.q_out + row * a.qo_row + head * a.qo_head
                         : (T*)c.block(layer, page, part - 1, head) + (size_t)(pos % kPageTokens) * D;
#pragma unroll
      for (int i = 0; i < V; ++i) dst[lane * V + i] = Act<T>::from_f(x[i]);
    } else {
      // the first value of largest magnitude of the lane's 32-dim block
      float m = 0.f;
      int at = 1 << 20;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        bad |= !(fabsf(x[i]) <= 3.4e38f);
        if (fabsf(x[i]) > fabsf(m)) m = x[i], at = lane * V + i;
      }
#pragma unroll
      for (int o = 16 / V; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oat = __shfl_xor_sync(0xffffffffu, at, o);
        if (fabsf(om) > fabsf(m) || (fabsf(om) == fabsf(m) && oat < at)) m = om, at = oat;
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
      }
      m = fminf(fmaxf(m, -65504.f), 65504.f);
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = m == 0.f ? 8.5f : __fdiv_rn(-8.f * x[i], m) + 8.5f;
        const uint32_t code = (uint32_t)fminf(fmaxf(floorf(t), 0.f), 15.f);
        const int e = (lane * V + i) & 7;
        word |= code << (4 * (part == 1 ? (e >> 1) + 4 * (e & 1) : e));
      }
#pragma unroll
      for (int o = 1; o < 8 / V; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
      uint8_t* blk = c.block(layer, page, part - 1, head);
      const int d0 = lane * V, pr = pos % kPageTokens;
      if (d0 % 8 == 0) {
        const int wi = part == 1 ? ((d0 % 32) / 8) * (D / 32) + d0 / 32 : d0 / 8;
        reinterpret_cast<uint32_t*>(blk + pr * (D / 2))[wi] = word;
      }
      if (d0 % 32 == 0)
        reinterpret_cast<__half*>(blk + kPageTokens * (D / 2))[pr * (D / 32) + d0 / 32] =
            bad ? __ushort_as_half(0x7fff) : __float2half_rn(m * -0.125f);
    }
  }
}

// ---- read ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) k_cache_read(CacheView c, int layer, CacheRows r, float* k, float* v, int* status) {
  const int n_seqs = r.count();
  const int n_rows = r.row0 ? min(r.row0[n_seqs], r.n_rows) : min(n_seqs, r.n_rows);
  const int chunks = D / 8;  // 8 values a thread
  const long long works = (long long)n_rows * 2 * c.kv_heads * chunks;
  for (long long w = (long long)blockIdx.x * blockDim.x + threadIdx.x; w < works;
       w += (long long)gridDim.x * blockDim.x) {
    const int ch = (int)(w % chunks);
    const int head = (int)(w / chunks % c.kv_heads);
    const int kv = (int)(w / (chunks * c.kv_heads) & 1);
    const int row = (int)(w / (2LL * chunks * c.kv_heads));
    int lo = r.row0 ? 0 : row;
    if (r.row0) {
      int hi = n_seqs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (r.row0[mid] <= row) lo = mid;
        else hi = mid - 1;
      }
    }
    int slot, p0, r0, n;
    r.get(lo, slot, p0, r0, n);
    if (row < r0 || row >= r0 + n || !cache_slot_ok(c, slot, status)) continue;
    const int pos = p0 + row - r0;
    const int page = cache_page(c, slot, pos, status);
    if (page < 0) continue;
    const uint8_t* blk = c.block(layer, page, kv, head);
    const int pr = pos % kPageTokens;
    float x[8];
    if (c.format == FMD_CACHE_Q4) {
      const int wi = kv == 0 ? (ch % 4) * (D / 32) + ch / 4 : ch;
      const uint32_t word = reinterpret_cast<const uint32_t*>(blk + pr * (D / 2))[wi];
      const float d =
          __half2float(reinterpret_cast<const __half*>(blk + kPageTokens * (D / 2))[pr * (D / 32) + ch / 4]);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = (float)((int)(word >> (4 * (kv == 0 ? (e >> 1) + 4 * (e & 1) : e)) & 15) - 8) * d;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(blk + ((size_t)pr * D + ch * 8) * 2);
      const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = c.format == FMD_CACHE_BF16 ? Act<__nv_bfloat16>::unpack2(uu[e]) : Act<__half>::unpack2(uu[e]);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
      }
    }
    float4* dst = reinterpret_cast<float4*>((kv ? v : k) + ((size_t)row * c.kv_heads + head) * D + ch * 8);
    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// ---- pages --------------------------------------------------------------------------

constexpr int kCopyBatch = 128;  // host pairs of one launch, passed by value
struct CopyList {
  int src[kCopyBatch], dst[kCopyBatch], rows[kCopyBatch];
};
struct ForkList {
  int src[kCopyBatch], dst[kCopyBatch], len[kCopyBatch], page[kCopyBatch];
};

// The first `rows` positions of a block: one prefix of the codes or values and,
// in 4 bits, one of the scales. Both start 16-byte aligned; a scale prefix is a
// multiple of 4 bytes, a code or value prefix of 32.
FMD_DEV void copy_block_rows(const CacheView& c, const uint8_t* src, uint8_t* dst, int rows, int tid, int nt) {
  const int rowb = c.format == FMD_CACHE_Q4 ? c.head_dim / 2 : c.head_dim * 2;
  for (int i = tid; i < rows * rowb / 16; i += nt) ((int4*)dst)[i] = ((const int4*)src)[i];
  if (c.format == FMD_CACHE_Q4) {
    const int off = kPageTokens * rowb, n = rows * (c.head_dim / 16) / 4;
    for (int i = tid; i < n; i += nt) ((int*)(dst + off))[i] = ((const int*)(src + off))[i];
  }
}

// grid (pairs, layers x 2 x kv heads)
__global__ void __launch_bounds__(128) k_cache_copy(CacheView c, CopyList l) {
  const int i = blockIdx.x, bk = blockIdx.y % (2 * c.kv_heads), layer = blockIdx.y / (2 * c.kv_heads);
  const int s = l.src[i], d = l.dst[i];
  copy_block_rows(c, c.block(layer, s, 0, 0) + bk * c.block_bytes(), c.block(layer, d, 0, 0) + bk * c.block_bytes(),
                  l.rows[i], threadIdx.x, blockDim.x);
}

__global__ void __launch_bounds__(128) k_cache_fork(CacheView c, int* table, ForkList l, int* status) {
  const int i = blockIdx.x, bk = blockIdx.y % (2 * c.kv_heads), layer = blockIdx.y / (2 * c.kv_heads);
  const int full = l.len[i] / kPageTokens, part = l.len[i] % kPageTokens;
  const int* from = table + (size_t)l.src[i] * c.max_pages;
  int* to = table + (size_t)l.dst[i] * c.max_pages;
  if (blockIdx.y == 0) {
    for (int k = threadIdx.x; k < full; k += blockDim.x) to[k] = from[k];
    if (threadIdx.x == 0 && part) to[full] = l.page[i];
  }
  if (part) {
    const int s = from[full];
    if (s < 0 || s >= c.n_pages) {
      cache_report(status, FMD_EINVAL);
      return;
    }
    copy_block_rows(c, c.block(layer, s, 0, 0) + bk * c.block_bytes(),
                    c.block(layer, l.page[i], 0, 0) + bk * c.block_bytes(), part, threadIdx.x, blockDim.x);
  }
}

// Compaction: the used pages as a bitmap, then each word's rank, then the moves.
__global__ void k_compact_mark(CacheView c, const int* n_entries, uint32_t* bits, int* status) {
  const int slot = blockIdx.x, n = min(n_entries[slot], c.max_pages);
  for (int k = threadIdx.x; k < n; k += blockDim.x) {
    const int p = c.page_table[(size_t)slot * c.max_pages + k];
    if (p == -1) continue;
    if (p < 0 || p >= c.n_pages) cache_report(status, FMD_EINVAL);
    else atomicOr(&bits[p >> 5], 1u << (p & 31));
  }
}

// One CTA: U, and for the i-th used page >= U and the i-th free page < U
// src[i], dst[i] and map[src] = dst. counts[0] = U, counts[1] = moves.
__global__ void __launch_bounds__(1024) k_compact_plan(int n_pages, const uint32_t* bits, int* map, int* src, int* dst,
                                                       int* counts, int* n_used) {
  __shared__ int s_warp[2][32], s_tot[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int words = (n_pages + 31) / 32;
  int mine = 0;
  for (int w = tid; w < words; w += 1024) mine += __popc(bits[w]);
  mine = (int)__reduce_add_sync(0xffffffffu, (unsigned)mine);
  if (lane == 0) s_warp[0][warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const int t = (int)__reduce_add_sync(0xffffffffu, (unsigned)s_warp[0][lane]);
    if (lane == 0) s_tot[0] = t;
  }
  __syncthreads();
  const int U = s_tot[0];
  int run_s = 0, run_d = 0;
  for (int w0 = 0; w0 < words; w0 += 1024) {
    const int w = w0 + tid;
    uint32_t b = 0, below = 0;  // bits of pages < U in this word
    if (w < words) {
      b = bits[w];
      const int first = w * 32;
      below = U >= first + 32 ? 0xffffffffu : U <= first ? 0u : (1u << (U - first)) - 1u;
    }
    const uint32_t sm = b & ~below, dm = ~b & below;
    const int ns = __popc(sm), nd = __popc(dm);
    int is = ns, id = nd;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, is, o), y = __shfl_up_sync(0xffffffffu, id, o);
      if (lane >= o) is += x, id += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[0][warp] = is, s_warp[1][warp] = id;
    __syncthreads();
    int bs = 0, bd = 0, ts = 0, td = 0;
    for (int k = 0; k < 32; ++k) {
      if (k < warp) bs += s_warp[0][k], bd += s_warp[1][k];
      ts += s_warp[0][k], td += s_warp[1][k];
    }
    int ps = run_s + bs + is - ns, pd = run_d + bd + id - nd;
    for (uint32_t m = sm; m; m &= m - 1) src[ps++] = w * 32 + __ffs(m) - 1;
    for (uint32_t m = dm; m; m &= m - 1) dst[pd++] = w * 32 + __ffs(m) - 1;
    run_s += ts;
    run_d += td;
  }
  __syncthreads();  // src and dst of every thread are visible to the CTA
  for (int i = tid; i < run_s; i += 1024) map[src[i]] = dst[i];
  if (tid == 0) {
    counts[0] = U;
    counts[1] = run_s;
    *n_used = U;
  }
}

__global__ void k_compact_remap(CacheView c, int* table, const int* n_entries, const int* map, const int* counts) {
  const int slot = blockIdx.x, n = min(n_entries[slot], c.max_pages), U = counts[0];
  for (int k = threadIdx.x; k < n; k += blockDim.x) {
    const int p = table[(size_t)slot * c.max_pages + k];
    if (p >= U && p < c.n_pages) table[(size_t)slot * c.max_pages + k] = map[p];
  }
}

__global__ void __launch_bounds__(256) k_compact_move(CacheView c, int layers, const int* src, const int* dst,
                                                      const int* counts) {
  const int n = counts[1];
  const size_t pb = c.page_bytes();
  const long long works = (long long)n * layers;
  for (long long w = blockIdx.x; w < works; w += gridDim.x) {
    const int i = (int)(w % n), layer = (int)(w / n);
    const int4* s = (const int4*)c.block(layer, src[i], 0, 0);
    int4* d = (int4*)c.block(layer, dst[i], 0, 0);
    for (size_t k = threadIdx.x; k < pb / 16; k += blockDim.x) d[k] = s[k];
  }
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace

cudaError_t launch_cache_append(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAppend& a,
                                int* status, cudaStream_t s) {
  const long long works = (long long)r.n_rows * (a.n_heads + 2 * c.kv_heads);
  const int grid = (int)std::min<long long>((works + 7) / 8, 148 * 8);
  auto go = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return c.format == FMD_CACHE_Q4
               ? launch(k_cache_append<T, D, true>, dim3(grid), dim3(256), 0, s, c, layer, r, a, status)
               : launch(k_cache_append<T, D, false>, dim3(grid), dim3(256), 0, s, c, layer, r, a, status);
  };
  auto dim = [&](auto t) {
    return c.head_dim == 128 ? go(t, std::integral_constant<int, 128>{}) : go(t, std::integral_constant<int, 64>{});
  };
  return bf16 ? dim(__nv_bfloat16{}) : dim(__half{});
}

}  // namespace fmd

// =====================================================================================
using namespace fmd;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Device memory of the current device (or managed memory).
bool on_current_device(const void* p) {
  cudaPointerAttributes a{};
  int dev = -1;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess || cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev);
}

int check_cache(const fmd_cache* c) {
  if (!c || !c->pool || !c->page_table || !aligned16(c->pool)) return FMD_EINVAL;
  if (c->format != FMD_CACHE_F16 && c->format != FMD_CACHE_BF16 && c->format != FMD_CACHE_Q4) return FMD_EINVAL;
  if (c->head_dim != 64 && c->head_dim != 128) return FMD_ENOTSUP;
  if (c->layers < 1 || c->n_pages < 1 || c->kv_heads < 1 || c->max_slots < 1 || c->max_pages_per_slot < 1)
    return FMD_EINVAL;
  // positions are 32-bit
  if ((int64_t)c->max_pages_per_slot * kPageTokens > INT32_MAX || c->kv_heads > 1024) return FMD_ENOTSUP;
  return FMD_OK;
}

int check_rows(const fmd_cache* c, int32_t layer, const fmd_cache_rows* r) {
  if (!r || layer < 0 || layer >= c->layers) return FMD_EINVAL;
  if (r->n_seqs < 0 || r->n_rows < 0 || r->max_rows < 0 || (!r->row0 && r->n_rows < r->n_seqs)) return FMD_EINVAL;
  if (r->n_seqs > 0 && (!r->slot || !r->pos0)) return FMD_EINVAL;
  return FMD_OK;
}

bool bad_stride(int64_t s) { return s < 0 || (s & 7); }

CacheView view_of(const fmd_cache* c) {
  return CacheView{(uint8_t*)c->pool, c->page_table, c->format,    c->n_pages,
                   c->kv_heads,       c->head_dim,   c->max_slots, c->max_pages_per_slot};
}
CacheRows rows_of(const fmd_cache_rows* r) {
  return CacheRows{r->slot, r->pos0, r->row0, nullptr, nullptr, r->n_seqs, r->n_rows};
}
int done(cudaError_t e) {
  if (e == cudaSuccess) return FMD_OK;
  cudaGetLastError();  // the call's own failure, returned here
  return FMD_EIO;
}

}  // namespace

extern "C" {

int64_t fmd_cache_block_bytes(int32_t format, int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return 0;
  if (format == FMD_CACHE_Q4) return (int64_t)kPageTokens * (head_dim / 2 + head_dim / 16);
  if (format == FMD_CACHE_F16 || format == FMD_CACHE_BF16) return (int64_t)kPageTokens * head_dim * 2;
  return 0;
}

int64_t fmd_cache_pool_bytes(const fmd_cache* c) {
  if (!c || c->layers < 1 || c->n_pages < 1 || c->kv_heads < 1) return 0;
  return (int64_t)c->layers * c->n_pages * 2 * c->kv_heads * fmd_cache_block_bytes(c->format, c->head_dim);
}

int fmd_cache_append(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows, const fmd_cache_append_args* a,
                     int32_t* status, void* stream) {
  int rc = check_cache(c);
  if (rc || (rc = check_rows(c, layer, rows))) return rc;
  if (!a || !a->k || !a->v || !aligned16(a->k) || !aligned16(a->v)) return FMD_EINVAL;
  if (a->dtype != FMD_DT_F16 && a->dtype != FMD_DT_BF16) return FMD_EINVAL;
  if (c->format != FMD_CACHE_Q4 && c->format != a->dtype) return FMD_EINVAL;
  if (a->n_heads < 0 || a->n_heads > 16384 || (a->n_heads > 0) != (a->q != nullptr) || (a->q && !a->q_out))
    return FMD_EINVAL;
  if (a->q && (!aligned16(a->q) || !aligned16(a->q_out))) return FMD_EINVAL;
  if (a->rot_dim < 0 || a->rot_dim > c->head_dim || a->rot_dim % 8) return FMD_EINVAL;
  if (a->rot_dim > 0 && (!a->cos_table || !a->sin_table || a->table_rows < 1 || !aligned16(a->cos_table) ||
                         !aligned16(a->sin_table)))
    return FMD_EINVAL;
  if ((a->q_norm || a->k_norm) && !(a->eps >= 0.f)) return FMD_EINVAL;
  if ((a->q_norm && !aligned16(a->q_norm)) || (a->k_norm && !aligned16(a->k_norm))) return FMD_EINVAL;
  for (int64_t s : {a->k_row, a->k_head, a->v_row, a->v_head})
    if (bad_stride(s)) return FMD_EINVAL;
  if (a->q)
    for (int64_t s : {a->q_row, a->q_head, a->q_out_row, a->q_out_head})
      if (bad_stride(s)) return FMD_EINVAL;
  if (rows->n_seqs == 0 || rows->n_rows == 0) return FMD_OK;
  if (!on_current_device(c->pool) || !on_current_device(a->k)) return FMD_EINVAL;
  CacheAppend p{a->q,      a->k,      a->v,     a->q_out,     a->q_row,     a->q_head, a->k_row,
                a->k_head, a->v_row,  a->v_head, a->q_out_row, a->q_out_head, a->q_norm, a->k_norm,
                a->cos_table, a->sin_table, a->eps, a->n_heads, a->rot_dim, a->table_rows, a->interleaved};
  return done(launch_cache_append(a->dtype == FMD_DT_BF16, view_of(c), layer, rows_of(rows), p, status,
                                  (cudaStream_t)stream));
}

int fmd_cache_read(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows, float* k, float* v, int32_t* status,
                   void* stream) {
  int rc = check_cache(c);
  if (rc || (rc = check_rows(c, layer, rows))) return rc;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return FMD_EINVAL;
  if (rows->n_seqs == 0 || rows->n_rows == 0) return FMD_OK;
  if (!on_current_device(c->pool) || !on_current_device(k)) return FMD_EINVAL;
  const long long works = (long long)rows->n_rows * 2 * c->kv_heads * (c->head_dim / 8);
  const int grid = (int)std::min<long long>((works + 255) / 256, 148 * 16);
  return done(launch(c->head_dim == 128 ? k_cache_read<128> : k_cache_read<64>, dim3(grid), dim3(256), 0,
                     (cudaStream_t)stream, view_of(c), layer, rows_of(rows), k, v, status));
}

int64_t fmd_cache_attend_workspace(const fmd_cache* c, int32_t n_heads, int32_t n_seqs, int32_t max_rows) {
  if (check_cache(c) || n_heads < 1 || n_heads % c->kv_heads || n_seqs < 1 || max_rows < 1) return 0;
  const CacheView v = view_of(c);
  return (int64_t)(cache_decode_fits(v, n_heads, max_rows) ? cache_decode_workspace(v, n_heads, max_rows)
                                                           : cache_chunk_workspace(v, n_heads, n_seqs, max_rows));
}

int fmd_cache_attend(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows, const fmd_cache_attend_args* a,
                     void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  int rc = check_cache(c);
  if (rc || (rc = check_rows(c, layer, rows))) return rc;
  if (!a || !a->q || !a->out || !aligned16(a->q) || !aligned16(a->out)) return FMD_EINVAL;
  if (a->dtype != FMD_DT_F16 && a->dtype != FMD_DT_BF16) return FMD_EINVAL;
  if (c->format != FMD_CACHE_Q4 && c->format != a->dtype) return FMD_EINVAL;
  if (a->n_heads < 1 || a->n_heads % c->kv_heads) return FMD_EINVAL;
  const int group = a->n_heads / c->kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8 && group != 16) return FMD_ENOTSUP;
  if (a->window < 0 || a->sinks < 0 || !(a->scale > 0.f) || !(a->scale <= 3.4e38f)) return FMD_EINVAL;
  for (int64_t s : {a->q_row, a->q_head, a->out_row, a->out_head})
    if (bad_stride(s)) return FMD_EINVAL;
  if (rows->n_seqs == 0 || rows->n_rows == 0 || rows->max_rows == 0) return FMD_OK;
  const int64_t need = fmd_cache_attend_workspace(c, a->n_heads, rows->n_seqs, rows->max_rows);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return FMD_EINVAL;
  if (!on_current_device(c->pool) || !on_current_device(a->q)) return FMD_EINVAL;
  CacheAttend p{a->q,     a->out,     a->q_row,  a->q_head, a->out_row, a->out_head,
                a->scale, a->n_heads, a->window, a->sinks,  rows->max_rows};
  const CacheView v = view_of(c);
  return done((cache_decode_fits(v, a->n_heads, rows->max_rows) ? launch_cache_decode : launch_cache_chunk)(
      a->dtype == FMD_DT_BF16, v, layer, rows_of(rows), p, workspace, status, (cudaStream_t)stream));
}

int fmd_cache_copy_pages(const fmd_cache* c, int32_t n, const int32_t* src, const int32_t* dst, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!src || !dst))) return FMD_EINVAL;
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= c->n_pages || dst[i] < 0 || dst[i] >= c->n_pages) return FMD_EINVAL;
  if (n == 0) return FMD_OK;
  if (!on_current_device(c->pool)) return FMD_EINVAL;
  for (int i = 0; i < n; i += kCopyBatch) {
    CopyList l;
    const int m = std::min(kCopyBatch, n - i);
    std::memcpy(l.src, src + i, m * sizeof(int));
    std::memcpy(l.dst, dst + i, m * sizeof(int));
    for (int k = 0; k < m; ++k) l.rows[k] = kPageTokens;
    const cudaError_t e = launch(k_cache_copy, dim3(m, c->layers * 2 * c->kv_heads), dim3(128), 0,
                                 (cudaStream_t)stream, view_of(c), l);
    if (e != cudaSuccess) return done(e);
  }
  return FMD_OK;
}

int fmd_cache_fork(const fmd_cache* c, int32_t n, const int32_t* src_slot, const int32_t* dst_slot, const int32_t* len,
                   const int32_t* new_page, int32_t* status, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!src_slot || !dst_slot || !len || !new_page))) return FMD_EINVAL;
  for (int i = 0; i < n; ++i) {
    if (src_slot[i] < 0 || src_slot[i] >= c->max_slots || dst_slot[i] < 0 || dst_slot[i] >= c->max_slots ||
        src_slot[i] == dst_slot[i] || len[i] < 0)
      return FMD_EINVAL;
    if (len[i] > c->max_pages_per_slot * kPageTokens) return FMD_EOVERFLOW;
    if (len[i] % kPageTokens && (new_page[i] < 0 || new_page[i] >= c->n_pages)) return FMD_EINVAL;
  }
  if (n == 0) return FMD_OK;
  if (!on_current_device(c->pool)) return FMD_EINVAL;
  for (int i = 0; i < n; i += kCopyBatch) {
    ForkList l;
    const int m = std::min(kCopyBatch, n - i);
    std::memcpy(l.src, src_slot + i, m * sizeof(int));
    std::memcpy(l.dst, dst_slot + i, m * sizeof(int));
    std::memcpy(l.len, len + i, m * sizeof(int));
    std::memcpy(l.page, new_page + i, m * sizeof(int));
    const cudaError_t e = launch(k_cache_fork, dim3(m, c->layers * 2 * c->kv_heads), dim3(128), 0,
                                 (cudaStream_t)stream, view_of(c), c->page_table, l, status);
    if (e != cudaSuccess) return done(e);
  }
  return FMD_OK;
}

// bitmap, map, src, dst, counts
int64_t fmd_cache_compact_workspace(const fmd_cache* c) {
  if (!c || c->n_pages < 1) return 0;
  const int64_t words = ((int64_t)c->n_pages + 31) / 32;
  return 4 * (words + 3 * (int64_t)c->n_pages + 4);
}

int fmd_cache_compact(const fmd_cache* c, const int32_t* n_entries, void* workspace, int64_t workspace_bytes,
                      int32_t* n_used, int32_t* status, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!n_entries || !workspace || !n_used || workspace_bytes < fmd_cache_compact_workspace(c) || !aligned16(workspace))
    return FMD_EINVAL;
  if (!on_current_device(c->pool) || !on_current_device(workspace)) return FMD_EINVAL;
  const size_t words = ((size_t)c->n_pages + 31) / 32, P = c->n_pages;
  uint32_t* bits = (uint32_t*)workspace;
  int *map = (int*)bits + words, *src = map + P, *dst = src + P, *counts = dst + P;
  cudaStream_t s = (cudaStream_t)stream;
  const CacheView v = view_of(c);
  cudaError_t e = cudaMemsetAsync(bits, 0, words * 4, s);
  if (e == cudaSuccess) e = launch(k_compact_mark, dim3(c->max_slots), dim3(256), 0, s, v, n_entries, bits, status);
  if (e == cudaSuccess) e = launch(k_compact_plan, dim3(1), dim3(1024), 0, s, c->n_pages, bits, map, src, dst, counts, n_used);
  if (e == cudaSuccess)
    e = launch(k_compact_remap, dim3(c->max_slots), dim3(256), 0, s, v, c->page_table, n_entries, map, counts);
  if (e == cudaSuccess) e = launch(k_compact_move, dim3(148 * 8), dim3(256), 0, s, v, c->layers, src, dst, counts);
  return done(e);
}

}  // extern "C"
