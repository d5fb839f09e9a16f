// Attention over the paged cache with a window and sinks (include/fmd_cache.h).
#include <algorithm>

#include "fmd_cache.cuh"

namespace fmd {

namespace {

// One warp per (row, query head): lane l holds dims V l .. V l + V - 1 of the
// query and walks the visible keys with a running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_cache_attend(CacheView c, int layer, CacheRows r, CacheAttend a, int* status) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.y;
  if (i >= r.count()) return;
  int slot, p0, r0, n;
  r.get(i, slot, p0, r0, n);
  if (!cache_slot_ok(c, slot, status)) return;
  const int G = a.n_heads / c.kv_heads;
  for (long long w = (long long)blockIdx.x * 8 + warp; w < (long long)n * a.n_heads; w += (long long)gridDim.x * 8) {
    const int ri = (int)(w / a.n_heads), h = (int)(w % a.n_heads), kh = h / G;
    const int row = r0 + ri, pos = p0 + ri;
    if (pos < 0 || pos / kPageTokens >= c.max_pages) {
      cache_report(status, FMD_EOVERFLOW);
      continue;
    }
    const T* q = (const T*)a.q + row * a.q_row + h * a.q_head;
    float qv[V], o[V], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) qv[k] = Act<T>::to_f(q[lane * V + k]), o[k] = 0.f;
    const int first = a.window && pos >= a.window ? pos - a.window + 1 : 0;
    const int sinks = min(a.sinks, first);
    for (int j = sinks > 0 ? 0 : first; j <= pos; j = j + 1 == sinks ? first : j + 1) {
      const int page = cache_page(c, slot, j, status);
      if (page < 0) continue;
      float x[2][V];
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* blk = c.block(layer, page, kv, kh);
        const int pr = j % kPageTokens;
        for (int k = 0; k < V; ++k) {
          const int d = lane * V + k, e = d & 7;
          if (c.format == FMD_CACHE_Q4) {
            const int wi = kv == 0 ? ((d % 32) / 8) * (D / 32) + d / 32 : d / 8;
            const uint32_t word = ((const uint32_t*)(blk + pr * (D / 2)))[wi];
            const float sc = __half2float(((const __half*)(blk + kPageTokens * (D / 2)))[pr * (D / 32) + d / 32]);
            x[kv][k] = (float)((int)(word >> (4 * (kv == 0 ? (e >> 1) + 4 * (e & 1) : e)) & 15) - 8) * sc;
          } else {
            x[kv][k] = Act<T>::to_f(((const T*)blk)[pr * D + d]);
          }
        }
      }
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) s = fmaf(qv[k], x[0][k], s);
      s = warp_sum(s) * a.scale;
      const float mn = fmaxf(m, s), corr = expf(m - mn), p = expf(s - mn);
      l = l * corr + p;
      m = mn;
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = fmaf(p, x[1][k], o[k] * corr);
    }
    T* out = (T*)a.out + row * a.out_row + h * a.out_head;
#pragma unroll
    for (int k = 0; k < V; ++k) out[lane * V + k] = Act<T>::from_f(o[k] / l);
  }
}

}  // namespace

cudaError_t launch_cache_attend(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAttend& a,
                                void* workspace, int* status, cudaStream_t s) {
  if (cache_decode_fits(c, a.n_heads, a.max_rows)) return launch_cache_decode(bf16, c, layer, r, a, workspace, status, s);
  const int gx = (int)std::min<long long>(((long long)a.max_rows * a.n_heads + 7) / 8, 4096);
  const dim3 grid(gx, r.n_seqs);
  if (bf16) {
    if (c.head_dim == 128) k_cache_attend<__nv_bfloat16, 128><<<grid, 256, 0, s>>>(c, layer, r, a, status);
    else k_cache_attend<__nv_bfloat16, 64><<<grid, 256, 0, s>>>(c, layer, r, a, status);
  } else {
    if (c.head_dim == 128) k_cache_attend<__half, 128><<<grid, 256, 0, s>>>(c, layer, r, a, status);
    else k_cache_attend<__half, 64><<<grid, 256, 0, s>>>(c, layer, r, a, status);
  }
  return cudaPeekAtLastError();
}

}  // namespace fmd
