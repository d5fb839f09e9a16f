// Attention of a few rows per sequence over the paged cache: the decode form
// of fmd_cache_attend, for at most 16 (row, query head) pairs per kv head.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j
//
// over the visible keys j of each row, in one pass: a running reference m, the
// sum and o are kept in f32 and rescaled when a score exceeds m by more than
// 2^8. The bound is the cache's bytes: visible keys x 2 x head_dim x 2 (16 bits)
// or x 9/16 (4 bits), each read once per (sequence, kv head).
//
// Split: the (sequence, kv head) segments, each the units of 64 (4 bits: 32) keys
// that its rows see (those of the sinks, then those of the window), form one
// sequence of T units; CTA c of G takes units [c T / G, (c + 1) T / G), whatever
// the lengths. A segment cut by CTA boundaries leaves (m, l, o) partials in the
// workspace; the last of its CTAs to arrive merges them in CTA order, so results
// do not depend on timing.
//
// The products are transposed, keys or dims on the 16-row side and the up to 8
// query pairs on the 8-column side of mma.sync m16n8k16: half the instructions
// and accumulators of queries on the 16-row side, most of whose rows would be
// empty. (tcgen05's smallest tile has 64 rows and operands in shared memory: the
// 4-bit codes would have to be written back there in 16 bits, more traffic than
// the cache itself.)
//   S^T = K Q^T: A = 16 keys x 16 dims, B = the queries.
//   O^T += V^T P^T: A = 16 dims x 16 keys, B = P^T, turned with movmatrix.
//
// Measured (8 kv heads of 128, 16 query heads, launches back to back): 64 sequences of 8,192
// positions 326 us from 16 bits, 6.6 TB/s, and 166 us from 4 bits, 3.6 TB/s; one sequence over
// 4,096 positions 11.6 us (16 bits), over 16,384 18 us (4 bits), of which launch, lookup and
// first loads are 6 and the merge of 34 and 74 pieces 4 and 6.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <float.h>
#include <limits.h>

#include <algorithm>

#include "fmd_cache.cuh"
#include "fmd_kernels.cuh"

namespace fmd {

namespace {

constexpr int kDcSeqs = 256;      // sequences of one launch at most
// Merge counters of a launch, [sequences][kv heads]: at the same place in every
// workspace, since they are zero between calls of any shape.
constexpr int kDcCounters = 16384;
constexpr uint32_t kDcWait = 1u << 22;
constexpr float kDcHeadroom = 8.f;  // log2: how far a score may exceed the reference

struct DcArgs {
  CacheRows r;
  CacheAttend a;
  float* part;      // [2 x grid][rows][D + 4] partials of cut segments
  int* counters;    // [sequences][kv heads], zero between calls
  int seq0, seqs;   // the sequences of this launch
  int tile_rows;    // (row, head) pairs of a segment at most
  uint32_t f64;     // f16 pair (64, 64)
  int stages, red_off, red_row;  // ring stages, merge buffer: its offset, its floats per pair
};

// A launch's sequences: units before each, slot, first position, first row, rows.
struct DcSeqs {
  int prefix[kDcSeqs + 1], slot[kDcSeqs], pos[kDcSeqs], row[kDcSeqs], cnt[kDcSeqs];
  int last;  // this CTA merges the segment
};

FMD_DEV uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
FMD_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// CTA whose range [c T / G, (c + 1) T / G) holds unit x.
FMD_DEV int dc_cta(long long x, long long T, int G) { return (int)(((x + 1) * G - 1) / T); }

// The keys of a sequence whose first row is at p0 as units of K: kSetup units
// without keys, which stand for what a segment costs beside its keys (its queries
// and its merge: a CTA's second piece took 5.5 us and more, a unit of 32 keys 0.7),
// so that ranges over short segments are not the last to finish (64 streams of
// 300 .. 16,384 positions in 4 bits: 89.5 us with 4 units, 84.5 with 7 or 10); then
// `sinks` units from position 0, then units from unit `w0` on.
template <int K> struct DcKeys {
  static constexpr int kSetup = K == 32 ? 8 : 1;
  int sinks, w0;
  FMD_DEV DcKeys(const CacheAttend& a, int p0) {
    const int first = a.window && p0 >= a.window ? p0 - a.window + 1 : 0;
    w0 = first / K;
    sinks = (min(a.window ? a.sinks : 0, w0 * K) + K - 1) / K;
  }
  FMD_DEV int unit(int j) const { return j < kSetup ? -1 : j - kSetup < sinks ? j - kSetup : w0 + j - kSetup - sinks; }
};

// Reads the launch's sequences into shared memory (all threads).
template <int K, int THREADS>
FMD_DEV void dc_plan(DcSeqs& q, const DcArgs& p, const CacheView& c, int ns, int* status) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < ns; i += THREADS) {
    int slot, p0, r0, n;
    p.r.get(p.seq0 + i, slot, p0, r0, n);
    int units = 0;
    if (n > 0 && cache_slot_ok(c, slot, status)) {
      if (n > p.a.max_rows || p0 < 0 || p0 > c.max_pages * kPageTokens - n) {
        cache_report(status, n > p.a.max_rows ? FMD_EINVAL : FMD_EOVERFLOW);
      } else {
        const DcKeys<K> k(p.a, p0);
        units = k.kSetup + k.sinks + (p0 + n - 1) / K - k.w0 + 1;
      }
    }
    q.prefix[i] = units;
    q.slot[i] = slot;
    q.pos[i] = p0;
    q.row[i] = r0;
    q.cnt[i] = n;
  }
  __syncthreads();
  if (tid < 32) {
    constexpr int PER = kDcSeqs / 32;
    int loc[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = lane * PER + k;
      loc[k] = r < ns ? q.prefix[r] : 0;
      sum += loc[k];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int run = incl - sum;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = lane * PER + k;
      if (r < ns) q.prefix[r] = run;
      run += loc[k];
    }
    if (lane == 31) q.prefix[ns] = incl;
  }
  __syncthreads();
}

// Sequence r, kv head h and unit j of unit x: the last sequence with units that
// starts at or before it.
FMD_DEV void dc_locate(const DcSeqs& q, int ns, int H, long long x, int& r, int& h, int& j) {
  int lo = 0, hi = ns - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((long long)H * q.prefix[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  r = lo;
  const int tr = q.prefix[r + 1] - q.prefix[r];
  const int off = (int)(x - (long long)H * q.prefix[r]);
  h = off / tr;
  j = off - h * tr;
}

FMD_DEV int dc_page(const DcSeqs& q, const CacheView& c, int r, int index, int* status) {
  const int page = c.page_table[(size_t)q.slot[r] * c.max_pages + index];
  if (page >= 0 && page < c.n_pages) return page;
  cache_report(status, FMD_EINVAL);
  return -1;
}

// A piece of a segment: units of segment (r, h), which has `units`; `x` is the
// segment's first unit among all T, [x0, x1) this CTA's.
struct DcPiece {
  int r, h, units, nq;
  bool inside;  // the whole segment lies in this CTA
  long long seg0, x0, T;
  int G;
};

// Merges the four warps' (o, m, l) of a piece, in `red` as [warp][pair][D + 2];
// writes the output, or the piece's partial, and, as the last CTA of a cut
// segment, the output from its partials. 128 threads, after their stores to red.
template <typename T, int D>
FMD_DEV void dc_merge(float* red, DcSeqs& q, const DcArgs& p, const DcPiece& s, int H, int gs, bool aborted) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int rs = D + 4;     // floats of a partial's row: o, m, l and two to keep 16 bytes
  constexpr int ls = D + 2;     // of a warp's row in `red`
  auto out_at = [&](int row, int d0) {
    return (T*)p.a.out + (size_t)(q.row[s.r] + (row >> gs)) * p.a.out_row +
           (size_t)((s.h << gs) + (row & ((1 << gs) - 1))) * p.a.out_head + d0;
  };
  named_sync(1, 128);
  const int pslot = 2 * (int)blockIdx.x + (s.seg0 < s.x0 ? 0 : 1);
  for (int i = tid; i < s.nq * (D / 2); i += 128) {
    const int row = i / (D / 2), d0 = (i % (D / 2)) * 2;
    float mm[4], Mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) Mx = fmaxf(Mx, mm[w] = red[(size_t)(w * p.tile_rows + row) * ls + D]);
    const float base = Mx == -INFINITY ? 0.f : Mx;
    float L = 0.f, A0 = 0.f, A1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float* rw = red + (size_t)(w * p.tile_rows + row) * ls;
      const float f = ex2(mm[w] - base);  // 0 for a warp that saw nothing
      L = fmaf(rw[D + 1], f, L);
      A0 = fmaf(rw[d0], f, A0);
      A1 = fmaf(rw[d0 + 1], f, A1);
    }
    if (s.inside) {
      if (!aborted) *reinterpret_cast<uint32_t*>(out_at(row, d0)) = Act<T>::pack2(A0 / L, A1 / L);
    } else {
      float* pt = p.part + ((size_t)pslot * p.tile_rows + row) * rs;
      *reinterpret_cast<float2*>(pt + d0) = make_float2(A0, A1);
      if (d0 == 0) *reinterpret_cast<float2*>(pt + D) = make_float2(Mx, L);
    }
  }
  if (!s.inside) {
    const int cf = dc_cta(s.seg0, s.T, s.G), cl = dc_cta(s.seg0 + s.units - 1, s.T, s.G);
    int* counter = &p.counters[(size_t)s.r * H + s.h];
    named_sync(1, 128);
    if (tid == 0) {
      __threadfence();
      q.last = atomicAdd(counter, 1) == cl - cf;
      if (q.last) __threadfence();
    }
    named_sync(1, 128);
    if (q.last) {
      // weights of the pieces (one warp per pair), then the weighted sums
      const int np = cl - cf + 1, ws = p.red_row;  // floats of `red` per pair, > pieces
      auto piece = [&](int k) {
        return p.part + (size_t)(2 * (cf + k) + (k == 0 ? 1 : 0)) * p.tile_rows * rs;
      };
      for (int row = warp; row < s.nq; row += 4) {
        float Mx = -INFINITY, L = 0.f;
        float2 ml[4];  // the first 128 pieces' (m, l), loaded together
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = lane + 32 * i;
          ml[i] = k < np ? __ldcg(reinterpret_cast<const float2*>(piece(k) + row * rs + D)) : make_float2(-INFINITY, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) Mx = fmaxf(Mx, ml[i].x);
        for (int k = lane + 128; k < np; k += 32) Mx = fmaxf(Mx, __ldcg(piece(k) + row * rs + D));
        Mx = warp_max(Mx);
        const float base = Mx == -INFINITY ? 0.f : Mx;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = ex2(ml[i].x - base);
          if (lane + 32 * i < np) red[row * ws + lane + 32 * i] = f;
          L = fmaf(ml[i].y, f, L);
        }
        for (int k = lane + 128; k < np; k += 32) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(piece(k) + row * rs + D));
          const float f = ex2(v.x - base);
          red[row * ws + k] = f;
          L = fmaf(v.y, f, L);
        }
        L = warp_sum(L);
        if (lane == 0) red[row * ws + np] = L;
      }
      named_sync(1, 128);
      // four dims a thread; where that leaves threads, groups of them share the pieces
      // (one stream over 4,096 keys: 12.5 us, 13.5 without groups)
      const int work = s.nq * (D / 4), groups = max(1, 128 / work);
      float4* join = reinterpret_cast<float4*>(red + p.tile_rows * ws);
      for (int i0 = 0; i0 < work; i0 += 128) {
        const int grp = groups > 1 ? tid / work : 0, i = groups > 1 ? tid - grp * work : i0 + tid;
        const int row = i / (D / 4), d0 = (i % (D / 4)) * 4;
        const float* w = red + row * ws;
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
        if (grp < groups && i < work) {
          const size_t step = (size_t)2 * p.tile_rows * rs * groups;
          const float* pt = p.part + (size_t)2 * (cf + grp) * p.tile_rows * rs + row * rs + d0;
#pragma unroll 16
          for (int k = grp; k < np; k += groups, pt += step) {
            // the segment's first piece is its CTA's second slot
            const float4 x = __ldcg(reinterpret_cast<const float4*>(pt + (k == 0 ? p.tile_rows * rs : 0)));
            const float f = w[k];
            A.x = fmaf(x.x, f, A.x);
            A.y = fmaf(x.y, f, A.y);
            A.z = fmaf(x.z, f, A.z);
            A.w = fmaf(x.w, f, A.w);
          }
        }
        if (groups > 1) {
          join[tid] = A;
          named_sync(1, 128);
          for (int k = 1; grp == 0 && k < groups; ++k) {
            const float4 x = join[tid + k * work];
            A.x += x.x, A.y += x.y, A.z += x.z, A.w += x.w;
          }
        }
        if (grp == 0 && i < work && !aborted) {
          const float L = w[np];
          *reinterpret_cast<uint2*>(out_at(row, d0)) = make_uint2(Act<T>::pack2(A.x / L, A.y / L), Act<T>::pack2(A.z / L, A.w / L));
        }
      }
      if (tid == 0) *counter = 0;
    }
  }
  named_sync(1, 128);  // `red` is used again
}

// A warp's scores of U steps of 16 keys become P: sc (raw, keys g and g + 8 x
// columns 2 t, 2 t + 1) is scaled, hidden keys drop out, the reference moves
// when it must (with l and o), and P^T's B fragments come back in pb (HILO: its
// rounding error in pl). vis: bit masks of this thread's value pairs.
template <typename M, int U, int MT, int NT, bool HILO>
FMD_DEV void dc_softmax(float (&sc)[NT][U][4], const float (&sl)[NT][2], float (&m)[NT][2], float (&l)[NT][2],
                        float (&o)[NT][MT][4], uint32_t (&pb)[NT][U][2], uint32_t (&pl)[HILO ? NT : 1][U][2],
                        uint32_t (&vis)[U][2], bool whole, int k0, int p0, int p1, int W, int S, int gs, float pscale) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[n][u][e] *= sl[n][e & 1];
#pragma unroll
  for (int u = 0; u < U; ++u) vis[u][0] = vis[u][1] = 0xffffffffu;
  if (!whole) {
    auto seen = [&](int k, int lo, int hi) { return k <= hi && (W == 0 || k > lo - W || k < S); };
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pos = p0 + ((n * 8 + 2 * t + (e & 1)) >> gs);
          if (!seen(k0 + u * 16 + g + (e >> 1) * 8, pos, pos)) sc[n][u][e] = -INFINITY;
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!seen(k0 + u * 16 + 2 * t + (e & 1) + (e >> 1) * 8, p0, p1))
          vis[u][e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
    }
  }
  float mx[NT][2];
  bool up = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mx[n][k] = fmaxf(sc[n][0][k], sc[n][0][2 + k]);
#pragma unroll
      for (int u = 1; u < U; ++u) mx[n][k] = fmaxf(mx[n][k], fmaxf(sc[n][u][k], sc[n][u][2 + k]));
      up |= mx[n][k] > m[n][k] + kDcHeadroom;
    }
  if (__any_sync(0xffffffffu, up)) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = mx[n][k];
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float mn = fmaxf(m[n][k], x);
        const float f = mn == -INFINITY ? 1.f : ex2(m[n][k] - mn);
        m[n][k] = mn;
        l[n][k] *= f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i][k] *= f, o[n][i][2 + k] *= f;
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float base[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) base[k] = m[n][k] == -INFINITY ? 0.f : m[n][k] - pscale;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float e4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        e4[e] = ex2(sc[n][u][e] - base[e & 1]);
        l[n][e & 1] += e4[e];
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t hi = Act<M>::pack2(e4[2 * b], e4[2 * b + 1]);
        pb[n][u][b] = movmatrix_t(hi);
        if constexpr (HILO) {
          const float2 f = Act<M>::unpack2(hi);
          pl[n][u][b] = movmatrix_t(Act<M>::pack2(e4[2 * b] - f.x, e4[2 * b + 1] - f.y));
        }
      }
    }
  }
}

// A warp's accumulators into the merge buffer. DIM(i, e): the dim of row g + 8 e
// of output tile i.
template <int D, int NT, typename Dim>
FMD_DEV void dc_store(float* red, int tile_rows, int nq, const float (&o)[NT][D / 16][4], const float (&m)[NT][2],
                      const float (&l)[NT][2], Dim dim) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float lw = l[n][k];
      lw += __shfl_xor_sync(0xffffffffu, lw, 4);
      lw += __shfl_xor_sync(0xffffffffu, lw, 8);
      lw += __shfl_xor_sync(0xffffffffu, lw, 16);
      const int col = n * 8 + 2 * t + k;
      if (col < nq) {
        float* rw = red + (size_t)(warp * tile_rows + col) * (D + 2);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) rw[dim(i, e)] = o[n][i][2 * e + k];
        if (g == 0) {
          rw[D] = m[n][k];
          rw[D + 1] = lw;
        }
      }
    }
}

// ---- 16 bits ------------------------------------------------------------------------
//
// One producer warp looks up pages and keeps a ring of page tiles in flight (2D
// TMA with the 128-byte swizzle, so that ldmatrix is conflict-free); four
// consumer warps take 16 keys of every tile each. P goes in as two terms, so that its
// rounding (half a step: 2^-9 for bf16, 2^-12 for f16) does not show: the products are not
// the bound. Error against 64 bits in f16 2.1e-4 of the output, that of its one rounding;
// 2.9e-4 with one term, 71.5 us instead of 72 for the 64 streams below.
// 64 streams of 300 .. 16,384 positions over their newest 2,048 and 64 sinks: 72 us,
// 408 MB at 5.7 TB/s. At head_dim 128 more than 8 pairs spill 36 bytes a thread.

constexpr int kDc16Threads = 160;

// Swizzled byte offset of 16-byte chunk ch (of D / 8) of row `row` in a [64][D] tile.
FMD_DEV uint32_t dc_swz(int row, int ch) {
  return (uint32_t)((ch >> 3) * 8192 + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
}

// NT: 8-column tiles of (row, head) pairs.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kDc16Threads, 2)
    k_cache_decode(const __grid_constant__ CUtensorMap tmap, CacheView c, DcArgs p, int* status) {
  constexpr int KS = D / 16;  // 16-wide steps of the head
  constexpr int MT = D / 16;  // 16-dim tiles of the output
  constexpr int BLK = 64 * D * 2;
  constexpr float kPScale = Act<T>::kIsBf16 ? 0.f : 7.f;  // log2 factor of P: f16 keeps what is 2^-21 of the reference

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float* red = reinterpret_cast<float*>(smem + p.red_off);
  __shared__ DcSeqs q;
  __shared__ __align__(8) uint64_t full[8], empty[8];
  __shared__ int s_bad[8];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int stages = p.stages, H = c.kv_heads;
  griddep_wait();
  griddep_launch();
  const int ns = min(p.r.count() - p.seq0, p.seqs);
  if (ns <= 0) return;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_barrier_init();
    prefetch_tmap(&tmap);
  }
  dc_plan<64, kDc16Threads>(q, p, c, ns, status);
  const long long T_ = (long long)H * q.prefix[ns];
  const int G = (int)min((long long)gridDim.x, T_), cta = blockIdx.x;
  if (cta >= G) return;
  const long long x0 = (long long)cta * T_ / G, x1 = (long long)(cta + 1) * T_ / G;
  const int ntl = (int)(x1 - x0);

  if (warp == 4) {
    // ---------------- producer ----------------
    bool ok = true;
    int issued = 0, s = 0, round = 0;  // tile `issued` goes to stage s, used `round` times before
    for (int b0 = 0; b0 < ntl && ok; b0 += 32) {
      int lh = 0, lpage = -1;
      if (b0 + lane < ntl) {
        int lr, lj;
        dc_locate(q, ns, H, x0 + b0 + lane, lr, lh, lj);
        const int u = DcKeys<64>(p.a, q.pos[lr]).unit(lj);
        if (u >= 0) lpage = dc_page(q, c, lr, u, status);
      }
      const int cnt = min(32, ntl - b0);
      for (int i = 0; i < cnt; ++i) {
        const int h = __shfl_sync(0xffffffffu, lh, i), page = __shfl_sync(0xffffffffu, lpage, i);
        if (round > 0 && !mbar_wait_warp(&empty[s], (round - 1) & 1, kDcWait)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          s_bad[s] = page < 0;
          if (page < 0) {
            mbar_arrive(&full[s]);
          } else {
            uint8_t* dst = smem + s * 2 * BLK;
            mbar_arrive_expect_tx(&full[s], 2 * BLK);
            const int yk = (page * 2 * H + h) * kPageTokens, yv = yk + H * kPageTokens;
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
              tma_load_2d(dst + b * 8192, &tmap, b * 64, yk, &full[s]);
              tma_load_2d(dst + BLK + b * 8192, &tmap, b * 64, yv, &full[s]);
            }
          }
        }
        __syncwarp();
        ++issued;
        if (++s == stages) s = 0, ++round;
      }
    }
    if (lane == 0) {
      if (!ok) report_timeout(status, kSiteCacheDecode);
      // copies in flight land before the CTA retires, whatever the consumers do (bounded)
      for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
        mbar_wait_bounded(&full[i % stages], (i / stages) & 1, kDcWait);
    }
    return;
  }

  // ---------------- consumers ----------------
  bool aborted = false;
  const int gs = __ffs(p.a.n_heads / H) - 1;  // log2 of the query heads of a kv head
  const int W = p.a.window, S = W ? p.a.sinks : 0;
  int cr, ch, cj;
  dc_locate(q, ns, H, x0, cr, ch, cj);
  int ctr = q.prefix[cr + 1] - q.prefix[cr];
  uint32_t qf[NT][KS][2];
  float sl[NT][2], o[NT][MT][4], m[NT][2], l[NT][2];
  int s = 0, phase = 0;
  for (int x = 0; x < ntl;) {
    // a piece: tiles cj .. cj + len - 1 of segment (cr, ch)
    const int len = min(ctr - cj, ntl - x);
    const int nq = q.cnt[cr] << gs, p0 = q.pos[cr], p1 = p0 + q.cnt[cr] - 1;
    const DcKeys<64> keys(p.a, p0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
      sl[n][0] = sl[n][1] = p.a.scale * 1.4426950408889634f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      const int pr = n * 8 + g;  // this thread's column of the B fragments
      const T* src = (const T*)p.a.q + (size_t)(q.row[cr] + (pr >> gs)) * p.a.q_row +
                     (size_t)((ch << gs) + (pr & ((1 << gs) - 1))) * p.a.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          qf[n][ks][b] = pr < nq ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + b * 8 + 2 * t) : 0u;
    }
    for (int j = cj; j < cj + len; ++j) {
      // one outcome for the warp: what follows is warp-wide
      if (!aborted && !mbar_wait_warp(&full[s], phase, kDcWait)) aborted = true;
      // keys k0 .. k0 + 15 of this warp
      const int k0 = keys.unit(j) * 64 + warp * 16;
      const bool whole = k0 + 15 <= p0 && (W == 0 || k0 > p1 - W || k0 + 15 < S);
      const bool any = k0 <= p1 && (W == 0 || k0 + 15 > p0 - W || k0 < S);
      if (!aborted && any && !s_bad[s]) {
        const uint32_t ka = smem_u32(smem + s * 2 * BLK), va = ka + BLK;
        float sc[NT][1][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][0][0] = sc[n][0][1] = sc[n][0][2] = sc[n][0][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t a[4];
          ldmatrix_x4(a, ka + dc_swz(warp * 16 + (lane & 15), 2 * ks + (lane >> 4)));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<T>(sc[n][0], a, qf[n][ks][0], qf[n][ks][1]);
        }
        uint32_t pb[NT][1][2], pl[NT][1][2], vis[1][2];
        dc_softmax<T, 1, MT, NT, true>(sc, sl, m, l, o, pb, pl, vis, whole, k0, p0, p1, W, S, gs, kPScale);
        // matrices: (keys 0-7, dims 0-7), (keys 0-7, dims 8-15), (keys 8-15, dims 0-7), ...
        const int row = warp * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t a[4];
          ldmatrix_x4_trans(a, va + dc_swz(row, 2 * i + ((lane >> 3) & 1)));
          if (!whole) a[0] &= vis[0][0], a[1] &= vis[0][0], a[2] &= vis[0][1], a[3] &= vis[0][1];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816<T>(o[n][i], a, pb[n][0][0], pb[n][0][1]);
            mma16816<T>(o[n][i], a, pl[n][0][0], pl[n][0][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == stages) s = 0, phase ^= 1;
    }
    dc_store<D, NT>(red, p.tile_rows, nq, o, m, l, [&](int i, int e) { return 16 * i + 8 * e + g; });
    const DcPiece pc{cr, ch, ctr, nq, len == ctr, (long long)H * q.prefix[cr] + (long long)ch * ctr, x0, T_, G};
    dc_merge<T, D>(red, q, p, pc, H, gs, aborted);
    x += len;
    if ((cj += len) == ctr) {
      cj = 0;
      if (++ch == H) {
        ch = 0;
        do {
          ++cr;
        } while (cr < ns && q.prefix[cr + 1] == q.prefix[cr]);
        if (cr < ns) ctr = q.prefix[cr + 1] - q.prefix[cr];
      }
    }
  }
  if (aborted && lane == 0) report_timeout(status, kSiteCacheDecode);
}

// ---- 4 bits -------------------------------------------------------------------------
//
// Instructions are the scarce thing here (a 16-bit cache has 3.6 times the bytes
// to hide them behind), so no warp only loads: four warps, unit u to warp u mod 4,
// each with its own ring of units of 32 keys that its first lane refills with bulk
// copies, and four CTAs an SM.
//
// Keys: a word's nibbles are f16 as they stand, subnormals c 2^-24 (low nibble
// of a byte) and c 2^-20 (high nibble, whose query dims are scaled by 2^-4): one
// "and" for two. S = sum_b d_b sum_i c_i q_i - 8 sum_b d_b sum_i q_i: the scale d_b
// multiplies block b's f32 sum, exact up to f32 sums, and the second term is one
// product of the scales with the queries' block sums. Queries are scaled by a power
// of two per row to [2^14, 2^15) at most, which keeps what is 2^-24 of the row's largest.
// Values: f16 pairs 64 + c by one shift and one and-or (mantissa bits 4-7), then
// (c - 8) d in f16 (one rounding, 2^-11): the scale differs by key, which is
// the sum's index there. (A common exponent for a block's scales, so that one
// multiply-add makes the value, saved 20 of 433 instructions per 16 keys and 0.5 us of
// 90, and cost digits next to much larger values.) With f16 outputs, whose own rounding
// is no larger, P goes in as two terms: rms error 2.66e-4 of the rms output, 3.02e-4
// with one, of which the output's rounding is 2.07e-4 (4,096 normal keys).
// Units of 64 keys, with half the copies and waits, took 142 us instead of 153 for 64
// sequences of 8,192 positions, but 70 instead of 63 for 256 of 500 and 358 instead of
// 261 with 16 query heads to a kv head, whose scores then spill. Units of 32 keys spill as
// well at head_dim 128: 36 to 52 bytes a thread up to 8 pairs, 228 above.
// 62 % of the issue slots are used (16 warps an SM, 128 registers): what is left are the
// latencies between an instruction and the next of the same warp.

constexpr int kDq4Threads = 128;

FMD_DEV uint32_t h2sub(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
FMD_DEV uint32_t h2mul(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
// Nibble N of both 16-bit halves as the f16 pair 64 + c. f64 = 0x54005400 comes in
// a register: with two literal operands the and-or became two instructions.
template <int N> FMD_DEV uint32_t nibble64(uint32_t w, uint32_t f64) {
  const uint32_t x = N == 0 ? w << 4 : N == 1 ? w : N == 2 ? w >> 4 : w >> 8;
  return (x & 0x00f000f0u) | f64;
}
// d = a x b (m16n8k16, f16)
FMD_DEV void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kDq4Threads, NT == 1 ? 4 : 3)
    k_cache_decode_q4(CacheView c, int layer, DcArgs p, int* status) {
  constexpr int MT = D / 16;                  // 16-dim tiles of the output
  constexpr int NB = D / 32;                  // 32-dim blocks
  constexpr int K = 32;                       // keys of a unit
  constexpr int CB = K * D / 2, SB = K * D / 16;  // its code and scale bytes
  constexpr int UB = 2 * (CB + SB);
  constexpr int U = 2;                        // 16-key steps
  constexpr bool kHiLo = !Act<T>::kIsBf16;    // f16 outputs: P as two f16 terms (see below)

  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem + p.red_off);
  __shared__ DcSeqs q;
  __shared__ __align__(8) uint64_t full[4][4];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int stages = p.stages, H = c.kv_heads;
  uint8_t* ring = smem + warp * stages * UB;
  griddep_wait();
  griddep_launch();
  const int ns = min(p.r.count() - p.seq0, p.seqs);
  if (ns <= 0) return;
  if (tid == 0) {
    for (int s = 0; s < 16; ++s) mbar_init(&full[s >> 2][s & 3], 1);
    fence_barrier_init();
  }
  dc_plan<K, kDq4Threads>(q, p, c, ns, status);
  const long long T_ = (long long)H * q.prefix[ns];
  const int G = (int)min((long long)gridDim.x, T_), cta = blockIdx.x;
  if (cta >= G) return;
  const long long x0 = (long long)cta * T_ / G, x1 = (long long)(cta + 1) * T_ / G;
  const int ntl = (int)(x1 - x0);
  const int own = ntl > warp ? (ntl - warp + 3) / 4 : 0;  // this warp's units

  // lane i holds the key block of own unit 32 b + i as its offset in the pool, with
  // the unit's half of the page in bit 0 (-1: no keys)
  int issued = 0, is = 0;  // units issued, the stage of the next
  long long l_at = -1;
  uint32_t bad = 0;        // stages without data
  const uint32_t v_at = H * 2 * (CB + SB);  // from a key block to its value block
  auto issue = [&]() {
    if ((issued & 31) == 0) {
      l_at = -1;
      if (issued + lane < own) {
        int r, h, j;
        dc_locate(q, ns, H, x0 + warp + 4LL * (issued + lane), r, h, j);
        const int u = DcKeys<K>(p.a, q.pos[r]).unit(j);
        const int page = u < 0 ? -1 : dc_page(q, c, r, u >> 1, status);
        if (page >= 0) l_at = (c.block(layer, page, 0, h) - c.pool) + (u & 1);
      }
    }
    const long long at = __shfl_sync(0xffffffffu, l_at, issued & 31);
    bad = at < 0 ? bad | 1u << is : bad & ~(1u << is);
    if (lane == 0) {
      uint64_t* bar = &full[warp][is];
      if (at < 0) {
        mbar_arrive(bar);
      } else {
        uint8_t* dst = ring + is * UB;
        const uint32_t half = (uint32_t)at & 1u, codes = half * CB, scales = 2 * CB + half * SB;
        const uint8_t* k = c.pool + (at - half);
        mbar_arrive_expect_tx(bar, UB);
        bulk_load(dst, k + codes, CB, bar);
        bulk_load(dst + CB, k + scales, SB, bar);
        bulk_load(dst + CB + SB, k + v_at + codes, CB, bar);
        bulk_load(dst + 2 * CB + SB, k + v_at + scales, SB, bar);
      }
    }
    ++issued;
    if (++is == stages) is = 0;
  };
  for (int i = 0; i < stages && i < own; ++i) issue();

  bool aborted = false;
  const uint32_t f64 = p.f64;
  const int gs = __ffs(p.a.n_heads / H) - 1;
  const int W = p.a.window, S = W ? p.a.sinks : 0;
  int cr, ch, cj;
  dc_locate(q, ns, H, x0, cr, ch, cj);
  int ctr = q.prefix[cr + 1] - q.prefix[cr];
  uint32_t qf[NT][2 * NB][2];
  uint32_t qb[NT];      // B fragment of the queries' block sums (below)
  float sl[NT][2], o[NT][MT][4], m[NT][2], l[NT][2];
  // this warp's next unit of the CTA's range, its stage and the stage's phase
  int mine = warp, s = 0, phase = 0;
  for (int x = 0; x < ntl;) {
    // a piece: units cj .. cj + len - 1 of segment (cr, ch)
    const int len = min(ctr - cj, ntl - x);
    const int nq = q.cnt[cr] << gs, p0 = q.pos[cr], p1 = p0 + q.cnt[cr] - 1;
    const DcKeys<K> keys(p.a, p0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      const int pr = n * 8 + g;  // this thread's column of the B fragments
      const T* src = (const T*)p.a.q + (size_t)(q.row[cr] + (pr >> gs)) * p.a.q_row +
                     (size_t)((ch << gs) + (pr & ((1 << gs) - 1))) * p.a.q_head;
      // dims 32 b + 8 t .. + 7: the words of chunk t of a key row, in their order
      uint4 u[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b)
        u[b] = pr < nq ? *reinterpret_cast<const uint4*>(src + b * 32 + t * 8) : make_uint4(0, 0, 0, 0);
      float amax = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t w[4] = {u[b].x, u[b].y, u[b].z, u[b].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Act<T>::unpack2(w[e]);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // 2^e brings the largest magnitude to [2^14, 2^15)
      int e = amax > 0.f && amax <= FLT_MAX ? 141 - (int)(__float_as_uint(amax) >> 23) : 0;
      e = min(126, e);
      const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
      float sum[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t w[4] = {u[b].x, u[b].y, u[b].z, u[b].w};
        sum[b] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Act<T>::unpack2(w[k]);
          const float k4 = k & 1 ? 0.0625f : 1.f;
          const uint32_t h2 = Act<__half>::pack2(f.x * up * k4, f.y * up * k4);
          qf[n][2 * b + (k >> 1)][k & 1] = h2;
          const float2 r = Act<__half>::unpack2(h2);
          sum[b] += (r.x + r.y) * (k & 1 ? 16.f : 1.f);
        }
        sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
        sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
      }
      // -8 x 2^-24 sum_b d_b sum_i q_i as a product of its own: rows 0-3 (b) of the
      // B operand hold the sums' f16, rows 4-7 what that rounds off (2^-22 stays off).
      // The sums are 2^-10 of theirs to fit f16; the scores' product takes 2^-24 x 2^10
      float pick[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int b = (2 * t + k) & 3;  // this thread's rows 2 t, 2 t + 1
        float v = b < NB ? sum[0] : 0.f;
#pragma unroll
        for (int i = 1; i < NB; ++i) v = b == i ? sum[i] : v;
        v *= -8.f / 1024.f;
        const float hi = Act<__half>::to_f(Act<__half>::from_f(v));
        pick[k] = t < 2 ? hi : v - hi;
      }
      qb[n] = Act<__half>::pack2(pick[0], pick[1]);
      // accumulators hold columns 2 t, 2 t + 1: their scales. Queries from 2^120 on can take
      // one past f32, where a score of 0 would become a NaN; the largest f32 in its place keeps
      // the order of the others
#pragma unroll
      for (int k = 0; k < 2; ++k)
        sl[n][k] = fminf(p.a.scale * (16777216.f * 1.4426950408889634f) *
                             __shfl_sync(0xffffffffu, down, (2 * t + k) * 4), FLT_MAX);
    }
    for (; mine < x + len; mine += 4) {
      if (aborted || !mbar_wait_warp(&full[warp][s], phase, kDcWait)) {
        aborted = true;
        continue;
      }
      // keys k0 .. k0 + 31
      const int k0 = keys.unit(cj + mine - x) * K;
      const bool whole = k0 + K - 1 <= p0 && (W == 0 || k0 > p1 - W || k0 + K - 1 < S);
      if (!(bad >> s & 1)) {
        const uint8_t* kt = ring + s * UB;
        const uint8_t* vt = kt + CB + SB;
        float sc[NT][U][4];  // [16-key step][keys g: columns 2t, 2t+1 | keys g + 8]
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int ra = u * 16 + g;  // keys g and g + 8 of the step
          {
            // A: the keys' scales, blocks 0-3 and again 0-3 (D 64: 0, 1, -, -)
            const uint32_t e0 = NB == 4 || !(t & 1) ? *reinterpret_cast<const uint32_t*>(kt + CB + (ra * NB + (t & 1) * 2) * 2) : 0u;
            const uint32_t e1 = NB == 4 || !(t & 1) ? *reinterpret_cast<const uint32_t*>(kt + CB + ((ra + 8) * NB + (t & 1) * 2) * 2) : 0u;
            const uint32_t a[4] = {e0, e1, 0u, 0u};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16_zero(sc[n][u], a, qb[n], 0u);
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[n][u][e] *= 1024.f / 16777216.f;
            }
          }
          uint32_t wa[NB], wb[NB];
          float da[NB], db[NB];
          if constexpr (NB == 4) {
            const uint4 A = *reinterpret_cast<const uint4*>(kt + ra * 64 + t * 16);
            const uint4 B = *reinterpret_cast<const uint4*>(kt + (ra + 8) * 64 + t * 16);
            wa[0] = A.x, wa[1] = A.y, wa[2] = A.z, wa[3] = A.w;
            wb[0] = B.x, wb[1] = B.y, wb[2] = B.z, wb[3] = B.w;
            const uint2 E = *reinterpret_cast<const uint2*>(kt + CB + ra * 8);
            const uint2 F = *reinterpret_cast<const uint2*>(kt + CB + (ra + 8) * 8);
            float2 f = Act<__half>::unpack2(E.x);
            da[0] = f.x, da[1] = f.y;
            f = Act<__half>::unpack2(E.y);
            da[2] = f.x, da[3] = f.y;
            f = Act<__half>::unpack2(F.x);
            db[0] = f.x, db[1] = f.y;
            f = Act<__half>::unpack2(F.y);
            db[2] = f.x, db[3] = f.y;
          } else {
            const uint2 A = *reinterpret_cast<const uint2*>(kt + ra * 32 + t * 8);
            const uint2 B = *reinterpret_cast<const uint2*>(kt + (ra + 8) * 32 + t * 8);
            wa[0] = A.x, wa[1] = A.y, wb[0] = B.x, wb[1] = B.y;
            float2 f = Act<__half>::unpack2(*reinterpret_cast<const uint32_t*>(kt + CB + ra * 4));
            da[0] = f.x, da[1] = f.y;
            f = Act<__half>::unpack2(*reinterpret_cast<const uint32_t*>(kt + CB + (ra + 8) * 4));
            db[0] = f.x, db[1] = f.y;
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            constexpr uint32_t lo = 0x000f000fu, hi = 0x00f000f0u;
            const uint32_t xa = wa[b] >> 8, xb = wb[b] >> 8;
            const uint32_t a0[4] = {wa[b] & lo, wb[b] & lo, wa[b] & hi, wb[b] & hi};
            const uint32_t a1[4] = {xa & lo, xb & lo, xa & hi, xb & hi};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float acc[4];
              mma_f16_zero(acc, a0, qf[n][2 * b][0], qf[n][2 * b][1]);
              mma16816<__half>(acc, a1, qf[n][2 * b + 1][0], qf[n][2 * b + 1][1]);
              sc[n][u][0] = fmaf(acc[0], da[b], sc[n][u][0]);
              sc[n][u][1] = fmaf(acc[1], da[b], sc[n][u][1]);
              sc[n][u][2] = fmaf(acc[2], db[b], sc[n][u][2]);
              sc[n][u][3] = fmaf(acc[3], db[b], sc[n][u][3]);
            }
          }
        }
        uint32_t pb[NT][U][2], pl[kHiLo ? NT : 1][U][2], vis[U][2];
        dc_softmax<__half, U, MT, NT, kHiLo>(sc, sl, m, l, o, pb, pl, vis, whole, k0, p0, p1, W, S, gs, 7.f);
        // O^T += V^T P^T; this thread's keys: kb, kb + 1, kb + 8, kb + 9
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int kb = u * 16 + 2 * t;
          const uint8_t* vs = vt + CB;
          const int blk = NB == 4 ? g >> 1 : g >> 2;  // this thread's dims lie in one block
          uint32_t d2[2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t lo = *reinterpret_cast<const uint16_t*>(vs + ((kb + b * 8) * NB + blk) * 2);
            const uint32_t hi = *reinterpret_cast<const uint16_t*>(vs + ((kb + b * 8 + 1) * NB + blk) * 2);
            d2[b] = __byte_perm(lo, hi, 0x5410) & vis[u][b];
          }
          uint32_t w[4][D / 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint8_t* src = vt + (kb + (e & 1) + (e >> 1) * 8) * (D / 2);
            if constexpr (D == 128) {
              const uint2 y = *reinterpret_cast<const uint2*>(src + g * 8);
              w[e][0] = y.x, w[e][1] = y.y;
            } else {
              w[e][0] = *reinterpret_cast<const uint32_t*>(src + g * 4);
            }
          }
          // dims (D / 8) g + 8 i + {0..3 | 4..7}: nibbles of the low and high halves
#pragma unroll
          for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const uint32_t sel = hf ? 0x7632 : 0x5410;
              const uint32_t y0 = __byte_perm(w[0][i], w[1][i], sel), y1 = __byte_perm(w[2][i], w[3][i], sel);
              const uint32_t k72 = 0x54805480u;  // f16 72
              const uint32_t a0[4] = {
                  h2mul(h2sub(nibble64<0>(y0, f64), k72), d2[0]), h2mul(h2sub(nibble64<1>(y0, f64), k72), d2[0]),
                  h2mul(h2sub(nibble64<0>(y1, f64), k72), d2[1]), h2mul(h2sub(nibble64<1>(y1, f64), k72), d2[1])};
              const uint32_t a1[4] = {
                  h2mul(h2sub(nibble64<2>(y0, f64), k72), d2[0]), h2mul(h2sub(nibble64<3>(y0, f64), k72), d2[0]),
                  h2mul(h2sub(nibble64<2>(y1, f64), k72), d2[1]), h2mul(h2sub(nibble64<3>(y1, f64), k72), d2[1])};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816<__half>(o[n][i * 4 + hf * 2], a0, pb[n][u][0], pb[n][u][1]);
                mma16816<__half>(o[n][i * 4 + hf * 2 + 1], a1, pb[n][u][0], pb[n][u][1]);
                if constexpr (kHiLo) {
                  mma16816<__half>(o[n][i * 4 + hf * 2], a0, pl[n][u][0], pl[n][u][1]);
                  mma16816<__half>(o[n][i * 4 + hf * 2 + 1], a1, pl[n][u][0], pl[n][u][1]);
                }
              }
            }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (issued < own) issue();
      if (++s == stages) s = 0, phase ^= 1;
    }
    dc_store<D, NT>(red, p.tile_rows, nq, o, m, l, [&](int i, int e) {
      return (D / 8) * g + 8 * (i >> 2) + 4 * ((i >> 1) & 1) + 2 * (i & 1) + e;
    });
    const DcPiece pc{cr, ch, ctr, nq, len == ctr, (long long)H * q.prefix[cr] + (long long)ch * ctr, x0, T_, G};
    dc_merge<T, D>(red, q, p, pc, H, gs, aborted);
    x += len;
    if ((cj += len) == ctr) {
      cj = 0;
      if (++ch == H) {
        ch = 0;
        do {
          ++cr;
        } while (cr < ns && q.prefix[cr + 1] == q.prefix[cr]);
        if (cr < ns) ctr = q.prefix[cr + 1] - q.prefix[cr];
      }
    }
  }
  if (aborted) {
    // copies in flight land before the CTA retires (bounded)
    for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
      mbar_wait_warp(&full[warp][i % stages], (i / stages) & 1, kDcWait);
    if (lane == 0) report_timeout(status, kSiteCacheDecode);
  }
}

// ---- launch -------------------------------------------------------------------------

struct DcShape {
  int nt, per_sm, grid, stages, red_off, red_row, smem, threads;
};

// CTAs of an SM, ring stages and shared memory for segments of `rows` pairs.
DcShape dc_shape(const CacheView& c, int rows) {
  const bool q4 = c.format == FMD_CACHE_Q4;
  const int D = c.head_dim;
  DcShape s;
  s.nt = rows <= 8 ? 1 : 2;
  s.threads = q4 ? kDq4Threads : kDc16Threads;
  const int stage = q4 ? 4 * 2 * 32 * (D / 2 + D / 16) : 2 * (int)c.block_bytes();  // 4 bits: of all four warps
  const int fixed = 1024 + 1024 + (int)sizeof(DcSeqs) + 512;  // alignment, the CTA's reserve, static arrays
  for (s.per_sm = q4 ? (s.nt == 1 ? 4 : 3) : 2;; --s.per_sm) {
    s.grid = 148 * s.per_sm;
    // merge buffer: four warps' rows, or a weight per piece of a segment (at most one a CTA) and the sum
    s.red_row = std::max(4 * (D + 2), s.grid + 4);
    const int red = (rows * s.red_row + 4 * 128) * 4;
    s.stages = std::min(q4 ? 4 : 8, (227 * 1024 / s.per_sm - fixed - red) / stage);
    if (s.stages >= 2 || s.per_sm == 1) {
      s.stages = std::max(s.stages, 2);
      s.red_off = s.stages * stage;
      s.smem = s.red_off + red + (q4 ? 0 : 1024);
      return s;
    }
  }
}

// The shared memory of the largest call of the kernel that takes segments of `rows`
// pairs. The limit belongs to the function, not to a call: every call sets this one
// value, so that calls of other shapes, from other host threads, do not lower it
// between another's setting and its launch.
int dc_limit(const CacheView& c, int rows) {
  int most = 0;
  for (int r = rows <= 8 ? 1 : 9; r <= (rows <= 8 ? 8 : 16); ++r) most = std::max(most, dc_shape(c, r).smem);
  return most;
}

}  // namespace

bool cache_decode_fits(const CacheView& c, int n_heads, int max_rows) {
  return (long long)max_rows * (n_heads / c.kv_heads) <= 16;
}

// counters, then partials, of the largest grid: fewer rows may run on a larger one
size_t cache_decode_workspace(const CacheView& c, int n_heads, int max_rows) {
  const int rows = max_rows * (n_heads / c.kv_heads);
  return (kDcCounters + (size_t)2 * dc_shape(c, 1).grid * rows * (c.head_dim + 4)) * 4;
}

bool cache_tensor_map(CUtensorMap* m, const CacheView& c, int layer) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) != cudaSuccess ||
        qr != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  const uint64_t rows = (uint64_t)c.n_pages * 2 * c.kv_heads * kPageTokens;
  if (!encode || rows > (uint64_t)INT32_MAX) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)c.head_dim * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)kPageTokens};
  const cuuint32_t estr[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c.block(layer, 0, 0, 0), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t launch_cache_decode(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAttend& a,
                                void* workspace, int* status, cudaStream_t s) {
  const bool q4 = c.format == FMD_CACHE_Q4;
  const int rows = a.max_rows * (a.n_heads / c.kv_heads), D = c.head_dim;
  const DcShape sh = dc_shape(c, rows);
  const int limit = dc_limit(c, rows);
  CUtensorMap map{};
  if (!q4 && !cache_tensor_map(&map, c, layer)) return cudaErrorNotSupported;
  DcArgs p;
  p.r = r;
  p.a = a;
  p.tile_rows = rows;
  p.counters = (int*)workspace;
  p.part = (float*)workspace + kDcCounters;
  p.seqs = std::min(kDcSeqs, kDcCounters / c.kv_heads);
  p.seqs = (int)std::min<long long>(p.seqs, INT_MAX / (cache_units(c) * c.kv_heads));  // >= 1, as the caller has seen to
  p.stages = sh.stages;
  p.red_off = sh.red_off;
  p.red_row = sh.red_row;
  p.f64 = 0x54005400u;
  auto each = [&](auto kern, auto&&... head) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
    for (int s0 = 0; e == cudaSuccess && s0 < r.n_seqs; s0 += p.seqs) {
      p.seq0 = s0;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr.val.programmaticStreamSerializationAllowed = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(sh.grid);
      cfg.blockDim = dim3(sh.threads);
      cfg.dynamicSmemBytes = sh.smem;
      cfg.stream = s;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, kern, head..., p, status);
    }
    return e;
  };
  auto by_nt = [&](auto t, auto d, auto n) {
    using T = decltype(t);
    constexpr int DD = decltype(d)::value, NT = decltype(n)::value;
    return q4 ? each(k_cache_decode_q4<T, DD, NT>, c, layer) : each(k_cache_decode<T, DD, NT>, map, c);
  };
  auto by_d = [&](auto t, auto d) {
    return sh.nt == 1 ? by_nt(t, d, std::integral_constant<int, 1>{}) : by_nt(t, d, std::integral_constant<int, 2>{});
  };
  auto by_t = [&](auto t) {
    return D == 128 ? by_d(t, std::integral_constant<int, 128>{}) : by_d(t, std::integral_constant<int, 64>{});
  };
  return bf16 ? by_t(__nv_bfloat16{}) : by_t(__half{});
}

}  // namespace fmd
