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
// Split: the (sequence, kv head) segments, each its visible page tiles (those of
// the sinks, then those of the window), form one sequence of T tiles; CTA c of G
// takes tiles [c T / G, (c + 1) T / G), whatever the lengths. A segment cut by
// CTA boundaries leaves (m, l, o) partials in the workspace; the last of its
// CTAs to arrive merges them in CTA order, so results do not depend on timing.
//
// A CTA is one producer warp, which looks up pages and keeps a ring of page
// tiles in flight (16 bits: 2D TMA with the 128-byte swizzle, so that ldmatrix is
// conflict-free; 4 bits: bulk copies of the blocks), and four consumer warps: in
// 16 bits 16 keys each of every tile, in 4 bits, where instructions are scarce,
// 32 keys each of alternate tiles. The products are transposed, keys or dims on
// the 16-row side and the up to 8 query pairs on the 8-column side of mma.sync
// m16n8k16: half the instructions and accumulators of queries on the 16-row
// side, most of whose rows would be empty. (tcgen05's smallest tile has 64 rows
// and operands in shared memory: the 4-bit codes would have to be written back
// there in 16 bits, more traffic than the cache itself.)
//
// A stage of the ring is always read by the same warps: each waits for every
// phase of its stages in turn, which a parity wait needs.
//   S^T = K Q^T: A = 16 keys x 16 dims, B = the queries.
//   O^T += V^T P^T: A = 16 dims x 16 keys, B = P^T, turned with movmatrix.
//
// 4 bits: a word's nibbles become f16 pairs 64 + c by one shift and one
// and-or (64 + c has the code in mantissa bits 4-7). Keys are used so: with
// S = sum_g d_g (sum_i (64 + c_i) q_i - 72 sum_i q_i), the accumulator of block g
// starts at -72 sum q and the scale d_g multiplies its f32 result, exact up to
// f32 sums. Values become (c - 8) d in f16 (one rounding, 2^-11): the scale
// differs by key, which is the sum's index there. Queries are scaled by a
// power of two per row to fit f16 (exact but for what is 2^-24 of its row).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <float.h>

#include <algorithm>

#include "fmd_cache.cuh"
#include "fmd_kernels.cuh"

namespace fmd {

namespace {

constexpr int kDcSeqs = 256;      // sequences of one launch at most
// Merge counters of a launch, [sequences][kv heads]: at the same place in every
// workspace, since they are zero between calls of any shape.
constexpr int kDcCounters = 16384;
constexpr int kDcThreads = 160;   // 4 consumer warps, 1 producer warp
constexpr int kDcQ4Ctas = 3;      // CTAs an SM holds over a 4-bit cache (one column tile)
constexpr uint32_t kDcWait = 1u << 22;
constexpr float kDcHeadroom = 8.f;  // log2: how far a score may exceed the reference

struct DcSmem {
  int stage_bytes, stages, red_off, red_row;
};

struct DcArgs {
  CacheRows r;
  CacheAttend a;
  float* part;      // [2 x grid][rows][D + 2] partials of cut segments
  int* counters;    // [sequences][kv heads], zero between calls
  int seq0, seqs;   // the sequences of this launch
  int tile_rows;    // rows of a segment's tile at most
  uint32_t f64;     // f16 pair (64, 64)
  DcSmem sm;
};

FMD_DEV uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
FMD_DEV uint32_t h2sub(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
FMD_DEV uint32_t h2mul(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
// Nibble N of both 16-bit halves as the f16 pair 64 + c. f64 = 0x54005400 comes in
// a register: with two literal operands the and-or became two instructions
// (145 of them for 16 keys instead of 64).
template <int N> FMD_DEV uint32_t nibble64(uint32_t w, uint32_t f64) {
  const uint32_t x = N == 0 ? w << 4 : N == 1 ? w : N == 2 ? w >> 4 : w >> 8;
  return (x & 0x00f000f0u) | f64;
}
// d = a x b + c (m16n8k16, f16), c left as it is
FMD_DEV void mma_f16_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%10,%11};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
FMD_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// CTA whose range [c T / G, (c + 1) T / G) holds tile x.
FMD_DEV int dc_cta(long long x, long long T, int G) { return (int)(((x + 1) * G - 1) / T); }

// Swizzled byte offset of 16-byte chunk ch (of D / 8) of row `row` in a [64][D] tile.
FMD_DEV uint32_t dc_swz(int row, int ch) {
  return (uint32_t)((ch >> 3) * 8192 + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
}

// NT: 8-column tiles of (row, head) pairs.
template <typename T, int D, bool Q4, int NT>
__global__ void __launch_bounds__(kDcThreads, Q4 && NT == 1 ? kDcQ4Ctas : 2)
    k_cache_decode(const __grid_constant__ CUtensorMap tmap, CacheView c, int layer, DcArgs p, int* status) {
  constexpr int KS = D / 16;                    // 16-wide steps of the head
  constexpr int MT = D / 16;                    // 16-dim tiles of the output
  constexpr int NB = D / 32;                    // 32-dim blocks
  constexpr int U = Q4 ? 2 : 1;                 // 16-key steps of a warp and tile; tiles in turn
  constexpr int WPT = 4 / U;                    // warps of a tile
  constexpr int BLK = Q4 ? 64 * (D / 2 + D / 16) : 64 * D * 2;
  using M = typename std::conditional<Q4, __half, T>::type;  // operand type of the products
  constexpr bool kHiLo = !Q4 && Act<T>::kIsBf16;  // P as two bf16 terms
  constexpr float kPScale = kHiLo ? 0.f : 7.f;    // log2 factor of P: f16 keeps what is 2^-21 of the reference

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float* red = reinterpret_cast<float*>(smem + p.sm.red_off);
  __shared__ int s_prefix[kDcSeqs + 1], s_slot[kDcSeqs], s_pos[kDcSeqs], s_row[kDcSeqs], s_cnt[kDcSeqs];
  __shared__ __align__(8) uint64_t full[8], empty[8];
  __shared__ int s_bad[8];
  __shared__ int s_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int stages = p.sm.stages;
  griddep_wait();
  griddep_launch();
  const int ns = min(p.r.count() - p.seq0, p.seqs);
  if (ns <= 0) return;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], WPT);
    }
    fence_barrier_init();
    if (!Q4) prefetch_tmap(&tmap);
  }
  const int W = p.a.window, S = W ? p.a.sinks : 0;
  // tiles of a sequence whose first row is at p0 and last at p1: the sinks' first
  auto split = [&](int p0, int& sink_tiles, int& wt0) {
    const int first = W && p0 >= W ? p0 - W + 1 : 0;
    wt0 = first / kPageTokens;
    sink_tiles = (min(S, wt0 * kPageTokens) + kPageTokens - 1) / kPageTokens;
  };
  for (int i = tid; i < ns; i += kDcThreads) {
    int slot, p0, r0, n;
    p.r.get(p.seq0 + i, slot, p0, r0, n);
    int tiles = 0;
    if (n > 0 && cache_slot_ok(c, slot, status)) {
      if (n > p.a.max_rows || p0 < 0 || p0 > c.max_pages * kPageTokens - n) {
        cache_report(status, n > p.a.max_rows ? FMD_EINVAL : FMD_EOVERFLOW);
      } else {
        int st, wt0;
        split(p0, st, wt0);
        tiles = st + (p0 + n - 1) / kPageTokens - wt0 + 1;
      }
    }
    s_prefix[i] = tiles;
    s_slot[i] = slot;
    s_pos[i] = p0;
    s_row[i] = r0;
    s_cnt[i] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int loc[kDcSeqs / 32], sum = 0;
#pragma unroll
    for (int k = 0; k < kDcSeqs / 32; ++k) {
      const int r = lane * (kDcSeqs / 32) + k;
      loc[k] = r < ns ? s_prefix[r] : 0;
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
    for (int k = 0; k < kDcSeqs / 32; ++k) {
      const int r = lane * (kDcSeqs / 32) + k;
      if (r < ns) s_prefix[r] = run;
      run += loc[k];
    }
    if (lane == 31) s_prefix[ns] = incl;
  }
  __syncthreads();
  const int H = c.kv_heads;
  const long long Tt = (long long)H * s_prefix[ns];
  const int G = (int)min((long long)gridDim.x, Tt), cta = blockIdx.x;
  if (cta >= G) return;
  const long long x0 = (long long)cta * Tt / G, x1 = (long long)(cta + 1) * Tt / G;
  const int ntl = (int)(x1 - x0);
  auto locate = [&](long long x, int& r, int& h, int& j) {
    int lo = 0, hi = ns - 1;  // the last sequence with prefix <= x that has tiles
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)H * s_prefix[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    r = lo;
    const int tr = s_prefix[r + 1] - s_prefix[r];
    const int off = (int)(x - (long long)H * s_prefix[r]);
    h = off / tr;
    j = off - h * tr;
  };
  auto page_index = [&](int r, int j) {
    int st, wt0;
    split(s_pos[r], st, wt0);
    return j < st ? j : wt0 + j - st;
  };

  if (warp == 4) {
    // ---------------- producer ----------------
    bool ok = true;
    int issued = 0, s = 0, round = 0;  // tile `issued` goes to stage s, used `round` times before
    for (int b0 = 0; b0 < ntl && ok; b0 += 32) {
      int lh = 0, lpage = -1;
      if (b0 + lane < ntl) {
        int lr, lj;
        locate(x0 + b0 + lane, lr, lh, lj);
        lpage = c.page_table[(size_t)s_slot[lr] * c.max_pages + page_index(lr, lj)];
        if (lpage < 0 || lpage >= c.n_pages) {
          cache_report(status, FMD_EINVAL);
          lpage = -1;
        }
      }
      const int cnt = min(32, ntl - b0);
      for (int i = 0; i < cnt; ++i) {
        const int h = __shfl_sync(0xffffffffu, lh, i), page = __shfl_sync(0xffffffffu, lpage, i);
        if (round > 0 && !mbar_wait_bounded(&empty[s], (round - 1) & 1, kDcWait)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          s_bad[s] = page < 0;
          if (page < 0) {
            mbar_arrive(&full[s]);
          } else {
            uint8_t* dst = smem + s * p.sm.stage_bytes;
            mbar_arrive_expect_tx(&full[s], 2 * BLK);
            if constexpr (Q4) {
              bulk_load(dst, c.block(layer, page, 0, h), BLK, &full[s]);
              bulk_load(dst + BLK, c.block(layer, page, 1, h), BLK, &full[s]);
            } else {
              const int yk = (page * 2 * H + h) * kPageTokens, yv = yk + H * kPageTokens;
#pragma unroll
              for (int b = 0; b < D / 64; ++b) {
                tma_load_2d(dst + b * 8192, &tmap, b * 64, yk, &full[s]);
                tma_load_2d(dst + BLK + b * 8192, &tmap, b * 64, yv, &full[s]);
              }
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
  const uint32_t f64 = p.f64;
  const int gs = __ffs(p.a.n_heads / H) - 1;  // log2 of the query heads of a kv head
  const int koff = (warp % WPT) * 16 * U, which = warp / WPT;
  int cr, ch, cj;
  locate(x0, cr, ch, cj);
  int ctr = s_prefix[cr + 1] - s_prefix[cr];
  int nq = 0, p0 = 0, p1 = 0, stt = 0, wt0 = 0;  // of the current sequence: pairs, positions, tile split
  uint32_t qf[NT][KS][2];
  float qs[Q4 ? NT : 1][Q4 ? NB : 1][2];  // -72 x sum of the queries of each block, per column
  float sl[NT][2];                        // scale per column
  float o[NT][MT][4], m[NT][2], l[NT][2];
  // this warp's next tile of the CTA's range, its stage and the stage's phase
  int mine = which, s = which, phase = 0;
  for (int x = 0; x < ntl;) {
    // a piece: tiles cj .. cj + len - 1 of segment (cr, ch)
    const int len = min(ctr - cj, ntl - x);
    {
      nq = s_cnt[cr] << gs;
      p0 = s_pos[cr];
      p1 = p0 + s_cnt[cr] - 1;
      split(p0, stt, wt0);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        // B fragments: this thread's column is pair 8 n + g
        const int pr = n * 8 + g;
        const T* q = (const T*)p.a.q + (size_t)(s_row[cr] + (pr >> gs)) * p.a.q_row +
                     (size_t)((ch << gs) + (pr & ((1 << gs) - 1))) * p.a.q_head;
        if constexpr (!Q4) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < 2; ++b)
              qf[n][ks][b] = pr < nq ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + b * 8 + 2 * t) : 0u;
          sl[n][0] = sl[n][1] = p.a.scale * 1.4426950408889634f;
        } else {
          // dims 32 b + 8 t .. + 7: the words of chunk t of a key row, in their order
          uint4 u[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b)
            u[b] = pr < nq ? *reinterpret_cast<const uint4*>(q + b * 32 + t * 8) : make_uint4(0, 0, 0, 0);
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
          // 2^e brings the largest magnitude to [1, 2): blocks sum to at most 2^6 x 72
          int e = amax > 0.f && amax <= FLT_MAX ? 127 - (int)(__float_as_uint(amax) >> 23) : 0;
          e = max(-126, min(126, e));
          const float f2 = __uint_as_float((uint32_t)(127 + e) << 23), b2 = __uint_as_float((uint32_t)(127 - e) << 23);
          float sum[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint32_t w[4] = {u[b].x, u[b].y, u[b].z, u[b].w};
            sum[b] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = Act<T>::unpack2(w[k]);
              const uint32_t h2 = Act<__half>::pack2(f.x * f2, f.y * f2);
              qf[n][2 * b + (k >> 1)][k & 1] = h2;
              const float2 r = Act<__half>::unpack2(h2);
              sum[b] += r.x + r.y;
            }
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
          }
          // accumulators hold columns 2 t, 2 t + 1: their sums and scales
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int b = 0; b < NB; ++b) qs[n][b][k] = -72.f * __shfl_sync(0xffffffffu, sum[b], (2 * t + k) * 4);
            sl[n][k] = p.a.scale * 1.4426950408889634f * __shfl_sync(0xffffffffu, b2, (2 * t + k) * 4);
          }
        }
      }
    }
    for (; mine < x + len; mine += U) {
      if (!aborted && !mbar_wait_bounded(&full[s], phase, kDcWait)) aborted = true;
      // keys k0 .. k0 + KW - 1 of this warp; visible to some row: up to p1, from the
      // oldest window's start or among the sinks
      constexpr int KW = 16 * U;
      const int jt = cj + mine - x;
      const int k0 = (jt < stt ? jt : wt0 + jt - stt) * kPageTokens + koff;
      auto seen = [&](int k, int pos) { return k <= pos && (W == 0 || k > pos - W || k < S); };
      const bool whole = k0 + KW - 1 <= p0 && (W == 0 || k0 > p1 - W || k0 + KW - 1 < S);
      const bool any = k0 <= p1 && (W == 0 || k0 + KW - 1 > p0 - W || k0 < S);
      if (!aborted && any && !s_bad[s]) {
        const uint8_t* kt = smem + s * p.sm.stage_bytes;
        const uint8_t* vt = kt + BLK;
        const uint32_t ka = smem_u32(kt), va = smem_u32(vt);
        float sc[NT][U][4];  // [16-key step][keys g: columns 2t, 2t+1 | keys g + 8]
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if constexpr (Q4) {
            const int ra = koff + u * 16 + g;  // keys g and g + 8 of the step
            uint32_t wa[NB], wb[NB];
            float da[NB], db[NB];
            if constexpr (NB == 4) {
              const uint4 A = *reinterpret_cast<const uint4*>(kt + ra * 64 + t * 16);
              const uint4 B = *reinterpret_cast<const uint4*>(kt + (ra + 8) * 64 + t * 16);
              wa[0] = A.x, wa[1] = A.y, wa[2] = A.z, wa[3] = A.w;
              wb[0] = B.x, wb[1] = B.y, wb[2] = B.z, wb[3] = B.w;
              const uint2 E = *reinterpret_cast<const uint2*>(kt + 4096 + ra * 8);
              const uint2 F = *reinterpret_cast<const uint2*>(kt + 4096 + (ra + 8) * 8);
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
              float2 f = Act<__half>::unpack2(*reinterpret_cast<const uint32_t*>(kt + 2048 + ra * 4));
              da[0] = f.x, da[1] = f.y;
              f = Act<__half>::unpack2(*reinterpret_cast<const uint32_t*>(kt + 2048 + (ra + 8) * 4));
              db[0] = f.x, db[1] = f.y;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][u][0] = sc[n][u][1] = sc[n][u][2] = sc[n][u][3] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const uint32_t a0[4] = {nibble64<0>(wa[b], f64), nibble64<0>(wb[b], f64), nibble64<1>(wa[b], f64), nibble64<1>(wb[b], f64)};
              const uint32_t a1[4] = {nibble64<2>(wa[b], f64), nibble64<2>(wb[b], f64), nibble64<3>(wa[b], f64), nibble64<3>(wb[b], f64)};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float acc[4];
                mma_f16_from(acc, a0, qf[n][2 * b][0], qf[n][2 * b][1], qs[n][b][0], qs[n][b][1]);
                mma16816<__half>(acc, a1, qf[n][2 * b + 1][0], qf[n][2 * b + 1][1]);
                sc[n][u][0] = fmaf(acc[0], da[b], sc[n][u][0]);
                sc[n][u][1] = fmaf(acc[1], da[b], sc[n][u][1]);
                sc[n][u][2] = fmaf(acc[2], db[b], sc[n][u][2]);
                sc[n][u][3] = fmaf(acc[3], db[b], sc[n][u][3]);
              }
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][u][0] = sc[n][u][1] = sc[n][u][2] = sc[n][u][3] = 0.f;
            const int row = koff + u * 16 + (lane & 15);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              uint32_t a[4];
              ldmatrix_x4(a, ka + dc_swz(row, 2 * ks + (lane >> 4)));
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16816<M>(sc[n][u], a, qf[n][ks][0], qf[n][ks][1]);
            }
          }
        }
        // scores in the exp2 domain; hidden ones are -inf
        float mx[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][u][e] *= sl[n][e & 1];
        uint32_t vis[U][2];  // bit masks of the value pairs (kb, kb + 1), (kb + 8, kb + 9) below
#pragma unroll
        for (int u = 0; u < U; ++u) vis[u][0] = vis[u][1] = 0xffffffffu;
        if (!whole) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!seen(k0 + u * 16 + g + (e >> 1) * 8, p0 + ((n * 8 + 2 * t + (e & 1)) >> gs)))
                  sc[n][u][e] = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = k0 + u * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
              if (!(k <= p1 && (W == 0 || k > p0 - W || k < S))) vis[u][e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            mx[n][k] = fmaxf(sc[n][0][k], sc[n][0][2 + k]);
            if constexpr (U == 2) mx[n][k] = fmaxf(mx[n][k], fmaxf(sc[n][U - 1][k], sc[n][U - 1][2 + k]));
          }
        bool up = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) up |= mx[n][0] > m[n][0] + kDcHeadroom || mx[n][1] > m[n][1] + kDcHeadroom;
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
        uint32_t pb[NT][U][2], pl[kHiLo ? NT : 1][U][2];  // B fragments of P^T (and its low part)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float base[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) base[k] = m[n][k] == -INFINITY ? 0.f : m[n][k] - kPScale;
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
              if constexpr (kHiLo) {
                const float2 f = Act<M>::unpack2(hi);
                pl[n][u][b] = movmatrix_t(Act<M>::pack2(e4[2 * b] - f.x, e4[2 * b + 1] - f.y));
              }
            }
          }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int kb = koff + u * 16 + 2 * t;  // this thread's keys: kb, kb + 1, kb + 8, kb + 9
          if constexpr (Q4) {
            const uint8_t* vs = vt + 64 * (D / 2);
            const int blk = NB == 4 ? g >> 1 : g >> 2;  // this thread's dims lie in one block
            uint32_t d2[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const uint32_t lo = *reinterpret_cast<const uint16_t*>(vs + ((kb + b * 8) * NB + blk) * 2);
              const uint32_t hi = *reinterpret_cast<const uint16_t*>(vs + ((kb + b * 8 + 1) * NB + blk) * 2);
              d2[b] = (lo | hi << 16) & vis[u][b];
            }
            uint32_t w[4][D / 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint8_t* src = vt + (kb + (e & 1) + (e >> 1) * 8) * (D / 2);
              if constexpr (D == 128) {
                const uint2 x = *reinterpret_cast<const uint2*>(src + g * 8);
                w[e][0] = x.x, w[e][1] = x.y;
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
                const uint32_t x = __byte_perm(w[0][i], w[1][i], sel), y = __byte_perm(w[2][i], w[3][i], sel);
                const uint32_t k72 = 0x54805480u;  // f16 72
                const uint32_t a0[4] = {
                    h2mul(h2sub(nibble64<0>(x, f64), k72), d2[0]), h2mul(h2sub(nibble64<1>(x, f64), k72), d2[0]),
                    h2mul(h2sub(nibble64<0>(y, f64), k72), d2[1]), h2mul(h2sub(nibble64<1>(y, f64), k72), d2[1])};
                const uint32_t a1[4] = {
                    h2mul(h2sub(nibble64<2>(x, f64), k72), d2[0]), h2mul(h2sub(nibble64<3>(x, f64), k72), d2[0]),
                    h2mul(h2sub(nibble64<2>(y, f64), k72), d2[1]), h2mul(h2sub(nibble64<3>(y, f64), k72), d2[1])};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma16816<__half>(o[n][i * 4 + hf * 2], a0, pb[n][u][0], pb[n][u][1]);
                  mma16816<__half>(o[n][i * 4 + hf * 2 + 1], a1, pb[n][u][0], pb[n][u][1]);
                }
              }
          } else {
            // matrices: (keys 0-7, dims 0-7), (keys 0-7, dims 8-15), (keys 8-15, dims 0-7), ...
            const int row = koff + u * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[4];
              ldmatrix_x4_trans(a, va + dc_swz(row, 2 * i + ((lane >> 3) & 1)));
              if (!whole) a[0] &= vis[u][0], a[1] &= vis[u][0], a[2] &= vis[u][1], a[3] &= vis[u][1];
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816<M>(o[n][i], a, pb[n][u][0], pb[n][u][1]);
                if constexpr (kHiLo) mma16816<M>(o[n][i], a, pl[n][u][0], pl[n][u][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if ((s += U) >= stages) s -= stages, phase ^= 1;
    }

    {
      // ---- merge the 4 warps over this piece of the segment ----
      constexpr int rs = D + 2;
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
            float* rw = red + (size_t)(warp * p.tile_rows + col) * rs;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                // row g + 8 e of tile i: natural dims, or the thread's nibble order
                const int d = Q4 ? (D / 8) * g + 8 * (i >> 2) + 4 * ((i >> 1) & 1) + 2 * (i & 1) + e : 16 * i + 8 * e + g;
                rw[d] = o[n][i][2 * e + k];
              }
            if (g == 0) {
              rw[D] = m[n][k];
              rw[D + 1] = lw;
            }
          }
        }
      named_sync(1, 128);
      const bool inside = len == ctr;
      const long long seg0 = (long long)H * s_prefix[cr] + (long long)ch * ctr;
      const int pslot = 2 * cta + (seg0 < x0 ? 0 : 1);
      for (int i = tid; i < nq * (D / 2); i += 128) {
        const int row = i / (D / 2), d0 = (i % (D / 2)) * 2;
        float mm[4], Mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) Mx = fmaxf(Mx, mm[w] = red[(size_t)(w * p.tile_rows + row) * rs + D]);
        const float base = Mx == -INFINITY ? 0.f : Mx;
        float L = 0.f, A0 = 0.f, A1 = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float* rw = red + (size_t)(w * p.tile_rows + row) * rs;
          const float f = ex2(mm[w] - base);  // 0 for a warp that saw nothing
          L = fmaf(rw[D + 1], f, L);
          A0 = fmaf(rw[d0], f, A0);
          A1 = fmaf(rw[d0 + 1], f, A1);
        }
        if (inside) {
          if (!aborted) {
            T* out = (T*)p.a.out + (size_t)(s_row[cr] + (row >> gs)) * p.a.out_row +
                     (size_t)((ch << gs) + (row & ((1 << gs) - 1))) * p.a.out_head + d0;
            *reinterpret_cast<uint32_t*>(out) = Act<T>::pack2(A0 / L, A1 / L);
          }
        } else {
          float* pt = p.part + ((size_t)pslot * p.tile_rows + row) * (D + 2);
          pt[d0] = A0;
          pt[d0 + 1] = A1;
          if (d0 == 0) pt[D] = Mx, pt[D + 1] = L;
        }
      }
      if (!inside) {
        const int cf = dc_cta(seg0, Tt, G), cl = dc_cta(seg0 + ctr - 1, Tt, G);
        int* counter = &p.counters[(size_t)cr * H + ch];
        named_sync(1, 128);
        if (tid == 0) {
          __threadfence();
          s_last = atomicAdd(counter, 1) == cl - cf;
          if (s_last) __threadfence();
        }
        named_sync(1, 128);
        if (s_last) {
          // weights of the pieces (one warp per row), then the weighted sums
          const int np = cl - cf + 1, ws = p.sm.red_row;  // floats of `red` per row, > pieces
          auto piece = [&](int k) {
            return p.part + (size_t)(2 * (cf + k) + (k == 0 ? 1 : 0)) * p.tile_rows * (D + 2);
          };
          for (int row = warp; row < nq; row += 4) {
            float Mx = -INFINITY, L = 0.f;
            for (int k = lane; k < np; k += 32) {
              const float x = __ldcg(piece(k) + row * (D + 2) + D);
              red[row * ws + k] = x;
              Mx = fmaxf(Mx, x);
            }
            Mx = warp_max(Mx);
            const float base = Mx == -INFINITY ? 0.f : Mx;
            for (int k = lane; k < np; k += 32) {
              const float f = ex2(red[row * ws + k] - base);
              red[row * ws + k] = f;
              L = fmaf(__ldcg(piece(k) + row * (D + 2) + D + 1), f, L);
            }
            L = warp_sum(L);
            if (lane == 0) red[row * ws + np] = L;
          }
          named_sync(1, 128);
          for (int i = tid; i < nq * (D / 2); i += 128) {
            const int row = i / (D / 2), d0 = (i % (D / 2)) * 2;
            const float* w = red + row * ws;
            float A0 = 0.f, A1 = 0.f;
            const float* pt = piece(0) + row * (D + 2) + d0;
            float2 x = __ldcg(reinterpret_cast<const float2*>(pt));
            A0 = x.x * w[0], A1 = x.y * w[0];
            pt = p.part + (size_t)2 * (cf + 1) * p.tile_rows * (D + 2) + row * (D + 2) + d0;
            const size_t step = (size_t)2 * p.tile_rows * (D + 2);
#pragma unroll 16
            for (int k = 1; k < np; ++k, pt += step) {
              x = __ldcg(reinterpret_cast<const float2*>(pt));
              A0 = fmaf(x.x, w[k], A0);
              A1 = fmaf(x.y, w[k], A1);
            }
            if (!aborted) {
              const float L = w[np];
              T* out = (T*)p.a.out + (size_t)(s_row[cr] + (row >> gs)) * p.a.out_row +
                       (size_t)((ch << gs) + (row & ((1 << gs) - 1))) * p.a.out_head + d0;
              *reinterpret_cast<uint32_t*>(out) = Act<T>::pack2(A0 / L, A1 / L);
            }
          }
          if (tid == 0) *counter = 0;
        }
      }
      named_sync(1, 128);  // `red` is reused by the next piece
    }
    x += len;
    if ((cj += len) == ctr) {
      cj = 0;
      if (++ch == H) {
        ch = 0;
        do {
          ++cr;
        } while (cr < ns && s_prefix[cr + 1] == s_prefix[cr]);
        if (cr < ns) ctr = s_prefix[cr + 1] - s_prefix[cr];
      }
    }
  }
  if (aborted && lane == 0) report_timeout(status, kSiteCacheDecode);
}

int dc_ctas_per_sm(bool q4, int nt) { return q4 && nt == 1 ? kDcQ4Ctas : 2; }

}  // namespace

bool cache_decode_fits(const CacheView& c, int n_heads, int max_rows) {
  return (long long)max_rows * (n_heads / c.kv_heads) <= 16;
}

// counters, then partials
size_t cache_decode_workspace(const CacheView& c, int n_heads, int n_seqs, int max_rows) {
  const int rows = max_rows * (n_heads / c.kv_heads), nt = rows <= 8 ? 1 : 2;
  const size_t grid = (size_t)148 * dc_ctas_per_sm(c.format == FMD_CACHE_Q4, nt);
  (void)n_seqs;
  return (kDcCounters + 2 * grid * rows * (c.head_dim + 2)) * 4;
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
  const int rows = a.max_rows * (a.n_heads / c.kv_heads), nt = rows <= 8 ? 1 : 2, D = c.head_dim;
  CUtensorMap map{};
  if (!q4 && !cache_tensor_map(&map, c, layer)) return cudaErrorNotSupported;
  DcArgs p;
  p.r = r;
  p.a = a;
  p.tile_rows = rows;
  p.f64 = 0x54005400u;
  const int per_sm = dc_ctas_per_sm(q4, nt);
  const int grid = 148 * per_sm;
  p.counters = (int*)workspace;
  p.part = (float*)workspace + kDcCounters;
  p.seqs = std::min(kDcSeqs, kDcCounters / c.kv_heads);
  // as many stages as fit (at most 8) with per_sm CTAs in an SM's 227 KB
  const int blk = (int)c.block_bytes();
  p.sm.stage_bytes = 2 * blk;
  // merge buffer: four warps' rows, or a weight per piece of a segment (at most one a CTA) and the sum
  p.sm.red_row = std::max(4 * (D + 2), grid + 4);
  const int red = rows * p.sm.red_row * 4;
  const int room = 227 * 1024 / per_sm - 8 * 1024 - red;  // static arrays, alignment, the CTA's reserve
  p.sm.stages = std::min(8, std::max(2, room / p.sm.stage_bytes));
  if (q4) p.sm.stages &= ~1;  // tiles alternate between two pairs of warps, and so must the stages
  p.sm.red_off = p.sm.stages * p.sm.stage_bytes;
  const int smem = 1024 + p.sm.red_off + red;
  auto go = [&](auto kern) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    for (int s0 = 0; e == cudaSuccess && s0 < r.n_seqs; s0 += p.seqs) {
      p.seq0 = s0;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr.val.programmaticStreamSerializationAllowed = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(grid);
      cfg.blockDim = dim3(kDcThreads);
      cfg.dynamicSmemBytes = smem;
      cfg.stream = s;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, kern, map, c, layer, p, status);
    }
    return e;
  };
  auto by_nt = [&](auto t, auto d, auto f) {
    using T = decltype(t);
    constexpr int DD = decltype(d)::value;
    constexpr bool F = decltype(f)::value;
    return nt == 1 ? go(k_cache_decode<T, DD, F, 1>) : go(k_cache_decode<T, DD, F, 2>);
  };
  auto by_f = [&](auto t, auto d) { return q4 ? by_nt(t, d, std::true_type{}) : by_nt(t, d, std::false_type{}); };
  auto by_d = [&](auto t) {
    return D == 128 ? by_f(t, std::integral_constant<int, 128>{}) : by_f(t, std::integral_constant<int, 64>{});
  };
  return bf16 ? by_d(__nv_bfloat16{}) : by_d(__half{});
}

}  // namespace fmd
