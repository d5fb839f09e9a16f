// The paged cache's row and page operators (include/fmd_cache.h): append, read,
// fork, copy and compact.
#include <algorithm>
#include <climits>
#include <cstring>
#include <memory>
#include <new>

#include "fmd_cache.cuh"
#include "fmd_views.h"

namespace fmd {

namespace {

// ---- rows ---------------------------------------------------------------------------
//
// append and read are bound by the bytes they move, as long as their instructions
// stay few. A block of one warp (read: two) takes one row, with few rows some of its
// heads; L = D / 8 lanes take a head, 8 dims (16 bytes) each, so that every access is a
// full sector, and each lane has HPG heads' loads in flight before it looks up the
// row's sequence, position and page, which they do not need. One warp, not eight: that
// lookup and the addresses cost about 400 instructions a warp, as much as four heads.

constexpr int kRowThreads = 32;
// Heads a lane has in flight, with many rows, and the blocks of an SM (80 registers a
// thread). 10,007 rows of 32 heads with norms and rotation, 16 bits, and 16,384 of 16 heads
// into 4 bits: 34.7 and 35.7 us; 39.9 and 38.0 with 2 heads and 32 blocks, 44.9 and 46.1 with
// 8 and 16, 38.5 and 40.3 with two warps, 2 heads and 16 blocks.
constexpr int kRowHeads = 4, kRowBlocks = 24;

// What a row is stored as: its position's place in a page, and the page's first
// block in the layer. False where the row takes no part.
struct CacheRow {
  int pos;
  uint8_t* page;
};
FMD_DEV bool cache_row(const CacheView& c, const CacheRows& r, int layer, int row, CacheRow& o, int* status) {
  const int n_seqs = r.count();
  int lo = row;
  if (r.row0) {
    int hi = n_seqs;  // the last sequence that starts at or before the row; n_seqs: behind the last
    lo = 0;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (r.row0[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
  }
  if (lo >= n_seqs || row >= r.n_rows) return false;
  int slot, p0, r0, n;
  r.get(lo, slot, p0, r0, n);
  if (row < r0 || row >= r0 + n || !cache_slot_ok(c, slot, status)) return false;
  // p0 near the largest integer must not wrap into the table
  o.pos = p0 <= INT_MAX - (row - r0) ? p0 + (row - r0) : -1;
  const int page = cache_page(c, slot, o.pos, status);
  if (page < 0) return false;
  o.page = c.block(layer, page, 0, 0);
  return true;
}
template <typename T> FMD_DEV void unpack8(uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Act<T>::unpack2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Two f32 lanes at once, each rounded as the scalar instruction rounds.
FMD_DEV unsigned long long f2(float x, float y) {
  unsigned long long d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
FMD_DEV unsigned long long f2_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
FMD_DEV unsigned long long f2_add(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
FMD_DEV unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The 4-bit code word and scale of a head: lane l of its L lanes holds dims
// 8 l .. 8 l + 7. The code is the exact floor(-8 x / m + 8.5): an estimate's
// nearest integer B is decided by the sign of (8.5 - B) |m| - 8 sgn(m) x, one fused
// multiply-add, instead of an IEEE division per value. Instructions issued are what
// bounds a 4-bit append, so values go in twos. Every lane of the warp calls.
FMD_DEV uint32_t quantise8(float (&x)[8], bool key, __half& scale) {
  const int lane = threadIdx.x & 31;
  float hi = x[0], lo = x[0];
  unsigned long long z2 = f2(0.f, 0.f);
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    hi = fmaxf(hi, x[i]);
    lo = fminf(lo, x[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; i += 2) z2 = f2_fma(f2(0.f, 0.f), f2(x[i], x[i + 1]), z2);
  // NaN once a value is NaN or infinite
  float z = __uint_as_float((uint32_t)z2) + __uint_as_float((uint32_t)(z2 >> 32));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    z += __shfl_xor_sync(0xffffffffu, z, o);
  }
  float mag = fmaxf(hi, -lo);
  float sgn = hi >= -lo ? 1.f : -1.f;
  if (__any_sync(0xffffffffu, hi == -lo)) {
    // both signs reach the magnitude: the first value counts
    float first = 0.f;
    bool has = false;
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (fabsf(x[i]) == mag) first = x[i], has = true;
    const uint32_t with = __ballot_sync(0xffffffffu, has) & (0xfu << (lane & ~3));
    first = __shfl_sync(0xffffffffu, first, with ? __ffs(with) - 1 : lane);
    if (hi == -lo) sgn = first < 0.f ? -1.f : 1.f;
  }
  if (__any_sync(0xffffffffu, mag > 65504.f)) {
    mag = fminf(mag, 65504.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
  }
  const float m8 = -8.f * sgn, r = mag > 0.f ? __fdividef(m8, mag) : 0.f;
  uint32_t word = 0;
  constexpr float kMagic = 12582912.f;  // 1.5 x 2^23: the nearest integer in the low bits
  constexpr uint32_t kBits = 0x4b400000u;
  const unsigned long long r2 = f2(r, r), m2 = f2(mag, mag), n2 = f2(m8, m8), c85 = f2(8.5f, 8.5f);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const unsigned long long x2 = f2(x[e], x[e + 1]);
    const unsigned long long t = f2_add(f2_fma(x2, r2, c85), f2(kMagic, kMagic));
    const unsigned long long b = f2_add(t, f2(-kMagic, -kMagic));
    const unsigned long long s = f2_fma(f2_fma(b, f2(-1.f, -1.f), c85), m2, f2_mul(n2, x2));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int below = (int)(s >> (32 * h)) >> 31;  // -1: the code is B - 1
      const int code = min((int)(uint32_t)(t >> (32 * h)) + below, (int)kBits + 15);
      const int i = e + h;
      word += (uint32_t)code << (4 * (key ? (i >> 1) + 4 * (i & 1) : i));
    }
  }
  word -= kBits * 0x11111111u;  // what the codes' upper bits came to
  scale = z == z ? __float2half_rn(mag * (sgn * -0.125f)) : __ushort_as_half(0x7fff);
  return word;
}

// ---- append -------------------------------------------------------------------------
//
// x * rsqrt(mean(x^2) + eps) * w, then (a, b) -> (a cos - b sin, b cos + a sin):
// about 10 flop a byte at most, far below the memory's. The queries', keys' and
// values' heads are passed over one after the other, so that what is done with a
// head is the same for the whole block. 10,007 rows of 16 + 8 + 8 heads with norms and
// rotation, 16 bits: 34.7 us, 4.9 TB/s; 16,384 rows of 8 + 8 heads into 4 bits 35.7 us, 2.4
// TB/s, the quantiser's instructions. One row: 2.8 us, 64 rows 3.0 (back to back).
template <typename T, int D, bool Q4, int HPG>
__global__ void __launch_bounds__(kRowThreads, kRowBlocks)
    k_cache_append(CacheView c, int layer, CacheRows r, CacheAppend a, int* status) {
  constexpr int L = D / 8, GROUPS = kRowThreads / L, PER = GROUPS * HPG;
  constexpr int BB = Q4 ? kPageTokens * (D / 2 + D / 16) : kPageTokens * D * 2;
  griddep_wait();
  griddep_launch();
  const int row = blockIdx.x, l = threadIdx.x % L, grp = threadIdx.x / L;
  const int H = c.kv_heads, nq = (a.n_heads + PER - 1) / PER, nk = (H + PER - 1) / PER;
  const int half = a.rot_dim / 2;
  bool known = false;
  CacheRow w{};
  float cs[8], sn[8];
  for (int it = blockIdx.y; it < nq + 2 * nk; it += gridDim.y) {
    const int kind = it < nq ? 0 : it < nq + nk ? 1 : 2;  // queries, keys, values
    const int h0 = (it - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk)) * PER + grp, n = kind ? H : a.n_heads;
    const T* src = (const T*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                   row * (kind == 0 ? a.q_row : kind == 1 ? a.k_row : a.v_row) + l * 8;
    const long long step = kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head;
    uint4 raw[HPG];
    if (!a.staged) {
#pragma unroll
      for (int k = 0; k < HPG; ++k)
        if (h0 + k * GROUPS < n && row < r.n_rows)
          raw[k] = *reinterpret_cast<const uint4*>(src + (h0 + k * GROUPS) * step);
    }
    if (!known) {
      known = true;
      if (!cache_row(c, r, layer, row, w, status)) return;  // the same for the whole block
      if (a.rot_dim > 0) {
        if (w.pos >= a.table_rows) {
          cache_report(status, FMD_EOVERFLOW);
          return;
        }
        const float* ct = a.cos + (size_t)w.pos * half;
        const float* st = a.sin + (size_t)w.pos * half;
        // this lane's factors: of dims 8 l + i (halves), or of pairs 4 l + i / 2; the
        // sine takes the sign that its place in the pair has
#pragma unroll
        for (int q4 = 0; q4 < 2; ++q4) {
          const int d = l * 8 + q4 * 4;
          float4 cv = make_float4(1.f, 1.f, 1.f, 1.f), sv = make_float4(0.f, 0.f, 0.f, 0.f);
          if (d < a.rot_dim) {
            if (!a.interleaved) {
              const int f = d < half ? d : d - half;  // half is a multiple of 4
              cv = *reinterpret_cast<const float4*>(ct + f);
              sv = *reinterpret_cast<const float4*>(st + f);
              if (d < half) sv = make_float4(-sv.x, -sv.y, -sv.z, -sv.w);
            } else {
              const float2 c2 = *reinterpret_cast<const float2*>(ct + d / 2);
              const float2 s2 = *reinterpret_cast<const float2*>(st + d / 2);
              cv = make_float4(c2.x, c2.x, c2.y, c2.y);
              sv = make_float4(-s2.x, s2.x, -s2.y, s2.y);
            }
          }
          cs[4 * q4] = cv.x, cs[4 * q4 + 1] = cv.y, cs[4 * q4 + 2] = cv.z, cs[4 * q4 + 3] = cv.w;
          sn[4 * q4] = sv.x, sn[4 * q4 + 1] = sv.y, sn[4 * q4 + 2] = sv.z, sn[4 * q4 + 3] = sv.w;
        }
      }
    }
    const int pr = w.pos % kPageTokens;
    if (a.staged) {
      // the same block of the staging pool, which has 16-bit blocks
      const uint8_t* at = a.staged + ((w.page - c.block(layer, 0, 0, 0)) / BB + (kind - 1) * H) * (kPageTokens * D * 2) +
                          pr * (D * 2) + l * 16;
#pragma unroll
      for (int k = 0; k < HPG; ++k)
        if (h0 + k * GROUPS < n)
          raw[k] = *reinterpret_cast<const uint4*>(at + (size_t)(h0 + k * GROUPS) * (kPageTokens * D * 2));
    }
    // head h of the output, this lane's 16 bytes (4 bits: the head's block)
    uint8_t* dst;
    long long dst_step;
    if (kind == 0) {
      dst = (uint8_t*)((T*)a.q_out + row * a.qo_row + l * 8);
      dst_step = a.qo_head * 2;
    } else {
      dst = w.page + (kind - 1) * H * BB + (Q4 ? 0 : pr * (D * 2) + l * 16);
      dst_step = BB;
    }
    const T* nw = (const T*)(kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr);
    const bool turn = a.rot_dim > 0 && kind < 2;
    if ((!Q4 || kind == 0) && !nw && !turn) {
      // stored as it is
#pragma unroll
      for (int k = 0; k < HPG; ++k)
        if (h0 + k * GROUPS < n) *reinterpret_cast<uint4*>(dst + (h0 + k * GROUPS) * dst_step) = raw[k];
      continue;
    }
    float wv[8];
    if (nw) unpack8<T>(*reinterpret_cast<const uint4*>(nw + l * 8), wv);
#pragma unroll
    for (int k = 0; k < HPG; ++k) {
      const bool live = h0 + k * GROUPS < n;  // the lanes of a warp stay together for the shuffles
      if (!__any_sync(0xffffffffu, live)) continue;
      float x[8];
      unpack8<T>(live ? raw[k] : make_uint4(0, 0, 0, 0), x);
      if (nw) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rs = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * rs * wv[i];
      }
      if (turn) {
        float y[8];  // the other of each pair
        const int base = threadIdx.x & 31 & ~(L - 1);
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        } else if (half % 8 == 0) {
          const int from = base + ((l < half / 8 ? l + half / 8 : l - half / 8) & (L - 1));
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from);
        } else {
          // halves of 4 (mod 8) dims: up from dim d to d + half, down from d to d - half
          const int q8 = half / 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float up = __shfl_sync(0xffffffffu, x[i ^ 4], base + ((l + q8 + (i >> 2)) & (L - 1)));
            const float down = __shfl_sync(0xffffffffu, x[i ^ 4], base + ((l - q8 - 1 + (i >> 2)) & (L - 1)));
            y[i] = l * 8 + i < half ? up : down;
          }
        }
        // dims behind rot_dim stay (their factors are 1 and 0, but what they would meet may be NaN)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          if (l * 8 + i < a.rot_dim)
#pragma unroll
            for (int e = i; e < i + 4; ++e) x[e] = fmaf(y[e], sn[e], x[e] * cs[e]);
      }
      uint8_t* at = dst + (h0 + k * GROUPS) * dst_step;
      if (Q4 && kind) {
        __half sc;
        const uint32_t word = quantise8(x, kind == 1, sc);
        if (live) {
          reinterpret_cast<uint32_t*>(at + pr * (D / 2))[kind == 1 ? (l & 3) * (D / 32) + l / 4 : l] = word;
          if ((l & 3) == 0)
            reinterpret_cast<__half*>(at + kPageTokens * (D / 2))[pr * (D / 32) + l / 4] = sc;
        }
      } else if (live) {
        uint4 u;
        u.x = Act<T>::pack2(x[0], x[1]);
        u.y = Act<T>::pack2(x[2], x[3]);
        u.z = Act<T>::pack2(x[4], x[5]);
        u.w = Act<T>::pack2(x[6], x[7]);
        *reinterpret_cast<uint4*>(at) = u;
      }
    }
  }
}

// ---- read ---------------------------------------------------------------------------
//
// 32,768 rows of 8 heads of 128 to f32: 63 us from 16 bits, 47 us from 4, 6.4 TB/s.
// Two warps a row: 24.3 us for 10,007 rows in 16 bits, 26.6 with one. Two lanes share
// their 64 bytes of output so that a store fills whole sectors: 16.7 us for those rows,
// 24.3 with each lane storing its own 32 in two halves.
constexpr int kReadThreads = 64;

template <int D, int FORMAT>
__global__ void __launch_bounds__(kReadThreads)
    k_cache_read(CacheView c, int layer, CacheRows r, float* k, float* v, int* status) {
  constexpr int L = D / 8, GROUPS = kReadThreads / L, HPG = 4;
  constexpr bool Q4 = FORMAT == FMD_CACHE_Q4;
  constexpr int BB = Q4 ? kPageTokens * (D / 2 + D / 16) : kPageTokens * D * 2;
  griddep_wait();
  griddep_launch();
  const int row = blockIdx.x, l = threadIdx.x % L, grp = threadIdx.x / L;
  CacheRow w;
  if (!cache_row(c, r, layer, row, w, status)) return;
  const int pr = w.pos % kPageTokens, H = c.kv_heads;
  // lanes l, l + 1 hold 16 dims and store them as two pieces of 8
  const bool odd = l & 1;
  float* kd = k + (size_t)row * H * D + (l & ~1) * 8 + odd * 4;
  float* vd = v + (size_t)row * H * D + (l & ~1) * 8 + odd * 4;
  for (int h0 = blockIdx.y * GROUPS * HPG; h0 < 2 * H; h0 += gridDim.y * GROUPS * HPG) {
    uint4 raw[HPG] = {};
    uint32_t word[HPG] = {};
    __half d[HPG] = {};
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      const int h = h0 + i * GROUPS + grp;
      if (h >= 2 * H) continue;
      const uint8_t* blk = w.page + h * BB;
      if constexpr (Q4) {
        word[i] = reinterpret_cast<const uint32_t*>(blk + pr * (D / 2))[h >= H ? l : (l & 3) * (D / 32) + l / 4];
        d[i] = reinterpret_cast<const __half*>(blk + kPageTokens * (D / 2))[pr * (D / 32) + l / 4];
      } else {
        raw[i] = *reinterpret_cast<const uint4*>(blk + pr * (D * 2) + l * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      const int h = h0 + i * GROUPS + grp;
      float x[8];
      if constexpr (Q4) {
        const float s = __half2float(d[i]);
        // a key's nibbles to dim order, so that one path reads both
        uint32_t t = word[i];
        if (h < H) {
          const uint32_t even = t & 0x0000ffffu, odd = t >> 16;  // dims 0 2 4 6 | 1 3 5 7
          uint32_t e = (even | even << 8) & 0x00ff00ffu, o = (odd | odd << 8) & 0x00ff00ffu;
          e = (e | e << 4) & 0x0f0f0f0fu;
          o = (o | o << 4) & 0x0f0f0f0fu;
          t = e | o << 4;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)((int)(t >> (4 * e) & 15) - 8) * s;
      } else if constexpr (FORMAT == FMD_CACHE_BF16) {
        unpack8<__nv_bfloat16>(raw[i], x);
      } else {
        unpack8<__half>(raw[i], x);
      }
      float own[4], other[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        own[e] = odd ? x[4 + e] : x[e];
        other[e] = __shfl_xor_sync(0xffffffffu, odd ? x[e] : x[4 + e], 1);
      }
      if (h >= 2 * H) continue;
      const float4 a = make_float4(own[0], own[1], own[2], own[3]);
      const float4 b = make_float4(other[0], other[1], other[2], other[3]);
      float4* dst = reinterpret_cast<float4*>(h < H ? kd + h * D : vd + (h - H) * D);
      __stcs(dst, odd ? b : a);
      __stcs(dst + 2, odd ? a : b);
    }
  }
}

// ---- pages --------------------------------------------------------------------------

constexpr int kCopyBatch = 128;  // host pairs of one launch, passed by value
struct CopyList {
  int src[kCopyBatch], dst[kCopyBatch];
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

// Whole pages [bytes] of a layer: a block's threads keep eight 16-byte loads each in
// flight before the stores. 16 bits: 512 pages of 4 layers (1,074 MB read and written)
// 212 us, 5.1 TB/s; a compaction that moves 1,536 MB 268 us, 5.7 TB/s.
FMD_DEV void copy_page(const uint8_t* src, uint8_t* dst, size_t bytes) {
  const int4* s = reinterpret_cast<const int4*>(src);
  int4* d = reinterpret_cast<int4*>(dst);
  const int n = (int)(bytes / 16), nt = blockDim.x;
  int i = threadIdx.x;
  for (; i + 7 * nt < n; i += 8 * nt) {
    int4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __ldcs(s + i + k * nt);
#pragma unroll
    for (int k = 0; k < 8; ++k) __stcs(d + i + k * nt, v[k]);
  }
  for (; i < n; i += nt) __stcs(d + i, __ldcs(s + i));
}

__global__ void __launch_bounds__(256) k_cache_copy(CacheView c, int layers, CopyList l, int n) {
  const long long works = (long long)n * layers;
  for (long long w = blockIdx.x; w < works; w += gridDim.x) {
    const int i = (int)(w % n), layer = (int)(w / n);
    copy_page(c.block(layer, l.src[i], 0, 0), c.block(layer, l.dst[i], 0, 0), c.page_bytes());
  }
}

// Block (i, b): fork i's table entries (b = 0) and its share of the blocks whose
// rows are copied, a warp each. Eight forks in 28 layers with 7 rows to copy: 4.4 us.
__global__ void __launch_bounds__(256) k_cache_fork(CacheView c, int layers, int* table, ForkList l, int* status) {
  const int i = blockIdx.x, lane = threadIdx.x & 31;
  const int full = l.len[i] / kPageTokens, part = l.len[i] % kPageTokens;
  const int* from = table + (size_t)l.src[i] * c.max_pages;
  int* to = table + (size_t)l.dst[i] * c.max_pages;
  if (blockIdx.y == 0) {
    for (int k = threadIdx.x; k < full; k += blockDim.x) to[k] = from[k];
    if (threadIdx.x == 0 && part) to[full] = l.page[i];
  }
  if (!part) return;
  const int s = from[full];
  if (s < 0 || s >= c.n_pages) {
    cache_report(status, FMD_EINVAL);
    return;
  }
  const long long blocks = (long long)layers * 2 * c.kv_heads;
  const size_t bb = c.block_bytes();
  for (long long b = (long long)blockIdx.y * 8 + (threadIdx.x >> 5); b < blocks; b += (long long)gridDim.y * 8) {
    const int layer = (int)(b / (2 * c.kv_heads)), bk = (int)(b % (2 * c.kv_heads));
    copy_block_rows(c, c.block(layer, s, 0, 0) + bk * bb, c.block(layer, l.page[i], 0, 0) + bk * bb, part, lane, 32);
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
  const long long works = (long long)n * layers;
  for (long long w = blockIdx.x; w < works; w += gridDim.x) {
    const int i = (int)(w % n), layer = (int)(w / n);
    copy_page(c.block(layer, src[i], 0, 0), c.block(layer, dst[i], 0, 0), c.page_bytes());
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
// The same with programmatic stream serialisation, for kernels that begin with griddep_wait.
template <typename... KArgs, typename... Args>
cudaError_t launch_dep(void (*kern)(KArgs...), dim3 grid, dim3 block, cudaStream_t s, Args&&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace

cudaError_t launch_cache_append(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAppend& a,
                                int* status, cudaStream_t s) {
  // With few rows a lane takes one head and a row as many blocks as its heads fill:
  // one row of 32 heads 2.6 us so, 4.75 as one block of two warps with two heads a lane.
  const bool few = r.n_rows < 148 * 4;
  const int g = kRowThreads / (c.head_dim / 8);
  const int passes = (a.n_heads + g - 1) / g + 2 * ((c.kv_heads + g - 1) / g);
  const dim3 grid(r.n_rows, few ? passes : 1);
  auto go = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    auto on = [&](auto kern) { return launch_dep(kern, grid, dim3(kRowThreads), s, c, layer, r, a, status); };
    if (c.format == FMD_CACHE_Q4) return few ? on(k_cache_append<T, D, true, 1>) : on(k_cache_append<T, D, true, kRowHeads>);
    return few ? on(k_cache_append<T, D, false, 1>) : on(k_cache_append<T, D, false, kRowHeads>);
  };
  auto dim = [&](auto t) {
    return c.head_dim == 128 ? go(t, std::integral_constant<int, 128>{}) : go(t, std::integral_constant<int, 64>{});
  };
  return bf16 ? dim(__nv_bfloat16{}) : dim(__half{});
}

cudaError_t launch_cache_fork_one(const CacheView& c, int layers, int* table, int src, int dst, int len, int page,
                                  cudaStream_t s) {
  ForkList l{};
  l.src[0] = src;
  l.dst[0] = dst;
  l.len[0] = len;
  l.page[0] = page;
  const int by = (int)std::min<long long>(((long long)layers * 2 * c.kv_heads + 7) / 8, 148 * 8);
  return launch(k_cache_fork, dim3(1, by), dim3(256), 0, s, c, layers, table, l, (int*)nullptr);
}

// bitmap, map, src, dst, counts
size_t cache_compact_workspace(int n_pages) {
  return 4 * (((size_t)n_pages + 31) / 32 + 3 * (size_t)n_pages + 4);
}

cudaError_t launch_cache_compact(const CacheView& c, int layers, int* table, const int* n_entries, void* workspace,
                                 int* n_used, int* status, cudaStream_t s) {
  const size_t words = ((size_t)c.n_pages + 31) / 32, P = c.n_pages;
  uint32_t* bits = (uint32_t*)workspace;
  int *map = (int*)bits + words, *src = map + P, *dst = src + P, *counts = dst + P;
  cudaError_t e = cudaMemsetAsync(bits, 0, words * 4, s);
  if (e == cudaSuccess) e = launch(k_compact_mark, dim3(c.max_slots), dim3(256), 0, s, c, n_entries, bits, status);
  if (e == cudaSuccess)
    e = launch(k_compact_plan, dim3(1), dim3(1024), 0, s, c.n_pages, bits, map, src, dst, counts, n_used);
  if (e == cudaSuccess) e = launch(k_compact_remap, dim3(c.max_slots), dim3(256), 0, s, c, table, n_entries, map, counts);
  if (e == cudaSuccess) e = launch(k_compact_move, dim3(148 * 8), dim3(256), 0, s, c, layers, src, dst, counts);
  return e;
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

// No rows at all: the row buffers are not looked at (an empty one has no address).
bool empty(const fmd_cache_rows* r) { return r->n_seqs == 0 || r->n_rows == 0; }
bool bad_stride(int64_t s) { return s < 0 || (s & 7); }
HeadRows rows_at(const void* at, int64_t row, int64_t head, int n_rows, int n_heads, int dim) {
  return HeadRows{(uint64_t)reinterpret_cast<uintptr_t>(at), n_rows > 1 ? row : 0, n_heads > 1 ? head : 0,
                  n_rows, n_heads, dim};
}
bool same(const HeadRows& a, const HeadRows& b) { return a.at == b.at && a.row == b.row && a.head == b.head; }

CacheView view_of(const fmd_cache* c) {
  return CacheView{(uint8_t*)c->pool, c->page_table, c->format,    c->n_pages,
                   c->kv_heads,       c->head_dim,   c->max_slots, c->max_pages_per_slot};
}
CacheRows rows_of(const fmd_cache_rows* r) {
  return CacheRows{r->slot, r->pos0, r->row0, nullptr, nullptr, r->n_seqs, r->n_rows};
}
// FMD_EINVAL if a value of dst occurs twice there, or in src.
int check_moves(int n, const int32_t* src, const int32_t* dst) {
  std::unique_ptr<int32_t[]> d(new (std::nothrow) int32_t[n]);
  if (!d) return FMD_ENOMEM;
  std::copy(dst, dst + n, d.get());
  std::sort(d.get(), d.get() + n);
  if (std::adjacent_find(d.get(), d.get() + n) != d.get() + n) return FMD_EINVAL;
  for (int i = 0; src && i < n; ++i)
    if (std::binary_search(d.get(), d.get() + n, src[i])) return FMD_EINVAL;
  return FMD_OK;
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
  if (!a || (a->dtype != FMD_DT_F16 && a->dtype != FMD_DT_BF16)) return FMD_EINVAL;
  if (c->format != FMD_CACHE_Q4 && c->format != a->dtype) return FMD_EINVAL;
  if (a->n_heads < 0 || a->n_heads > 16384) return FMD_EINVAL;
  if (!empty(rows)) {
    if (!a->k || !a->v || !aligned16(a->k) || !aligned16(a->v)) return FMD_EINVAL;
    if ((a->n_heads > 0) != (a->q != nullptr) || (a->q && !a->q_out)) return FMD_EINVAL;
    if (a->q && (!aligned16(a->q) || !aligned16(a->q_out))) return FMD_EINVAL;
  }
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
  if (empty(rows)) return FMD_OK;
  if (a->q) {
    // queries are written while others, keys and values are still read: in place, or nowhere near
    const int n = rows->n_rows, d = c->head_dim;
    const HeadRows out = rows_at(a->q_out, a->q_out_row, a->q_out_head, n, a->n_heads, d);
    const HeadRows q = rows_at(a->q, a->q_row, a->q_head, n, a->n_heads, d);
    if (out.overlaps() || (!same(out, q) && meet(out, q)) ||
        meet(out, rows_at(a->k, a->k_row, a->k_head, n, c->kv_heads, d)) ||
        meet(out, rows_at(a->v, a->v_row, a->v_head, n, c->kv_heads, d)))
      return FMD_EINVAL;
  }
  if (!on_current_device(c->pool) || !on_current_device(a->k)) return FMD_EINVAL;
  CacheAppend p{a->q,      a->k,      a->v,     a->q_out,     a->q_row,     a->q_head, a->k_row,
                a->k_head, a->v_row,  a->v_head, a->q_out_row, a->q_out_head, a->q_norm, a->k_norm,
                a->cos_table, a->sin_table, a->eps, a->n_heads, a->rot_dim, a->table_rows, a->interleaved, nullptr};
  return done(launch_cache_append(a->dtype == FMD_DT_BF16, view_of(c), layer, rows_of(rows), p, status,
                                  (cudaStream_t)stream));
}

int fmd_cache_read(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows, float* k, float* v, int32_t* status,
                   void* stream) {
  int rc = check_cache(c);
  if (rc || (rc = check_rows(c, layer, rows))) return rc;
  if (empty(rows)) return FMD_OK;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return FMD_EINVAL;
  const int64_t elems = (int64_t)rows->n_rows * c->kv_heads * c->head_dim;
  const uintptr_t ka = (uintptr_t)k, va = (uintptr_t)v;
  if (std::max(ka, va) - std::min(ka, va) < (uint64_t)elems * sizeof(float)) return FMD_EINVAL;  // on one another
  if (!on_current_device(c->pool) || !on_current_device(k)) return FMD_EINVAL;
  // blocks of a row: as in append
  const int per_block = kReadThreads / (c->head_dim / 8) * 4, most = (2 * c->kv_heads + per_block - 1) / per_block;
  const dim3 grid(rows->n_rows, rows->n_rows < 148 * 4 ? most : 1);
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return launch_dep(c->format == FMD_CACHE_Q4     ? k_cache_read<D, FMD_CACHE_Q4>
                      : c->format == FMD_CACHE_BF16 ? k_cache_read<D, FMD_CACHE_BF16>
                                                    : k_cache_read<D, FMD_CACHE_F16>,
                      grid, dim3(kReadThreads), (cudaStream_t)stream, view_of(c), layer, rows_of(rows), k, v, status);
  };
  return done(c->head_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{}));
}

int64_t fmd_cache_attend_workspace(const fmd_cache* c, int32_t n_heads, int32_t n_seqs, int32_t max_rows) {
  if (check_cache(c) || n_heads < 1 || n_heads % c->kv_heads || n_seqs < 1 || max_rows < 1) return 0;
  const CacheView v = view_of(c);
  return (int64_t)(cache_decode_fits(v, n_heads, max_rows) ? cache_decode_workspace(v, n_heads, max_rows)
                                                           : cache_chunk_workspace(v));
}

int fmd_cache_attend(const fmd_cache* c, int32_t layer, const fmd_cache_rows* rows, const fmd_cache_attend_args* a,
                     void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  int rc = check_cache(c);
  if (rc || (rc = check_rows(c, layer, rows))) return rc;
  if (!a || (!empty(rows) && (!a->q || !a->out || a->out == a->q || !aligned16(a->q) || !aligned16(a->out))))
    return FMD_EINVAL;
  if (a->dtype != FMD_DT_F16 && a->dtype != FMD_DT_BF16) return FMD_EINVAL;
  if (c->format != FMD_CACHE_Q4 && c->format != a->dtype) return FMD_EINVAL;
  if (a->n_heads < 1 || a->n_heads % c->kv_heads) return FMD_EINVAL;
  const int group = a->n_heads / c->kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8 && group != 16) return FMD_ENOTSUP;
  if (a->window < 0 || a->sinks < 0 || !(a->scale > 0.f) || !(a->scale <= 3.4e38f)) return FMD_EINVAL;
  for (int64_t s : {a->q_row, a->q_head, a->out_row, a->out_head})
    if (bad_stride(s)) return FMD_EINVAL;
  if (empty(rows)) return FMD_OK;
  if (rows->max_rows == 0) return rows->row0 ? FMD_OK : FMD_EINVAL;  // without row0 each sequence has a row
  const HeadRows out = rows_at(a->out, a->out_row, a->out_head, rows->n_rows, a->n_heads, c->head_dim);
  if (out.overlaps() || meet(out, rows_at(a->q, a->q_row, a->q_head, rows->n_rows, a->n_heads, c->head_dim)))
    return FMD_EINVAL;
  const int64_t need = fmd_cache_attend_workspace(c, a->n_heads, rows->n_seqs, rows->max_rows);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return FMD_EINVAL;
  if (cache_units(view_of(c)) * c->kv_heads > INT32_MAX) return FMD_ENOTSUP;
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
  if ((rc = check_moves(n, src, dst))) return rc;
  if (!on_current_device(c->pool)) return FMD_EINVAL;
  for (int i = 0; i < n; i += kCopyBatch) {
    CopyList l;
    const int m = std::min(kCopyBatch, n - i);
    std::memcpy(l.src, src + i, m * sizeof(int));
    std::memcpy(l.dst, dst + i, m * sizeof(int));
    const int grid = (int)std::min<long long>((long long)m * c->layers, 148 * 8);
    const cudaError_t e = launch(k_cache_copy, dim3(grid), dim3(256), 0, (cudaStream_t)stream, view_of(c), c->layers,
                                 l, m);
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
  if ((rc = check_moves(n, src_slot, dst_slot))) return rc;
  {
    std::unique_ptr<int32_t[]> pages(new (std::nothrow) int32_t[n]);
    if (!pages) return FMD_ENOMEM;
    int m = 0;
    for (int i = 0; i < n; ++i)
      if (len[i] % kPageTokens) pages[m++] = new_page[i];
    if ((rc = check_moves(m, nullptr, pages.get()))) return rc;
  }
  if (!on_current_device(c->pool)) return FMD_EINVAL;
  for (int i = 0; i < n; i += kCopyBatch) {
    ForkList l;
    const int m = std::min(kCopyBatch, n - i);
    std::memcpy(l.src, src_slot + i, m * sizeof(int));
    std::memcpy(l.dst, dst_slot + i, m * sizeof(int));
    std::memcpy(l.len, len + i, m * sizeof(int));
    std::memcpy(l.page, new_page + i, m * sizeof(int));
    // a warp per copied block, at most about eight blocks of threads an SM
    const int by = (int)std::min<long long>(((long long)c->layers * 2 * c->kv_heads + 7) / 8, std::max(1, 148 * 8 / m));
    const cudaError_t e = launch(k_cache_fork, dim3(m, by), dim3(256), 0, (cudaStream_t)stream, view_of(c), c->layers,
                                 c->page_table, l, status);
    if (e != cudaSuccess) return done(e);
  }
  return FMD_OK;
}

int64_t fmd_cache_compact_workspace(const fmd_cache* c) {
  if (!c || c->n_pages < 1) return 0;
  return (int64_t)cache_compact_workspace(c->n_pages);
}

int fmd_cache_compact(const fmd_cache* c, const int32_t* n_entries, void* workspace, int64_t workspace_bytes,
                      int32_t* n_used, int32_t* status, void* stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!n_entries || !workspace || !n_used || workspace_bytes < fmd_cache_compact_workspace(c) || !aligned16(workspace))
    return FMD_EINVAL;
  if (!on_current_device(c->pool) || !on_current_device(workspace)) return FMD_EINVAL;
  return done(launch_cache_compact(view_of(c), c->layers, c->page_table, n_entries, workspace, n_used, status,
                                   (cudaStream_t)stream));
}

}  // extern "C"
