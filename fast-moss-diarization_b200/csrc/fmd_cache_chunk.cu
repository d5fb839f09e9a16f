// Attention of many rows per sequence over the paged cache (prompt chunks): the
// form of fmd_cache_attend for more than 16 (row, query head) pairs per kv head.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j
//
// over the visible keys of each row. Every key tile is used by 256 pairs, so the
// bound is arithmetic: 4 x head_dim flop per (pair, visible key) on the tensor
// cores, and one exponential each on the special-function units, which at
// head_dim 128 take as long (64 keys x 256 pairs: 1,082 cycles of tcgen05 at its
// peak, 1,024 cycles of 16 exponentials a cycle).
//
// A work item is two consecutive tiles A, B of 128 pairs (row-major, then the
// query heads of the kv head) of one sequence and kv head: each key tile (a page)
// is read once for both. Its key tiles are those of the sinks, then those from
// A's oldest window to B's newest row; a tile that one of A, B does not see is
// skipped for it. Items are dealt in turn, or, where that would leave blocks idle for
// longer (few items, or items of very different lengths), the items' key tiles form one
// sequence, of which every block takes an equal range: an item cut by a range's end
// leaves (m, l, o) partials in the workspace, and the last of its blocks to finish
// merges them in order.
//
//  * warp 0: copies of the page tiles into a ring (16 bits: 2D TMA with the
//    128-byte swizzle; 4 bits: bulk copies of the blocks);
//  * warp 1 / 2: tcgen05.mma of A / B, f32 accumulators in tensor memory: S(j), then
//    O += P V (j - 1). One warp for both spent 3,350 cycles a key tile, most of them on
//    its waits and commits one after another, for 1,400 cycles of products;
//  * warps 4-7 / 8-11: the softmax of A / B, one thread per pair: a lazily moved
//    reference m (2^8 of headroom), P as 16-bit values over the scores it came from, the
//    A operand of its product with V, O rescaled only when m moves;
//  * 4 bits: warps 12-15 turn the codes into f16 tiles, (c - 8) d with one rounding,
//    keys and values; the queries are then f16 too, scaled by a power of two per
//    row.
// Registers go where they are needed: the softmax groups take what the others give.
// Values of positions that no pair of the item sees are cleared in shared memory
// before the product, so that what they hold (NaN x 0) has no influence.
// Roundings: P enters its product as one 16-bit term, as in the decoder's prefill attention,
// and from 16 bits that shows: outputs are off by 2.3e-3 of their magnitude (rms; f16 2.9e-4)
// where their own rounding alone is 1.7e-3 (2.1e-4). With a second term for what the first
// leaves out, as the decode form has, 1.7e-3 as well, but 220 us instead of 180 for the two
// chunks below.
// Measured (16 query heads to 8 kv heads of 128), launches back to back: 2,048 rows behind
// 8,192 positions 170 us, 909 TFLOP/s; two chunks of 2,048 behind 3,952 and 12,288 positions,
// window 4,096, 175 us, 786 TFLOP/s; the last 2,001 f16 rows of 9,001 positions in 4 bits 249 us,
// 527 TFLOP/s of 4 x head_dim a key (twice the products of P V are issued there). With inputs
// cold in L2 the last two take 180 and 255 us. A key tile of A and B takes 2,000
// cycles (4 bits: 3,900), an item's queries and outputs 8,000 more. Of the 2,000, a
// softmax warp spends 900 on its exponentials, the special-function unit half busy with
// those of A and B; no pipe is full (tensor 44 %, issue 37 %). A quarter of the
// exponentials as polynomials took 177 us instead of 173, half of them 183; one score
// buffer beside a P of its own, which lets S(j + 1) start before P V (j - 1), 185.
// Every wait is bounded; a timeout sets the status word, stops issuing work,
// waits (bounded) for copies and MMAs in flight and frees tensor memory.
#include <cuda.h>
#include <float.h>
#include <limits.h>

#include <algorithm>

#include "fmd_cache.cuh"
#include "fmd_kernels.cuh"

namespace fmd {

namespace {

constexpr int kCkBox = 8192;       // 64 rows x 128 bytes
constexpr int kCkMaxStages = 4;
constexpr uint32_t kCkWait = 1u << 24;
constexpr float kCkHeadroom = 8.f;

constexpr int kCkConv = 4;  // converter warps (4 bits)
constexpr int ck_threads(bool q4) { return 384 + (q4 ? kCkConv * 32 : 0); }
// Registers of a thread at launch, of a softmax thread, of any other; the sums fit.
//   16 bits: 384 x 168 = 256 x 208 + 128 x 88; 4 bits: 512 x 128 = 256 x 192 + 256 x 64.
// Eight converter warps leave 152 to a softmax thread, which then spills more: 241 us instead of
// 234 for the f16 chunk above. As it is, the compiler reports 60 bytes of spill stores a thread
// (16 bits) and 72 to 80 (4 bits).
template <int N> FMD_DEV void ck_more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N> FMD_DEV void ck_fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

struct CkArgs {
  CacheRows r;
  CacheAttend a;
  // partials of cut items: o as [2 x blocks][D / 4][256 pairs] of four dims, so that a warp's
  // threads, a pair each, write and read runs; then [2 x blocks][256] (m, l)
  float* part;
  int* counters;  // [(sequence, tile)][kv heads], zero between calls
  int tiles;      // 256-pair tiles of the longest sequence
  int split, stages;  // split: items may be cut
  uint32_t f64;   // f16 pair (64, 64)
};

FMD_DEV void ck_fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
FMD_DEV float ck_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 lanes at once, each rounded as the scalar instruction rounds.
FMD_DEV float2 ck_fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
FMD_DEV float2 ck_add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
// Descriptor of an MN-major operand with the 128-byte swizzle: 64 elements of the
// MN dimension per 128-byte row, a row per K index, MN blocks kCkBox apart.
FMD_DEV uint64_t ck_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((kCkBox >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// N consecutive columns of this warp's 32 lanes, there when the statement ends. The
// wait is part of it: between a load and a wait of their own the compiler could move or
// spill registers that the load has not written yet.
FMD_DEV void ck_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31"
      "}, [%32];\n tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
FMD_DEV void ck_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, "
      "%38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, "
      "%56, %57, %58, %59, %60, %61, %62, %63"
      "}, [%64];\n tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
        "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
// D[tmem] (+)= A[tmem] x B[smem], K = 16: A's rows are lanes, two 16-bit values a column.
FMD_DEV void ck_umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
FMD_DEV uint32_t ck_sub_mul(uint32_t a, uint32_t b, uint32_t d) {
  const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  const __half2 y = __hmul2(x, *reinterpret_cast<__half2*>(&d));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// What rounding a product of ck_sub_mul left out, (a - b) d - o: exact in f16, but for
// what is below its subnormals.
FMD_DEV uint32_t ck_sub_mul_rest(uint32_t a, uint32_t b, uint32_t d, uint32_t o) {
  const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  const __half2 y = __hfma2(x, *reinterpret_cast<__half2*>(&d), __hneg2(*reinterpret_cast<__half2*>(&o)));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// One item part of a CTA: tiles A and B of a sequence and kv head, key tiles
// [j0, j1) of the item's list.
struct CkWork {
  int slot, p0, r0, h;
  int first[2], count[2];  // first pair and pairs (0: none) of A, B
  int lo[2], hi[2];        // positions of their first and last row
  int sinks, w0;           // the item's key tiles: sinks, then from w0
  int lim, from[2], end[2];  // those A / B see: before lim, or from from[x] on, before end[x]
  int j0, j1, item, units;
  bool inside;      // the whole item is this work
  long long start;  // else: the item's first unit, for its other blocks
  FMD_DEV int tile(int j) const { return j < sinks ? j : w0 + j - sinks; }
};
// What concerns one of A, B, in registers of its own (a run-time index into
// CkWork's arrays would put them in local memory).
struct CkSide {
  int first, count, lim, from, end;
  FMD_DEV CkSide(const CkWork& w, int x)
      : first(x ? w.first[1] : w.first[0]),
        count(x ? w.count[1] : w.count[0]),
        lim(w.lim),
        from(x ? w.from[1] : w.from[0]),
        end(x ? w.end[1] : w.end[0]) {}
  FMD_DEV bool need(int j) const { return j < end && (j < lim || j >= from); }
};

// Bounded wait with one outcome for the warp; gives up early when another role has.
FMD_DEV bool ck_wait(uint64_t* bar, uint32_t parity, volatile int* abort_v) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1; !ok && i < kCkWait; ++i) {
      ok = mbar_try_wait(bar, parity);
      if (!ok && (*abort_v || ((i & 63) == 0 && globaltimer_ns() - t0 > kWaitNsCap))) break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Item (seq, tile) without its kv head and key range: its number of key tiles, 0 if
// there is none.
FMD_DEV int ck_item(const CkArgs& p, const CacheView& c, int seq, int tile, CkWork& w, int* status) {
  int n;
  p.r.get(seq, w.slot, w.p0, w.r0, n);
  if (n <= 0 || !cache_slot_ok(c, w.slot, status)) return 0;
  if (n > p.a.max_rows || w.p0 < 0 || w.p0 > c.max_pages * kPageTokens - n) {
    cache_report(status, n > p.a.max_rows ? FMD_EINVAL : FMD_EOVERFLOW);
    return 0;
  }
  const int gs = __ffs(p.a.n_heads / c.kv_heads) - 1;
  const long long pairs = (long long)n << gs;
  const long long f = (long long)tile * 256;
  if (f >= pairs) return 0;
  const int W = p.a.window, S = W ? p.a.sinks : 0;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    w.first[x] = (int)(f + x * 128);
    w.count[x] = (int)max(0LL, min(128LL, pairs - w.first[x]));
    w.lo[x] = w.p0 + (w.first[x] >> gs);
    w.hi[x] = w.p0 + ((w.first[x] + max(w.count[x], 1) - 1) >> gs);
  }
  const int oldest = W && w.lo[0] >= W ? w.lo[0] - W + 1 : 0;
  w.w0 = oldest / kPageTokens;
  w.sinks = (min(S, w.w0 * kPageTokens) + kPageTokens - 1) / kPageTokens;
  w.lim = w.sinks + max(0, (min(S, w.hi[1]) + kPageTokens - 1) / kPageTokens - w.w0);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    w.from[x] = w.sinks + (W && w.lo[x] >= W ? w.lo[x] - W + 1 : 0) / kPageTokens - w.w0;
    w.end[x] = w.count[x] > 0 ? w.sinks + w.hi[x] / kPageTokens - w.w0 + 1 : 0;
  }
  return w.sinks + (w.count[1] > 0 ? w.hi[1] : w.hi[0]) / kPageTokens - w.w0 + 1;
}

constexpr int kCkEntries = 1024;  // (sequence, tile) pairs of a split launch at most
// Units of an item beside its key tiles: what its queries, its first scores and its
// output cost, about two tiles.
constexpr int kCkSetup = 2;
constexpr int kCkLeast = 6;       // units of a range at least
// What cutting costs a block, in units (1.2 us; 4 bits 1.5 us): the partials' way through
// memory and the merge. 16 bits: 256 items of 70 units (two rounds of 148 blocks, 17 % of
// them idle) take 173 us whole and 169 cut, 64 items of 72 units 88 and 65, 128 items of
// 35 to 66 units 48 either way. 4 bits: the last 56 and 60, 128 items of 143 to 174 units
// 261 and 234.
constexpr int ck_cut(bool q4) { return q4 ? 24 : 16; }

// This block's range of units, and the units before each (sequence, tile).
struct CkPlan {
  int prefix[kCkEntries + 1];
};
struct CkRange {
  long long x0, x1, total;  // of units; whole items: total counts them
  int G;                    // blocks with a range
  bool whole;
};
struct CkIter {
  long long x;
  int round = 0;
};

// The block's next work: 1 a work, 0 none (skip), -1 no more.
FMD_DEV int ck_next(const CkArgs& p, const CacheView& c, const CkPlan& plan, const CkRange& g, CkIter& it, CkWork& w) {
  const int H = c.kv_heads, ns = p.r.count();
  if (p.split) {
    if (g.whole) {
      // the last pairs (the latest rows of a prompt) first, every other round the other way round
      const long long G = gridDim.x;
      if (it.round * G >= g.total) return -1;
      it.x = g.total - 1 - (it.round * G + ((it.round & 1) ? G - 1 - blockIdx.x : blockIdx.x));
      ++it.round;
      if (it.x < 0) return 0;
    } else if (it.x >= g.x1) {
      return -1;
    }
    int lo = 0, hi = ns * p.tiles - 1;  // the last pair with units that starts at or before x
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)H * plan.prefix[mid] <= it.x) lo = mid;
      else hi = mid - 1;
    }
    w.units = plan.prefix[lo + 1] - plan.prefix[lo];
    const int off = (int)(it.x - (long long)H * plan.prefix[lo]);
    w.h = off / w.units;
    w.item = lo * H + w.h;
    if (g.whole) {
      w.j0 = 0;
      w.j1 = ck_item(p, c, lo / p.tiles, lo % p.tiles, w, nullptr);
      w.inside = true;
      return 1;
    }
    const int j = off - w.h * w.units, len = (int)min((long long)(w.units - j), g.x1 - it.x);
    ck_item(p, c, lo / p.tiles, lo % p.tiles, w, nullptr);
    w.j0 = max(j - kCkSetup, 0);
    w.j1 = max(j + len - kCkSetup, 0);
    w.inside = len == w.units;
    w.start = it.x - j;
    it.x += len;
    return 1;
  }
  // latest rows first, every other round the other way round
  const long long G = gridDim.x, total = (long long)p.tiles * ns * H;
  const long long at = it.round * G + ((it.round & 1) ? G - 1 - blockIdx.x : blockIdx.x);
  if (it.round * G >= total) return -1;
  ++it.round;
  if (at >= total) return 0;
  w.h = (int)(at % H);
  w.j0 = 0;
  w.j1 = ck_item(p, c, ns - 1 - (int)(at / H % ns), p.tiles - 1 - (int)(at / H / ns), w, nullptr);
  w.inside = true;
  return w.j1 > 0;
}

template <typename T, int D, bool Q4>
__global__ void __launch_bounds__(ck_threads(Q4), 1)
    k_cache_chunk(const __grid_constant__ CUtensorMap tmap, CacheView c, int layer, CkArgs p, int* status) {
  using M = typename std::conditional<Q4, __half, T>::type;
  constexpr int QB = 128 * D * 2;                             // one query tile
  constexpr int BLK = Q4 ? 64 * (D / 2 + D / 16) : 64 * D * 2;  // K or V of a page as stored
  constexpr int TB = 64 * D * 2;                              // K or V of a page as an operand
  constexpr int NB = D / 32;
  constexpr int kMore = Q4 ? 192 : 208, kFew = Q4 ? 64 : 88;
  // f16 outputs of a 4-bit cache: P and V go in as two f16 terms each (their roundings,
  // 2^-11 each as the output's, would be two of the three that f16 operands cost; error
  // against 64 bits 2.7e-4 so, 3.8e-4 without, 2.1e-4 for the output's rounding alone)
  constexpr bool kFine = Q4 && !Act<T>::kIsBf16;
  constexpr int CVB = (kFine ? 3 : 2) * TB;  // an operand buffer: K | V (| V's second term)
  constexpr float kPScale = Act<M>::kIsBf16 ? 0.f : 7.f;      // log2 factor of P (f16 subnormals start at 2^-14)
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], kv_full[kCkMaxStages], kv_empty[kCkMaxStages], cv_full[2][2], cv_empty[2][2],
      s_full[2][2], p_full[2][2], pv_done[2], o_final[2], o_empty[2], mma_done[2];
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s, bad_s[kCkMaxStages], cbad_s[4], last_s;
  __shared__ CkPlan plan;
  __shared__ CkRange range;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* qp = base;                      // Q_A | Q_B | stages | (4 bits) two operand tiles
  uint8_t* kvp = qp + 2 * QB;
  uint8_t* cvp = kvp + p.stages * 2 * BLK;
  const int stages = p.stages, H = c.kv_heads;
  const int W = p.a.window, S = W ? p.a.sinks : 0;

  griddep_wait();
  griddep_launch();
  if (p.r.count() <= 0) return;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], Q4 ? kCkConv : 2);
    }
    for (int x = 0; x < 2; ++x) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&cv_full[x][b], kCkConv);
        mbar_init(&cv_empty[x][b], 2);
      }
      mbar_init(&mma_done[x], 1);
      mbar_init(&q_full[x], 4);
      for (int s = 0; s < 2; ++s) {
        mbar_init(&s_full[x][s], 1);
        // one per buffer: a warp may be a tile ahead of its group, whose P(j) is not complete
        mbar_init(&p_full[x][s], 4);
      }
      mbar_init(&pv_done[x], 1);
      mbar_init(&o_final[x], 1);
      mbar_init(&o_empty[x], 4);
    }
    abort_s = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_s, 512);
    tmem_relinquish();
  }
  CkIter it;
  const int entries = p.r.count() * p.tiles;
  if (p.split) {
    for (int e = tid; e < entries; e += ck_threads(Q4)) {
      CkWork w;
      const int n = ck_item(p, c, e / p.tiles, e % p.tiles, w, status);
      plan.prefix[e] = n > 0 ? n + kCkSetup : 0;
    }
    __syncthreads();
    if (warp == 0) {
      // each lane a run of pairs
      const int per = (entries + 31) / 32, e0 = min(lane * per, entries), e1 = min(e0 + per, entries);
      int sum = 0, have = 0, most = 0;
      for (int e = e0; e < e1; ++e) {
        const int v = plan.prefix[e];
        sum += v;
        have += v > 0;
        most = max(most, v);
      }
      const long long units = (long long)H * __reduce_add_sync(0xffffffffu, (unsigned)sum);
      const int items = H * (int)__reduce_add_sync(0xffffffffu, (unsigned)have), G = gridDim.x;
      most = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
      // whole items: the longest, or as many rounds of average ones; cut ones: an equal share
      const bool whole = items > 0 && max((long long)most, (items + G - 1) / G * (units / items)) <= units / G + ck_cut(Q4);
      if (whole) sum = have;
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      int run = incl - sum;
      for (int e = e0; e < e1; ++e) {
        const int v = whole ? plan.prefix[e] > 0 : plan.prefix[e];
        plan.prefix[e] = run;
        run += v;
      }
      if (lane == 31) {
        plan.prefix[entries] = incl;
        range.whole = whole;
        range.total = (long long)H * incl;
        range.G = (int)max(1LL, min((long long)G, range.total / kCkLeast));
        const bool has = (int)blockIdx.x < range.G;
        range.x0 = has ? (long long)blockIdx.x * range.total / range.G : 0;
        range.x1 = has ? (long long)(blockIdx.x + 1) * range.total / range.G : 0;
      }
    }
  } else if (blockIdx.x == 0) {
    // bad slots and positions are reported once
    for (int e = tid; e < entries; e += ck_threads(Q4)) {
      CkWork w;
      ck_item(p, c, e / p.tiles, e % p.tiles, w, status);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  it.x = p.split ? range.x0 : 0;
  const uint32_t tmem = tmem_s;
  volatile int* abort_v = &abort_s;

  if (warp < 4) {
  ck_fewer_regs<kFew>();
  if (warp == 0) {
    // ---------------- copies ----------------
    if (lane == 0) {
      if (!Q4) prefetch_tmap(&tmap);
      int issued = 0, s = 0, round_s = 0;
      bool ok = true;
      CkWork w;
      for (int k; ok && (k = ck_next(p, c, plan, range, it, w)) >= 0;) {
        if (k == 0) continue;
        const int* table = c.page_table + (size_t)w.slot * c.max_pages;
        for (int j = w.j0; j < w.j1; ++j) {
          if (round_s > 0 && (*abort_v || !mbar_wait_bounded(&kv_empty[s], (round_s - 1) & 1, kCkWait))) {
            ok = false;
            break;
          }
          const int page = table[w.tile(j)];
          const bool bad = page < 0 || page >= c.n_pages;
          bad_s[s] = bad;
          if (bad) {
            cache_report(status, FMD_EINVAL);
            mbar_arrive(&kv_full[s]);
          } else {
            uint8_t* dst = kvp + s * 2 * BLK;
            mbar_arrive_expect_tx(&kv_full[s], 2 * BLK);
            if constexpr (Q4) {
              bulk_load(dst, c.block(layer, page, 0, w.h), BLK, &kv_full[s]);
              bulk_load(dst + BLK, c.block(layer, page, 1, w.h), BLK, &kv_full[s]);
            } else {
              const int yk = (page * 2 * H + w.h) * kPageTokens, yv = yk + H * kPageTokens;
#pragma unroll
              for (int b = 0; b < D / 64; ++b) {
                tma_load_2d(dst + b * kCkBox, &tmap, b * 64, yk, &kv_full[s]);
                tma_load_2d(dst + BLK + b * kCkBox, &tmap, b * 64, yv, &kv_full[s]);
              }
            }
          }
          ++issued;
          if (++s == stages) s = 0, ++round_s;
        }
      }
      if (!ok) *abort_v = 1;
      // copies still in flight land before the CTA retires (bounded)
      for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
        mbar_wait_bounded(&kv_full[i % stages], (i / stages) & 1, kCkWait);
    }
  } else if (warp == 1 || warp == 2) {
    // ---------------- MMAs of tile x: the whole warp runs the loop, the elected lane issues ----------------
    const int x = warp - 1;
    constexpr bool kBf = Act<M>::kIsBf16;
    constexpr uint32_t idesc_s = umma_idesc_f16(kBf, 128, 64);
    constexpr uint32_t idesc_o = umma_idesc_f16(kBf, 128, D) | (1u << 16);  // B (V) MN-major
    // scores and products issued; products known to be done: at most one is not, since
    // the parity that pv_done is waited with tells one phase from the next, not from the one after
    int items = 0, sn = 0, pn = 0, done = 0;
    int st = 0, ph = 0;  // operand tile of the next key tile: its stage (4 bits: buffer) and phase
    int prev_ph = 0;
    const int ring = Q4 ? 2 : stages;
    // 4 bits: keys and values come and go by themselves; keys are free long before values
    uint64_t* full = Q4 ? cv_full[0] : kv_full;
    uint64_t* empty = Q4 ? cv_empty[1] : kv_empty;
    uint8_t* tiles = Q4 ? cvp : kvp;
    const uint32_t s_tmem = tmem + x * 256, o_tmem = s_tmem + 128;
    // descriptors of the first operand tiles; addresses below 256 KB never carry out of
    // the address field, so the others are sums
    const uint64_t dq = umma_desc_sw128(smem_u32(qp) + x * QB);
    constexpr int SB = Q4 ? CVB : 2 * TB;  // bytes from tile to tile
    const uint64_t dk = umma_desc_sw128(smem_u32(tiles)), dv = ck_desc_mn(smem_u32(tiles) + TB);
    bool ok = true;
    CkWork w;
    for (int k; ok && (k = ck_next(p, c, plan, range, it, w)) >= 0;) {
      if (k == 0) continue;
      const CkSide side(w, x);
      const int top = w.count[1] > 0 ? w.hi[1] : w.hi[0], low = w.lo[0];
      bool started = false, got_q = false;  // O holds a product, the queries are there
      int prev_st = 0;                      // operand tile of key tile j - 1
      for (int j = w.j0; j <= w.j1; ++j) {
        if (j < w.j1) {
          if (!(ok = ck_wait(&full[st], ph, abort_v))) break;
          if (side.need(j)) {
            // ---- S(j) = Q K^T
            if constexpr (!Q4) {
              // clear the values of positions that neither A nor B sees (both warps: the same zeros)
              const int k0 = w.tile(j) * kPageTokens;
              const bool bad = bad_s[st];
              if (bad || k0 + 63 > top || (W && k0 <= low - W && k0 + 63 >= S)) {
                for (int i = lane; i < 64 * (D / 64); i += 32) {
                  const int key = k0 + (i & 63);
                  if (bad || key > top || (W && key <= low - W && key >= S)) {
                    uint4* row =
                        reinterpret_cast<uint4*>(tiles + st * 2 * TB + TB + (i >> 6) * kCkBox + (i & 63) * 128);
#pragma unroll
                    for (int b = 0; b < 8; ++b) row[b] = make_uint4(0, 0, 0, 0);
                  }
                }
                ck_fence_async();
                __syncwarp();
              }
            }
            const int sb = sn & 1;
            if (!got_q) {
              if (!(ok = ck_wait(&q_full[x], items & 1, abort_v))) break;
              got_q = true;
            }
            // the buffer's last scores became a P whose product, the one two back, has to be done
            if (done < sn - 1) {
              if (!(ok = ck_wait(&pv_done[x], (pn - 1) & 1, abort_v))) break;
              done = pn;
            }
            tc_fence_after();
            const uint64_t kd = dk + (uint64_t)(st * (SB / 16));
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                umma_f16(s_tmem + sb * 64, dq + ((kk >> 2) * 2 * kCkBox + (kk & 3) * 32) / 16,
                         kd + ((kk >> 2) * kCkBox + (kk & 3) * 32) / 16, idesc_s, kk != 0);
              umma_commit(&s_full[x][sb]);
              if (Q4) umma_commit(&cv_empty[0][st]);
            }
            __syncwarp();
            ++sn;
          } else if (Q4 && lane == 0) {
            mbar_arrive(&cv_empty[0][st]);
          }
        }
        if (j > w.j0) {
          if (side.need(j - 1)) {
            // ---- O += P(j - 1) V
            if (!started && items >= 1 && !(ok = ck_wait(&o_empty[x], (items - 1) & 1, abort_v))) break;
            if (!(ok = ck_wait(&p_full[x][pn & 1], (pn >> 1) & 1, abort_v))) break;
            if (Q4 && !(ok = ck_wait(&cv_full[1][prev_st], prev_ph, abort_v))) break;
            if (done < pn) {  // not in a row of needed tiles, where S(j) has waited for it
              if (!(ok = ck_wait(&pv_done[x], (pn - 1) & 1, abort_v))) break;
              done = pn;
            }
            tc_fence_after();
            const uint64_t vd = dv + (uint64_t)(prev_st * (SB / 16));
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                ck_umma_ts(o_tmem, s_tmem + (pn & 1) * 64 + kk * 8, vd + kk * 2048 / 16, idesc_o, started || kk != 0);
              if constexpr (kFine) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                  ck_umma_ts(o_tmem, s_tmem + (pn & 1) * 64 + 32 + kk * 8, vd + kk * 2048 / 16, idesc_o, true);
                  ck_umma_ts(o_tmem, s_tmem + (pn & 1) * 64 + kk * 8, vd + (TB + kk * 2048) / 16, idesc_o, true);
                }
              }
              umma_commit(&pv_done[x]);
              umma_commit(&empty[prev_st]);  // this warp's products have read the tile when it fires
            }
            __syncwarp();
            started = true;
            ++pn;
          } else {
            // (4 bits: the buffer is free only once it has been filled)
            if (Q4 && !(ok = ck_wait(&cv_full[1][prev_st], prev_ph, abort_v))) break;
            if (lane == 0) mbar_arrive(&empty[prev_st]);
          }
        }
        if (j < w.j1) {
          prev_st = st;
          prev_ph = ph;
          if (++st == ring) st = 0, ph ^= 1;
        }
      }
      if (!ok) break;
      if (started) {
        if (elect_one()) umma_commit(&o_final[x]);
        __syncwarp();
        ++items;
      }
    }
    if (!ok) *abort_v = 1;
    if (elect_one()) umma_commit(&mma_done[x]);  // every MMA issued so far has completed when this fires
    __syncwarp();
    mbar_wait_warp(&mma_done[x], 0, kCkWait);
  }
  } else if (warp < 12) {
    ck_more_regs<kMore>();
    // ---------------- softmax and output of tile x: one thread per pair ----------------
    const int x = (warp - 4) >> 2, q4 = warp & 3, row = q4 * 32 + lane;
    const int gs = __ffs(p.a.n_heads / H) - 1;
    const uint32_t lane_addr = tmem + ((uint32_t)(q4 * 32) << 16) + x * 256, o_addr = lane_addr + 128;
    // tensor-memory loads and stores are warp-wide: a wait counts for all lanes or none
    auto wwait = [&](uint64_t* bar, uint32_t parity) -> bool { return ck_wait(bar, parity, abort_v); };
    int sn = 0, pn = 0, items = 0;
    bool ok = true;
    // where the next key tile's flag is. 4 bits: key tile j mod 4, written again once S(j + 2) is
    // done, before which this group's MMA warp has waited for P(j)
    int cb = 0;
    const int ring = Q4 ? 4 : stages;
    CkWork w;
    // a warp whose wait gave up goes on without work: the merge's barriers below count every warp
    for (int kd; (ok || p.split) && (kd = ck_next(p, c, plan, range, it, w)) >= 0;) {
      if (kd == 0) continue;
      const CkSide side(w, x);
      bool any = false;
      for (int j = w.j0; j < w.j1 && !any && ok; ++j) any = side.need(j);
      float m_ref = -INFINITY, l = 0.f, scale = p.a.scale * 1.4426950408889634f;
      const bool live = row < side.count;
      const int pos = w.p0 + ((side.first + row) >> gs);
      // queries come and outputs go through the query operand's rows, which the warp has to
      // itself, with D / 8 lanes a row (a row a lane: 177 us instead of 172, two chunks of 2,048 rows
      // over a window of 4,096)
      constexpr int LR = D / 8, RL = 32 / LR;
      const int ch = lane & (LR - 1);
      auto row_of = [&](int i) { return q4 * 32 + i * RL + lane / LR; };  // step i's row of this lane
      auto pair_at = [&](int r, long long row_stride, long long head_stride) {
        const int pr = side.first + r;
        return (size_t)(w.r0 + (pr >> gs)) * row_stride + (size_t)((w.h << gs) + (pr & ((1 << gs) - 1))) * head_stride;
      };
      auto chunk_at = [&](int r, int c8) {  // 16-byte chunk c8 of row r of the query operand
        return reinterpret_cast<uint4*>(qp + x * QB + (c8 >> 3) * 2 * kCkBox + r * 128 + (((c8 & 7) ^ (r & 7)) << 4));
      };
      auto flush = [&]() {
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < LR; ++i)
          if (row_of(i) < side.count)
            *reinterpret_cast<uint4*>((T*)p.a.out + pair_at(row_of(i), p.a.out_row, p.a.out_head) + ch * 8) =
                *chunk_at(row_of(i), ch);
        __syncwarp();
      };
      if (any) {
        // ---- queries into the operand tile. The last part's scores are complete (their
        // s_full was waited for), so its queries are no longer read
        uint4 u[LR];
        if constexpr (Q4) {
          // a row a lane, for the row's scale
          const T* src = (const T*)p.a.q + pair_at(row, p.a.q_row, p.a.q_head);
#pragma unroll
          for (int i = 0; i < LR; ++i)
            u[i] = live ? *reinterpret_cast<const uint4*>(src + i * 8) : make_uint4(0, 0, 0, 0);
          float amax = 0.f;
#pragma unroll
          for (int i = 0; i < LR; ++i) {
            const uint32_t v[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = Act<T>::unpack2(v[e]);
              amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
          // 2^e brings the largest magnitude to [1, 2), or to [2, 4) where 2^e would not be normal
          const int e2 = max(-126, min(126, amax > 0.f && amax <= FLT_MAX ? 127 - (int)(__float_as_uint(amax) >> 23) : 0));
          const float up = __uint_as_float((uint32_t)(127 + e2) << 23);
          scale *= __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
          for (int i = 0; i < LR; ++i) {
            uint32_t v[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = Act<T>::unpack2(v[e]);
              v[e] = Act<__half>::pack2(f.x * up, f.y * up);
            }
            *chunk_at(row, i) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < LR; ++i)
            u[i] = row_of(i) < side.count ? *reinterpret_cast<const uint4*>(
                                                (const T*)p.a.q + pair_at(row_of(i), p.a.q_row, p.a.q_head) + ch * 8)
                                          : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < LR; ++i) *chunk_at(row_of(i), ch) = u[i];
        }
        ck_fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[x]);
      }
      bool first = true;
      for (int j = w.j0; j < w.j1 && ok; ++j) {
        const int k0 = w.tile(j) * kPageTokens, stage = cb;
        if (++cb == ring) cb = 0;
        if (!side.need(j)) continue;
        const int sb = sn & 1;
        if (!wwait(&s_full[x][sb], (sn >> 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[64];
        {
          uint32_t v[64];
          ck_ld64(lane_addr + sb * 64, v);
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] = __uint_as_float(v[i]);
        }
        ++sn;
        const bool bad = Q4 ? cbad_s[stage] : bad_s[stage];
        if (bad || k0 + 63 > pos || (W && k0 <= pos - W && k0 + 63 >= S)) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (bad || k0 + i > pos || (W && k0 + i <= pos - W && k0 + i >= S)) s[i] = -INFINITY;
        }
        float mc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mc[i] = s[i];
#pragma unroll
        for (int i = 8; i < 64; ++i) mc[i & 7] = fmaxf(mc[i & 7], s[i]);
#pragma unroll
        for (int i = 1; i < 8; ++i) mc[0] = fmaxf(mc[0], mc[i]);
        const float mx = mc[0] * scale;  // the scale is positive
        bool moves = false;
        if (first) m_ref = mx;
        else moves = mx > m_ref + kCkHeadroom;
        if (__any_sync(0xffffffffu, moves)) {
          // O is complete up to the last P V of this tile
          if (!wwait(&pv_done[x], (pn - 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float f = moves ? ck_ex2(m_ref - mx) : 1.f;  // 0 when the row saw nothing yet
#pragma unroll
          for (int h2 = 0; h2 < D / 32; ++h2) {
            uint32_t v[32];
            ck_ld32(o_addr + h2 * 32, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
            tmem_st32(o_addr + h2 * 32, v);
          }
          tmem_st_wait();
          if (moves) {
            l *= f;
            m_ref = mx;
          }
        }
        {
          const float b = m_ref == -INFINITY ? 0.f : m_ref - kPScale;
          float2 a4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) a4[i] = make_float2(0.f, 0.f);
          const float2 sc2 = make_float2(scale, scale), nb = make_float2(-b, -b);
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            float2 v = ck_fma2(make_float2(s[i], s[i + 1]), sc2, nb);
            v.x = ck_ex2(v.x);
            v.y = ck_ex2(v.y);
            s[i] = v.x;
            s[i + 1] = v.y;
            a4[(i >> 1) & 3] = ck_add2(a4[(i >> 1) & 3], v);
          }
          l += ((a4[0].x + a4[0].y) + (a4[1].x + a4[1].y)) + ((a4[2].x + a4[2].y) + (a4[3].x + a4[3].y));
        }
        {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = Act<M>::pack2(s[2 * i], s[2 * i + 1]);
          tmem_st32(lane_addr + sb * 64, v);
          if constexpr (kFine) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float2 f = Act<M>::unpack2(v[i]);
              v[i] = Act<M>::pack2(s[2 * i] - f.x, s[2 * i + 1] - f.y);
            }
            tmem_st32(lane_addr + sb * 64 + 32, v);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x][sb]);
        ++pn;
        first = false;
      }
      if (ok && any) {
        if (wwait(&o_final[x], items & 1)) tc_fence_after();
        else ok = false;
      }
      if (!ok) {
        any = false;
        *abort_v = 1;
      }
      // a cut item's partial: slot 2 c holds an item that began in an earlier block, 2 c + 1 one
      // that goes on in a later one
      float2* ml = reinterpret_cast<float2*>(p.part + (size_t)2 * gridDim.x * 256 * D);
      const size_t pslot = 2 * blockIdx.x + (w.start < range.x0 ? 0 : 1);
      float4* pt = w.inside ? nullptr : reinterpret_cast<float4*>(p.part) + pslot * (D / 4) * 256 + x * 128 + row;
      const float inv = 1.f / l;
      if (any) {
#pragma unroll
        for (int h2 = 0; h2 < D / 32; ++h2) {
          uint32_t v[32];
          ck_ld32(o_addr + h2 * 32, v);
          if (!live) {
          } else if (pt) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(pt + (h2 * 8 + i) * 256) =
                  make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 y;
              y.x = Act<T>::pack2(__uint_as_float(v[8 * i + 0]) * inv, __uint_as_float(v[8 * i + 1]) * inv);
              y.y = Act<T>::pack2(__uint_as_float(v[8 * i + 2]) * inv, __uint_as_float(v[8 * i + 3]) * inv);
              y.z = Act<T>::pack2(__uint_as_float(v[8 * i + 4]) * inv, __uint_as_float(v[8 * i + 5]) * inv);
              y.w = Act<T>::pack2(__uint_as_float(v[8 * i + 6]) * inv, __uint_as_float(v[8 * i + 7]) * inv);
              *chunk_at(row, h2 * 4 + i) = y;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[x]);
        ++items;
        if (!pt) flush();
      }
      if (pt) {
        if (live) ml[pslot * 256 + x * 128 + row] = make_float2(m_ref, l);
        // the last block of the item to get here merges all, a thread its pair
        auto block_of = [&](long long u) { return (int)(((u + 1) * range.G - 1) / range.total); };
        const int cf = block_of(w.start), np = block_of(w.start + w.units - 1) - cf + 1;
        named_sync(1, 256);
        if (tid == 128) {
          __threadfence();
          last_s = atomicAdd(&p.counters[w.item], 1) == np - 1;
          if (last_s) {
            __threadfence();
            p.counters[w.item] = 0;
          }
        }
        named_sync(1, 256);
        const bool last = last_s;
        if (last) {
          auto at = [&](int sp) { return (size_t)(2 * (cf + sp) + (sp == 0 ? 1 : 0)); };
          const int k = x * 128 + row;
          float Mx = -INFINITY, L = 0.f;
#pragma unroll 4
          for (int sp = 0; sp < np; ++sp)
            if (live) Mx = fmaxf(Mx, __ldcg(&ml[at(sp) * 256 + k]).x);
          const float b = Mx == -INFINITY ? 0.f : Mx;
          constexpr int C = Q4 ? 8 : 16;  // float4s at a time: their loads are in flight together
          for (int c0 = 0; c0 < D / 4 && live; c0 += C) {
            float4 acc[C];
#pragma unroll
            for (int i = 0; i < C; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            L = 0.f;
            for (int sp = 0; sp < np; ++sp) {
              const float2 v = __ldcg(&ml[at(sp) * 256 + k]);
              if (v.y == 0.f) continue;  // the part saw none of the pair's keys and left its row alone
              const float4* src = reinterpret_cast<const float4*>(p.part) + (at(sp) * (D / 4) + c0) * 256 + k;
              float4 u[C];
#pragma unroll
              for (int i = 0; i < C; ++i) u[i] = __ldcg(src + i * 256);
              const float f = ck_ex2(v.x - b);
              L = fmaf(v.y, f, L);
#pragma unroll
              for (int i = 0; i < C; ++i) {
                acc[i].x = fmaf(u[i].x, f, acc[i].x);
                acc[i].y = fmaf(u[i].y, f, acc[i].y);
                acc[i].z = fmaf(u[i].z, f, acc[i].z);
                acc[i].w = fmaf(u[i].w, f, acc[i].w);
              }
            }
            const float r = 1.f / L;
#pragma unroll
            for (int i = 0; i < C; i += 2) {
              uint4 y;
              y.x = Act<T>::pack2(acc[i].x * r, acc[i].y * r);
              y.y = Act<T>::pack2(acc[i].z * r, acc[i].w * r);
              y.z = Act<T>::pack2(acc[i + 1].x * r, acc[i + 1].y * r);
              y.w = Act<T>::pack2(acc[i + 1].z * r, acc[i + 1].w * r);
              *chunk_at(k - x * 128, (c0 + i) / 2) = y;
            }
          }
          flush();
        }
      }
    }
    if (!ok) *abort_v = 1;
  } else {
    ck_fewer_regs<kFew>();
    if constexpr (Q4) {
    // ---------------- 4 bits: codes to f16 operand tiles ----------------
    const int cw = warp - 12;
    int s = 0, ph = 0, b = 0, round_b = 0;
    bool ok = true;
    const uint32_t f64 = p.f64, k72 = 0x54805480u;  // f16 64, 72
    CkWork w;
    for (int k; ok && (k = ck_next(p, c, plan, range, it, w)) >= 0;) {
      if (k == 0) continue;
      const int top = w.count[1] > 0 ? w.hi[1] : w.hi[0];
      for (int j = w.j0; j < w.j1; ++j) {
        const int k0 = w.tile(j) * kPageTokens;
        if (!ck_wait(&kv_full[s], ph, abort_v) ||
            (round_b > 0 && !ck_wait(&cv_empty[0][b], (round_b - 1) & 1, abort_v))) {
          ok = false;
          break;
        }
        const uint8_t* src = kvp + s * 2 * BLK;
        uint8_t* dst = cvp + b * CVB;
        const bool bad = bad_s[s];
        if (tid == 12 * 32) cbad_s[(round_b * 2 + b) & 3] = bad;
        // 8 keys a pass of a warp; a lane takes chunk lane & 3 of a key, keys 4 apart in a
        // quarter-warp, whose swizzled rows share no banks
        constexpr int PASS = 8 / kCkConv;
        const int kk = lane >> 2, ch = lane & 3;
        auto key_of = [&](int ps) { return (cw + ps * kCkConv) * 8 + (kk & 1) * 4 + (kk >> 1); };
        constexpr int CB = 64 * D / 2;  // code bytes of a block
#pragma unroll
        for (int ps = 0; ps < PASS; ++ps) {
          const int key = key_of(ps);
          // a key chunk: word g holds dims 32 g + 8 ch .. + 7
          uint32_t wd[NB], d2[NB];
          if constexpr (NB == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(src + key * 64 + ch * 16);
            const uint2 sc = *reinterpret_cast<const uint2*>(src + CB + key * 8);
            wd[0] = u.x, wd[1] = u.y, wd[2] = u.z, wd[3] = u.w;
            d2[0] = __byte_perm(sc.x, 0, 0x1010), d2[1] = __byte_perm(sc.x, 0, 0x3232);
            d2[2] = __byte_perm(sc.y, 0, 0x1010), d2[3] = __byte_perm(sc.y, 0, 0x3232);
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src + key * 32 + ch * 8);
            const uint32_t sc = *reinterpret_cast<const uint32_t*>(src + CB + key * 4);
            wd[0] = u.x, wd[1] = u.y;
            d2[0] = __byte_perm(sc, 0, 0x1010), d2[1] = __byte_perm(sc, 0, 0x3232);
          }
#pragma unroll
          for (int g = 0; g < NB; ++g) {
            uint4 o;
            o.x = ck_sub_mul(((wd[g] << 4) & 0x00f000f0u) | f64, k72, d2[g]);
            o.y = ck_sub_mul((wd[g] & 0x00f000f0u) | f64, k72, d2[g]);
            o.z = ck_sub_mul(((wd[g] >> 4) & 0x00f000f0u) | f64, k72, d2[g]);
            o.w = ck_sub_mul(((wd[g] >> 8) & 0x00f000f0u) | f64, k72, d2[g]);
            const int oc = 4 * g + ch;
            *reinterpret_cast<uint4*>(dst + (oc >> 3) * kCkBox + key * 128 + (((oc & 7) ^ (key & 7)) << 4)) = o;
          }
        }
        ck_fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&cv_full[0][b]);
        // a value chunk: its words are dims in order
        uint32_t wd[PASS][NB], dv[PASS];
#pragma unroll
        for (int ps = 0; ps < PASS; ++ps) {
          const int key = key_of(ps);
          if constexpr (NB == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(src + BLK + key * 64 + ch * 16);
            wd[ps][0] = u.x, wd[ps][1] = u.y, wd[ps][2] = u.z, wd[ps][3] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src + BLK + key * 32 + ch * 8);
            wd[ps][0] = u.x, wd[ps][1] = u.y;
          }
          dv[ps] = *reinterpret_cast<const uint16_t*>(src + BLK + CB + key * NB * 2 + (NB == 4 ? ch : ch >> 1) * 2);
          const int kp = k0 + key;
          const bool hide = bad || kp > top || (W && kp <= w.lo[0] - W && kp >= S);
          dv[ps] = hide ? 0u : dv[ps] | dv[ps] << 16;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_empty[s]);  // this warp has read its part of the stage
        if (round_b > 0 && !ck_wait(&cv_empty[1][b], (round_b - 1) & 1, abort_v)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int ps = 0; ps < PASS; ++ps) {
          const int key = key_of(ps);
#pragma unroll
          for (int g = 0; g < NB; ++g) {
            // nibbles 2 i, 2 i + 1 side by side: bytes of the even and the odd ones interleaved
            const uint32_t ev = (wd[ps][g] << 4) & 0xf0f0f0f0u, od = wd[ps][g] & 0xf0f0f0f0u;
            const uint32_t c4[4] = {__byte_perm(ev, od, 0x0400), __byte_perm(ev, od, 0x0501), __byte_perm(ev, od, 0x0602),
                                    __byte_perm(ev, od, 0x0703)};
            uint32_t o[4], rest[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[i] = ck_sub_mul((c4[i] & 0x00ff00ffu) | f64, k72, dv[ps]);
              if constexpr (kFine) rest[i] = ck_sub_mul_rest((c4[i] & 0x00ff00ffu) | f64, k72, dv[ps], o[i]);
            }
            const int oc = NB * ch + g;
            uint8_t* at = dst + TB + (oc >> 3) * kCkBox + key * 128 + (((oc & 7) ^ (key & 7)) << 4);
            *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
            if constexpr (kFine) *reinterpret_cast<uint4*>(at + TB) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
          }
        }
        ck_fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&cv_full[1][b]);
        if (++s == stages) s = 0, ph ^= 1;
        if (++b == 2) b = 0, ++round_b;
      }
    }
    if (!ok) *abort_v = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_s) report_timeout(status, kSiteCacheChunk);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct CkShape {
  int tiles, split, stages, smem;
};

CkShape ck_shape(bool bf16, const CacheView& c, int n_heads, int n_seqs, int max_rows) {
  CkShape s;
  const long long pairs = (long long)max_rows * (n_heads / c.kv_heads);
  s.tiles = (int)((pairs + 255) / 256);
  const long long entries = (long long)s.tiles * n_seqs;
  s.split = entries <= kCkEntries && entries * c.kv_heads <= FMD_CACHE_WORKSPACE_ZERO / 4 &&
            entries * cache_units(c) <= INT_MAX;
  const bool q4 = c.format == FMD_CACHE_Q4;
  const int tb = 64 * c.head_dim * 2, stage = 2 * (int)c.block_bytes();
  s.stages = 4;
  s.smem = 1024 + 2 * 128 * c.head_dim * 2 + s.stages * stage + (q4 ? 2 * (bf16 ? 2 : 3) * tb : 0);
  return s;
}

constexpr int kCkGrid = 148;

}  // namespace

// counters, then the partials of cut items (of smaller calls, where this size is not split)
size_t cache_chunk_workspace(const CacheView& c) {
  return FMD_CACHE_WORKSPACE_ZERO + (size_t)2 * kCkGrid * 256 * (c.head_dim + 2) * 4;
}

cudaError_t launch_cache_chunk(bool bf16, const CacheView& c, int layer, const CacheRows& r, const CacheAttend& a,
                               void* workspace, int* status, cudaStream_t s) {
  const bool q4 = c.format == FMD_CACHE_Q4;
  // no sequence has more rows than the buffers, and every (sequence, tile) is looked at
  const CkShape sh = ck_shape(bf16, c, a.n_heads, r.n_seqs, std::min(a.max_rows, r.n_rows));
  CUtensorMap map{};
  if (!q4 && !cache_tensor_map(&map, c, layer)) return cudaErrorNotSupported;
  CkArgs p;
  p.r = r;
  p.a = a;
  p.counters = (int*)workspace;
  p.part = (float*)((uint8_t*)workspace + FMD_CACHE_WORKSPACE_ZERO);
  p.tiles = sh.tiles;
  p.split = sh.split;
  p.stages = sh.stages;
  p.f64 = 0x54005400u;
  auto go = [&](auto kern) -> cudaError_t {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, sh.smem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCkGrid);
    cfg.blockDim = dim3(ck_threads(q4));
    cfg.dynamicSmemBytes = sh.smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, map, c, layer, p, status);
  };
  auto by_d = [&](auto t, auto f) {
    using T = decltype(t);
    constexpr bool F = decltype(f)::value;
    return c.head_dim == 128 ? go(k_cache_chunk<T, 128, F>) : go(k_cache_chunk<T, 64, F>);
  };
  auto by_f = [&](auto t) { return q4 ? by_d(t, std::true_type{}) : by_d(t, std::false_type{}); };
  return bf16 ? by_f(__nv_bfloat16{}) : by_f(__half{});
}

}  // namespace fmd
