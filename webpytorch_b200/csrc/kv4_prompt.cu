// Attention of prompt chunks over the paged 4-bit cache on the 5th-generation tensor cores: requests with
// kPromptRows rows (query tokens x heads of a key/value head) or more of fp16 or bf16 queries, HD 64 or 128, in calls
// with enough of them. The other requests of a call are the streaming kernel's.
//
// A CTA takes two tiles of 128 rows of one request and key/value head and walks the positions they see
// in steps of 128:
//   S = Q K^T  (tcgen05, Q and K in shared memory)      softmax  P = 2^(coef S - m)
//   O = O + P V  (P from tensor memory, where it takes the place of S; V in shared memory)
// The softmax takes a step in two halves of 64 columns. As soon as it has written P of one, its product and
// then S of the same half of the next step are issued, which finish while it works on the other: it never
// waits for the tensor cores in the steady state. Warps 0 - 3 and
// 4 - 7 are the tiles' softmax, a thread a row; warps 8 - 11 decode keys and values, once for both tiles;
// warp 12 issues the MMAs. The running maximum moves only when it grows by more than 2^kLazy, and
// then the row's O in tensor memory is scaled.
// What the codes stand for is an fp16 number, so K and V are exact; probabilities are rounded to fp16's
// 11 bits (outputs have 11 or 8), and sums are fp32.
// Shared memory holds K and V as [position][element] with the 128-byte swizzle: K-major rows for S, and
// the same layout read as MN-major for P V. The order of a position's elements is free (the contraction of
// S; the columns of O), so it is the one in which a lane's 16-byte load of 32 codes gives four 16-byte
// stores without bank conflicts.
// Bound. 4 NH HD operations a visible (query, position): chunks of 900 and 2000 tokens over 6000 and 3340 positions (32
// heads over 4, HD 128, bf16) are 159 GFLOP, 95 us at the measured rate, and take 231 us, 685 TFLOP/s. A step of 128
// positions takes a CTA about 4200 clocks, of which the exponentials (16 a clock and SM) and the tensor work are 2048
// each: no pipe is full (tensor 38 %, XU 38 %, issue slots 45 %), and what warps wait for most is loads from tensor
// memory, two for each score. 13 warps leave a thread 128 registers, and at HD 128 some are spilled. 368 pairs of
// tiles over 148 SMs leave the last wave half empty.
#include <type_traits>

#include "kv4_common.cuh"
#include "kv4_attn.cuh"
#include "sm100_ptx.cuh"

namespace ql {

__device__ int g_kv4_prompt_status = 0;

namespace {

using namespace kv4;

constexpr int kTileRows = 128, kTiles = 2, kStep = 128, kHalf = kStep / 2;
constexpr int kSoftWarps = 8, kDecodeWarps = 4, kWarps = kSoftWarps + kDecodeWarps + 1, kThreads = kWarps * 32;
constexpr int kMostSplits = 16;                 // pieces of a pair's positions
constexpr int kRing = 3;                        // blocks of a decoding warp in flight

template <int HD, int G>
struct Smem {
  static constexpr int kPanel = 128 * 128;      // 128 rows of 128 bytes
  static constexpr int kTile = kPanel * HD / 64;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kTiles * kTile;
  static constexpr int kV = kK + 2 * kTile;
  static constexpr int kRaw = kV + 2 * kTile;
  static constexpr int kBar = kRaw + kDecodeWarps * kRing * block_bytes(HD, G);
  // s_full[2][2], p_full[2][2], k_full[2], v_full[2], k_free[2], v_free[2], pv_done[2], q_full, done, ring[4][3]
  static constexpr int kRingBar = 20;
  static constexpr int kBars = kRingBar + kDecodeWarps * kRing;
  static constexpr int kMisc = kBar + kBars * 8;
  static constexpr int kItem = kMisc + 16;
  static constexpr int kBytes = kItem + 32 + 1024;   // + alignment slack
};

// Chunk (16 bytes, one word of 8 codes) of a row: word w of the row is at panel, column.
template <int HD>
__device__ __forceinline__ constexpr int panel_of(int w) { return HD == 64 ? 0 : (w & 3) >> 1; }
template <int HD>
__device__ __forceinline__ constexpr int column_of(int w) { return HD == 64 ? w : 2 * (w >> 2) + (w & 1); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

constexpr float kLazy = 6.f, kPShift = 9.f;      // as in the streaming kernel

constexpr int kRows = kTiles * kTileRows;

// Pair of tiles `item` of `items`, tiles of the longest rows first: rows r0 .. r0 + nrows - 1 of request b and a
// key/value head. nrows is 0 for one past a request's last row, or of a request that is not the prompt kernel's.
struct Item {
  int b, kvh, q0, ql, r0, nrows;
};
__device__ __forceinline__ Item item_at(const AttnArgs& a, int grp, int item, int items) {
  Item it;
  it.kvh = item % a.NKV;
  const int x = items / a.NKV - 1 - item / a.NKV;
  const auto tile_start = [&](int b) { return (int)((long)cu(a, b) * grp / kRows) + b; };
  it.b = 0;
  for (int hi = a.B - 1; it.b < hi;) {            // the last request whose first pair of tiles is at or before x
    const int mid = (it.b + hi + 1) >> 1;
    if (tile_start(mid) <= x) it.b = mid;
    else hi = mid - 1;
  }
  it.q0 = cu(a, it.b);
  it.ql = max(cu(a, it.b + 1) - it.q0, 0);
  const int rows = it.ql * grp;
  it.r0 = (x - tile_start(it.b)) * kRows;
  it.nrows = rows < a.prompt_rows || it.r0 >= rows ? 0 : min(kRows, rows - it.r0);
  return it;
}

// The rare paths of the kernel are functions that are called and find the row again, so that they take no registers
// from it: positions lo .. hi - 1 that row i of a pair of tiles sees, and those that all of its rows see.
struct Sight {
  int lo, hi, common_lo, common_hi;
};
__device__ __forceinline__ Sight sight_of(const AttnArgs& a, const Item& it, int i) {
  const int grp = a.NH / a.NKV, p0 = max(a.seq_lens[it.b], 0) - it.ql;
  const auto lo = [&](int p) { return a.window ? max(p - a.window + 1, 0) : 0; };
  const int pos = p0 + (it.r0 + min(i, it.nrows - 1)) / grp;
  return {lo(pos), min(pos + 1, a.width << a.page_shift), lo(p0 + (it.r0 + it.nrows - 1) / grp), p0 + it.r0 / grp + 1};
}

// Whether row i sees a page that is not the cache's.
__device__ __noinline__ bool sees_bad_page(const AttnArgs& a, const Item& it, int i) {
  const Sight see = sight_of(a, it, i);
  bool bad = false;
  for (int p = see.lo >> a.page_shift; p <= (see.hi - 1) >> a.page_shift; ++p)
    bad = bad || (unsigned)a.table[it.b * a.table_stride + p] >= (unsigned)a.num_pages;
  return bad;
}

// 32 codes of a position, words 4 t .. 4 t + 3 of row `row`, into a tile of keys or values. FINITE: values that are not
// count as zero.
template <int HD, bool FINITE>
__device__ __forceinline__ void decode_words(unsigned char* to, int row, int t, uint4 u, __half2 sm) {
  const __half2 s2 = __low2half2(sm), m2 = __high2half2(sm);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 h[4];
    codes_h2(w[i], h);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      h[q] = __hfma2(h[q], s2, m2);
      if (FINITE) h[q] = finite_or_zero(h[q]);
    }
    const int word = 4 * t + i;
    *reinterpret_cast<uint4*>(to + panel_of<HD>(word) * (128 * 128) + row * 128 + ((column_of<HD>(word) ^ (row & 7)) << 4)) =
        make_uint4(h2_as_u32(h[0]), h2_as_u32(h[1]), h2_as_u32(h[2]), h2_as_u32(h[3]));
  }
}
template <int HD>
__device__ __noinline__ void decode_finite(unsigned char* to, int row, int t, uint4 u, __half2 sm) {
  decode_words<HD, true>(to, row, t, u, sm);
}

// Columns 32 k .. of row i's output in tensor-memory order: 0 x, which is nan for values that are not finite and 0 for all
// others, is added for the positions that the row sees, but for those that all rows see, whose values were taken as they
// are.
template <int HD, int G>
__device__ __noinline__ void add_odd_values(const AttnArgs& a, const Item& it, int i, int k, uint32_t (&v)[32]) {
  const Sight see = sight_of(a, it, i);
#pragma unroll 1
  for (int p = see.lo; p < see.hi; ++p) {
    if (p >= see.common_lo && p < see.common_hi) continue;
    const uint32_t src = source(a, it.b, it.kvh, p >> 4, 0, 1);
    if (src == kNoBlock) continue;
    const uint8_t* vc = a.cache + (size_t)src * block_bytes(HD, G) + code_bytes(HD) + scale_bytes(HD, G);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int pc = 4 * k + c, w = HD == 64 ? pc : 4 * ((pc & 7) >> 1) + 2 * (pc >> 3) + (pc & 1);
      const __half2 sm = reinterpret_cast<const __half2*>(vc + code_bytes(HD))[(p & 15) * (HD / G) + 8 * w / G];
      __half2 n[4];
      codes_h2(*reinterpret_cast<const uint32_t*>(vc + (p & 15) * (HD / 2) + 4 * w), n);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 x = __half22float2(__hfma2(n[q], __low2half2(sm), __high2half2(sm)));
        v[8 * c + 2 * q] = __float_as_uint(fmaf(0.f, x.x, __uint_as_float(v[8 * c + 2 * q])));
        v[8 * c + 2 * q + 1] = __float_as_uint(fmaf(0.f, x.y, __uint_as_float(v[8 * c + 2 * q + 1])));
      }
    }
  }
}

// A row's running maximum (units of log2) and sum.
struct Row {
  float m, l;
};

// Half a step of a row: S in tensor memory to P over it. lo / hi: the positions that the row sees, relative to
// the half; product: the barrier and parity of the product before this one, which has to be complete before
// O is scaled; MASKED: they are not all of them for every row of the warp. The next 16 columns are loaded
// while the last are worked on.
template <int HD, bool MASKED>
__device__ __forceinline__ bool softmax_half(Row& row, uint32_t s_col, uint32_t o_col, float coef, bool first, int lo,
                                             int hi, uint32_t product, uint32_t parity, volatile int* abort_flag) {
  constexpr int NC = kHalf / 16;
  uint32_t v[2][16];
  float mx = -INFINITY;
  ptx::tmem_ld16(s_col, v[0]);
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    ptx::tmem_wait_ld();
    if (k + 1 < NC) ptx::tmem_ld16(s_col + 16u * (k + 1), v[(k + 1) & 1]);
    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int q = 0; q < 16; q += 2) {
      float x = __uint_as_float(v[k & 1][q]), y = __uint_as_float(v[k & 1][q + 1]);
      if (MASKED) {
        if (16 * k + q < lo || 16 * k + q >= hi) x = -INFINITY;
        if (16 * k + q + 1 < lo || 16 * k + q + 1 >= hi) y = -INFINITY;
      }
      m2[(q >> 1) & 1] = fmaxf(m2[(q >> 1) & 1], fmaxf(x, y));
    }
    mx = fmaxf(mx, fmaxf(m2[0], m2[1]));
  }
  const float mn = MASKED && mx == -INFINITY ? -INFINITY : mx * coef;   // coef may be 0
  if (__any_sync(0xffffffffu, mn > row.m + kLazy)) {
    const float top = fmaxf(row.m, mn), f = top > row.m ? ex2(row.m - top) : 1.f;
    row.m = top;
    row.l *= f;
    if (!first) {
      if (!warp_wait(product, parity, abort_flag)) return false;
      ptx::tc_fence_after();
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t o[16];
        ptx::tmem_ld16(o_col + 16u * k, o);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
        ptx::tmem_st16(o_col + 16u * k, o);
      }
    }
  }
  const float base = kPShift - (MASKED && row.m == -INFINITY ? 0.f : row.m);
  const float2 coef2 = make_float2(coef, coef), base2 = make_float2(base, base);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  ptx::tmem_ld16(s_col, v[0]);
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    ptx::tmem_wait_ld();
    if (k + 1 < NC) ptx::tmem_ld16(s_col + 16u * (k + 1), v[(k + 1) & 1]);
    uint32_t h[8];
#pragma unroll
    for (int q = 0; q < 16; q += 2) {
      float2 e = fma2(make_float2(__uint_as_float(v[k & 1][q]), __uint_as_float(v[k & 1][q + 1])), coef2, base2);
      e = make_float2(ex2(e.x), ex2(e.y));
      if (MASKED) {
        if (16 * k + q < lo || 16 * k + q >= hi) e.x = 0.f;
        if (16 * k + q + 1 < lo || 16 * k + q + 1 >= hi) e.y = 0.f;
      }
      sum[(q >> 1) & 1] = add2(sum[(q >> 1) & 1], e);
      h[q / 2] = h2_as_u32(__floats2half2_rn(e.x, e.y));
    }
    ptx::tmem_st8(s_col + 8u * k, h);
  }
  sum[0] = add2(sum[0], sum[1]);
  row.l += sum[0].x + sum[0].y;
  ptx::tmem_wait_st();
  return true;
}

// A part of a pair of tiles: HD / 4 x kRows fours of O (a row's four to a lane, so that lanes store and load next
// to each other), then (m, l) of the rows.
template <int HD>
constexpr int part_floats() { return kRows * (HD + 2); }
template <int HD>
__device__ __forceinline__ float* part_of(const AttnArgs& a, int split, int item, int items) {
  return a.parts + ((long)split * items + item) * part_floats<HD>();
}

// CUT: where a call has at most half as many pairs of tiles as the GPU has SMs, the positions of a pair are cut
// into gridDim.y equal pieces, and prompt_join_kernel adds up what they leave. (256 tokens over 6000 positions, 32
// heads over 4: 119 us whole, 49 cut; 64 tokens 117 and 36. One kernel for both was 2 % slower on large calls.)
template <int DT, int HD, int G, bool CUT>
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const __grid_constant__ AttnArgs a) {
  using L = Smem<HD, G>;
  constexpr int BB = block_bytes(HD, G), W = HD / 8;
  const int grp = a.NH / a.NKV;
  const Item item = item_at(a, grp, blockIdx.x, gridDim.x);
  if (item.nrows == 0) return;
  const int b = item.b, kvh = item.kvh, q0 = item.q0, ql = item.ql, r0 = item.r0, nrows = item.nrows;
  const int seq = max(a.seq_lens[b], 0), table_end = a.width << a.page_shift;
  const int p_first = seq - ql + r0 / grp, p_last = seq - ql + (r0 + nrows - 1) / grp;
  const int lo_all = a.window ? max(p_first - a.window + 1, 0) : 0, hi_all = min(p_last + 1, table_end);
  constexpr int kStepBlocks = kStep / kBlock;
  const int blk_lo = lo_all / kBlock, blk_all = max((hi_all + kBlock - 1) / kBlock - blk_lo, 0);
  const int all_steps = (blk_all + kStepBlocks - 1) / kStepBlocks;
  const int each = CUT ? (all_steps + gridDim.y - 1) / gridDim.y : all_steps;
  const int first_step = CUT ? min((int)blockIdx.y * each, all_steps) : 0, steps = min(each, all_steps - first_step);
  const int blk0 = blk_lo + first_step * kStepBlocks;
  const int nblk = CUT ? min(blk_all - first_step * kStepBlocks, steps * kStepBlocks) : blk_all;

  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = ptx::smem_addr(smem), bar0 = sbase + L::kBar;
  const auto s_full = [&](int i, int h) { return bar0 + 8u * (2 * i + h); };
  const auto p_full = [&](int i, int h) { return bar0 + 8u * (4 + 2 * i + h); };
  const auto k_full = [&](int s) { return bar0 + 8u * (8 + s); };
  const auto v_full = [&](int s) { return bar0 + 8u * (10 + s); };
  const auto k_free = [&](int s) { return bar0 + 8u * (12 + s); };
  const auto v_free = [&](int s) { return bar0 + 8u * (14 + s); };
  const auto pv_done = [&](int i) { return bar0 + 8u * (16 + i); };
  const uint32_t q_full = bar0 + 8u * 18, done = bar0 + 8u * 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 8);
  volatile int* odd_flag = reinterpret_cast<volatile int*>(smem + L::kMisc + 12);
  Item* kept_item = reinterpret_cast<Item*>(smem + L::kItem);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // uniform
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      for (int h = 0; h < 2; ++h) {
        ptx::mbar_init(s_full(i, h), 1);
        ptx::mbar_init(p_full(i, h), 4);
      }
      ptx::mbar_init(pv_done(i), 1);
      ptx::mbar_init(k_full(i), kDecodeWarps);
      ptx::mbar_init(v_full(i), kDecodeWarps);
      ptx::mbar_init(k_free(i), 1);
      ptx::mbar_init(v_free(i), 1);
    }
    ptx::mbar_init(q_full, kSoftWarps);
    ptx::mbar_init(done, 1);
    for (int i = 0; i < kDecodeWarps * kRing; ++i) ptx::mbar_init(bar0 + 8u * (L::kRingBar + i), 1);
    *abort_flag = 0;
    *bad_flag = 0;
    *odd_flag = 0;
    *kept_item = item;
    ptx::fence_mbar_init();
  }
  if (warp == kWarps - 1) {
    ptx::tmem_alloc(ptx::smem_addr(tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);   // known to be the same for all lanes
  // tensor memory of tile i: S (and P over it) at tmem + 256 i, O 128 columns on

  if (warp < kSoftWarps) {
    // ---------------- softmax: a thread a row
    const int tile = warp >> 2, row = (warp & 3) * 32 + lane, i = tile * kTileRows + row;
    const bool live = i < nrows;
    const int mine = r0 + min(i, nrows - 1);      // rows past the last repeat it and are not written
    const int tok = q0 + mine / grp, head = kvh * grp + mine % grp;
    float coef;
    {
      uint32_t raw[HD / 2];
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.q) + (long)tok * a.ldq + (long)head * HD);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const uint4 u = p[k];
        raw[4 * k] = u.x; raw[4 * k + 1] = u.y; raw[4 * k + 2] = u.z; raw[4 * k + 3] = u.w;
      }
      const auto element = [&](int k) -> float {
        const uint32_t u = raw[k / 2];
        if (DT == QL_F16) return k & 1 ? __high2float(u32_as_h2(u)) : __low2float(u32_as_h2(u));
        return __int_as_float(k & 1 ? u & 0xffff0000u : u << 16);
      };
      float mx = 0.f;
#pragma unroll
      for (int k = 0; k < HD; ++k) mx = fmaxf(mx, fabsf(element(k)));
      const int e = stage_exponent(mx);
      const float inv = copysignf(exp2i(-e), a.scale);
      coef = exp2i(e) * (fabsf(a.scale) * 1.4426950408889634f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t h[4];                            // the order that the nibble masks give: (j, j + 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = h2_as_u32(__floats2half2_rn(element(8 * w + j) * inv, element(8 * w + j + 4) * inv));
        *reinterpret_cast<uint4*>(smem + L::kQ + tile * L::kTile + panel_of<HD>(w) * L::kPanel + row * 128 +
                                  ((column_of<HD>(w) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    ptx::fence_async_smem();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(q_full);
    const int pos = seq - ql + mine / grp;
    const int row_lo = a.window ? max(pos - a.window + 1, 0) : 0, row_hi = pos + 1;
    // steps where every row of the warp sees every position
    const int warp_lo = __reduce_max_sync(0xffffffffu, row_lo), warp_hi = __reduce_min_sync(0xffffffffu, row_hi);
    const uint32_t s_col = tmem + 256u * tile + ((uint32_t)(warp & 3) << 21), o_col = s_col + 128u;
    Row run = {-INFINITY, 0.f};
    bool ok = true;
    volatile int* ab = const_cast<volatile int*>(abort_flag);
    for (int j = 0; ok && j < steps; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ok = warp_wait(s_full(tile, h), j & 1, ab);
        if (!ok) break;
        ptx::tc_fence_after();
        const int p0 = blk0 * kBlock + j * kStep + h * kHalf, n = 2 * j + h;
        const bool masked = p0 < warp_lo || p0 + kHalf > warp_hi;
        if (masked)
          ok = softmax_half<HD, true>(run, s_col + h * kHalf, o_col, coef, n == 0, row_lo - p0, row_hi - p0, pv_done(tile),
                                      (n & 1) ^ 1, ab);
        else
          ok = softmax_half<HD, false>(run, s_col + h * kHalf, o_col, coef, n == 0, 0, kHalf, pv_done(tile), (n & 1) ^ 1, ab);
        if (!ok) break;
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_full(tile, h));
        __syncwarp();
      }
    }
    if (steps > 0 && ok) ok = warp_wait(done, 0, ab);
    ptx::tc_fence_after();
    bool bad = !ok || seq > table_end;            // a length past the table: nan
    if (*bad_flag) bad = bad || sees_bad_page(a, *kept_item, i);
    if (bad) run.l = __int_as_float(0x7fc00000);
    const float inv = CUT ? 1.f : run.l == 0.f ? 0.f : 1.f / run.l;   // a row that sees nothing is zero
    float4* part = CUT ? reinterpret_cast<float4*>(part_of<HD>(a, blockIdx.y, blockIdx.x, gridDim.x)) : nullptr;
    if (CUT) reinterpret_cast<float2*>(part + HD / 4 * kRows)[i] = make_float2(run.m, run.l);
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + ((long)tok * a.NH + head) * HD;
    const bool odd = *odd_flag;
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) {
      uint32_t v[32];
      if (steps > 0) {
        ptx::tmem_ld32(o_col + 32u * k, v);
        ptx::tmem_wait_ld();
      }
      if (odd && steps > 0) {
        uint32_t x[32];                           // a copy that has an address
#pragma unroll
        for (int c = 0; c < 32; ++c) x[c] = v[c];
        add_odd_values<HD, G>(a, *kept_item, i, k, x);
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = x[c];
        __syncwarp();
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {               // columns 8 (4 k + c) ...: one word's elements
        const int pc = 4 * k + c, panel = pc >> 3, col = pc & 7;
        const int w = HD == 64 ? pc : 4 * (col >> 1) + 2 * panel + (col & 1);
        if constexpr (CUT) {
          if (steps > 0) {
            const auto f = [&](int e) { return __uint_as_float(v[8 * c + e]); };   // elements (0, 4), (1, 5), (2, 6), (3, 7)
            part[(2 * w) * kRows + i] = make_float4(f(0), f(2), f(4), f(6));
            part[(2 * w + 1) * kRows + i] = make_float4(f(1), f(3), f(5), f(7));
          }
        } else {
          uint32_t o[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // element e of the word is at 2 e, elements 4 + e at 2 e + 1
            const int e0 = 2 * q, e1 = 2 * q + 1;
            const float y0 = steps > 0 ? __uint_as_float(v[8 * c + (e0 < 4 ? 2 * e0 : 2 * (e0 - 4) + 1)]) * inv : 0.f * inv;
            const float y1 = steps > 0 ? __uint_as_float(v[8 * c + (e1 < 4 ? 2 * e1 : 2 * (e1 - 4) + 1)]) * inv : 0.f * inv;
            if (DT == QL_F16) {
              o[q] = h2_as_u32(__floats2half2_rn(y0, y1));
            } else {
              const __nv_bfloat162 t = __floats2bfloat162_rn(y0, y1);
              o[q] = *reinterpret_cast<const uint32_t*>(&t);
            }
          }
          if (live) {
            uint2* to = reinterpret_cast<uint2*>(out + 8 * w);
            to[0] = make_uint2(o[0], o[1]);
            to[1] = make_uint2(o[2], o[3]);
          }
        }
      }
    }
  } else if (warp < kSoftWarps + kDecodeWarps) {
    // ---------------- keys and values: warp d decodes blocks d, d + 4 of each step's 8
    const int d = warp - kSoftWarps;
    const uint32_t ring = sbase + L::kRaw + d * kRing * BB, bar = bar0 + 8u * (L::kRingBar + d * kRing);
    const unsigned char* raw = smem + L::kRaw + d * kRing * BB;
    constexpr int LP = HD / 32, PW = 32 / LP;     // lanes of a position, positions of a pass
    const int t = lane % LP, pr = lane / LP;
    const int common_lo = a.window ? max(p_last - a.window + 1, 0) : 0;   // all rows see common_lo .. p_first
    // the warp's blocks in order: n-th is block d + 4 n of the item. Lane i looks up block i of the next 32.
    const int mine = nblk > d ? (nblk - d + 3) / 4 : 0;
    const auto lookup = [&](int n) { return n < mine ? source(a, b, kvh, blk0, d + 4 * n, nblk) : kNoBlock; };
    uint32_t src = lookup(lane), next = kNoBlock;
    int issued = 0;
    const auto issue_one = [&](int ahead_of) {     // block `issued`, whose lookup is in src or next
      if (issued < mine && (issued & 31) == lane) {
        const uint32_t at = (issued ^ ahead_of) & 32 ? next : src;
        const int s = issued % kRing;
        issue<BB>(a, at, s, ring, bar);
      }
      ++issued;
    };
    for (int k = 0; k < kRing; ++k) issue_one(0);
    uint32_t missing = __ballot_sync(0xffffffffu, src == kNoBlock);
    bool ok = true;
    int n = 0;                                    // blocks decoded
    for (int j = 0; ok && j < steps; ++j) {
      const int st = j & 1, par = (j >> 1) & 1;
      // both of this step's blocks arrive, keys first
#pragma unroll
      for (int kv = 0; kv < 2 && ok; ++kv) {
        if (!warp_wait<true>(kv ? v_free(st) : k_free(st), par ^ 1, const_cast<volatile int*>(abort_flag))) {
          ok = false;
          break;
        }
        unsigned char* to = smem + (kv ? L::kV : L::kK) + st * L::kTile;
        for (int half = 0; half < 2; ++half) {
          const int bn = 2 * j + half;             // this warp's block, d + 4 bn of the item
          bool have = bn < mine;
          if (have && kv == 0) {
            if ((bn & 31) == 0) {
              if (bn > 0) {
                src = next;
                missing = __ballot_sync(0xffffffffu, src == kNoBlock);
              }
              next = lookup(bn + 32 + lane);
            }
            if (!warp_wait(bar + 8 * (bn % kRing), (bn / kRing) & 1, const_cast<volatile int*>(abort_flag))) {
              ok = false;
              break;
            }
          }
          if (have && ((missing >> (bn & 31)) & 1)) {
            have = false;
            if (lane == 0) *bad_flag = 1;          // a page that is not one of the cache's
          }
          const unsigned char* blk = raw + (bn % kRing) * BB + (kv ? code_bytes(HD) + scale_bytes(HD, G) : 0);
          // values that some row does not see: its p = 0 would make nan of one that is not finite
          const int start = (blk0 + 8 * j + d + 4 * half) * kBlock;
          const bool edge = kv == 1 && (start + kBlock - 1 > p_first || start < common_lo);
          // a loop for each, since the check within one takes the large calls from 301 to 311 us
          const auto passes = [&](auto at_edge) {
#pragma unroll
            for (int pass = 0; pass < kBlock / PW; ++pass) {
              const int p = pass * PW + pr, at = (2 * 4 * j + d + 4 * half) * kBlock + p;   // in the block, in the item
              const int row = (d + 4 * half) * kBlock + p;
              const int seen = blk0 * kBlock + at;
              uint4 u = make_uint4(0u, 0u, 0u, 0u);
              __half2 sm = h2_const(0u);
              // positions that no row sees are zero: their memory may never have been written
              if (have && seen >= lo_all && seen < hi_all) {
                u = *reinterpret_cast<const uint4*>(blk + p * (HD / 2) + t * 16);
                sm = reinterpret_cast<const __half2*>(blk + code_bytes(HD))[p * (HD / G) + t * 32 / G];
              }
              if (decltype(at_edge)::value && (seen > p_first || seen < common_lo) && may_not_be_finite(sm)) {
                *odd_flag = 1;
                decode_finite<HD>(to, row, t, u, sm);
              } else {
                decode_words<HD, false>(to, row, t, u, sm);
              }
            }
          };
          if (edge) passes(std::true_type());
          else passes(std::false_type());
          if (kv == 1 && bn < mine) {              // the block's values were its last part
            __syncwarp();
            ++n;
            issue_one(bn);
          }
        }
        if (!ok) break;                            // what was not decoded is not handed on
        ptx::fence_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(kv ? v_full(st) : k_full(st));
      }
    }
    if (!ok)                                       // no copy is left in flight
      for (int k = n; k < min(issued, mine); ++k) ptx::mbar_wait_drain(bar + 8 * (k % kRing), (k / kRing) & 1);
  } else if (steps > 0) {
    // ---------------- MMA issue: the warp runs converged, one lane issues, and what the MMAs take is the same
    // for all lanes by construction, which keeps descriptors in uniform registers (an MMA takes about 110 cycles to
    // issue without, against 64 of tensor work)
    constexpr uint32_t kIdescS = ptx::idesc_f16_f32(128, kHalf);
    constexpr uint32_t kIdescO = ptx::idesc_f16_f32(128, HD) | ptx::kIdescBMn;
    volatile int* ab = const_cast<volatile int*>(abort_flag);
    const uint64_t q_desc = ptx::smem_desc_sw128(sbase + L::kQ), k_desc = ptx::smem_desc_sw128(sbase + L::kK);
    const uint64_t v_desc = ptx::smem_desc_mn_sw128(sbase + L::kV, L::kPanel);
    const bool elected = ptx::elect_one();
    const auto scores = [&](int i, int h, int st) {
      const uint64_t qd = q_desc + (uint32_t)(i * (L::kTile >> 4));
      const uint64_t kd = k_desc + (uint32_t)((st * L::kTile + h * kHalf * 128) >> 4);
      if (elected) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t at = ((k >> 2) * L::kPanel + (k & 3) * 32) >> 4;
          ptx::mma_f16_ss(tmem + 256u * i + (uint32_t)(h * kHalf), qd + at, kd + at, kIdescS, k > 0);
        }
        ptx::mma_commit(s_full(i, h));
      }
      __syncwarp();
    };
    bool ok = warp_wait(q_full, 0, ab) && warp_wait(k_full(0), 0, ab);
    ptx::tc_fence_after();
    if (ok) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        scores(0, h, 0);
        scores(1, h, 0);
      }
      if (elected) ptx::mma_commit(k_free(0));
    }
    for (int j = 0; ok && j < steps; ++j) {
      const int st = j & 1, par = (j >> 1) & 1, st1 = st ^ 1, par1 = ((j + 1) >> 1) & 1;
#pragma unroll
      for (int hi = 0; hi < 2 * kTiles; ++hi) {
        const int h = hi >> 1, i = hi & 1;
        ok = warp_wait(p_full(i, h), j & 1, ab);
        if (hi == 0) ok = ok && warp_wait(v_full(st), par, ab) && (j + 1 == steps || warp_wait(k_full(st1), par1, ab));
        if (!ok) break;
        ptx::tc_fence_after();
        const uint64_t vd = v_desc + (uint32_t)((st * L::kTile + h * kHalf * 128) >> 4);
        if (elected) {
#pragma unroll
          for (int k = 0; k < kHalf / 16; ++k)
            ptx::mma_f16_ts_elected(tmem + 256u * i + 128u, tmem + 256u * i + (uint32_t)(h * kHalf) + 8u * k,
                                    vd + (uint32_t)(k * (2048 >> 4)), kIdescO, h > 0 || k > 0 || j > 0);
          ptx::mma_commit(pv_done(i));
        }
        __syncwarp();
        if (j + 1 < steps) scores(i, h, st1);
      }
      if (!ok) break;
      if (elected) {
        ptx::mma_commit(v_free(st));
        if (j + 1 < steps) ptx::mma_commit(k_free(st1));
      }
      __syncwarp();
    }
    // everything issued has completed before tensor memory is read for the output or released. One lane polls, and
    // the warp comes together before the end, which releases tensor memory once.
    if (elected) {
      ptx::mma_commit(done);
      ptx::mbar_wait_drain(done, 0);
    }
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_kv4_prompt_status, 1);
  __syncwarp();
  if (warp == kWarps - 1) ptx::tmem_dealloc(tmem, 512);
}

// Rows of pairs of tiles whose positions were cut: O = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s, in the order of
// the pieces. A thread has 32 elements of a row.
template <int DT, int HD>
__global__ void __launch_bounds__(kRows) prompt_join_kernel(AttnArgs a, int splits) {
  const int grp = a.NH / a.NKV, i = threadIdx.x;
  const Item item = item_at(a, grp, blockIdx.x, gridDim.x);
  if (i >= item.nrows) return;
  const auto part = [&](int s) { return reinterpret_cast<const float4*>(part_of<HD>(a, s, blockIdx.x, gridDim.x)); };
  const auto stats = [&](int s) { return reinterpret_cast<const float2*>(part(s) + HD / 4 * kRows)[i]; };
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, stats(s).x);
  float4 acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {
    const float2 ml = stats(s);
    if (ml.x == -INFINITY) {                      // nothing seen, and O may not have been written; l is 0 or nan
      l += ml.y;
      continue;
    }
    const float f = ex2(ml.x - m);
    l = fmaf(f, ml.y, l);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float4 v = part(s)[(8 * blockIdx.y + c) * kRows + i];
      acc[c].x = fmaf(f, v.x, acc[c].x);
      acc[c].y = fmaf(f, v.y, acc[c].y);
      acc[c].z = fmaf(f, v.z, acc[c].z);
      acc[c].w = fmaf(f, v.w, acc[c].w);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;     // a row that sees nothing is zero
  const int row = item.r0 + i;
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) +
                  ((long)(item.q0 + row / grp) * a.NH + item.kvh * grp + row % grp) * HD + 32 * blockIdx.y;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint2 o;
    if (DT == QL_F16) {
      o = make_uint2(h2_as_u32(__floats2half2_rn(acc[c].x * inv, acc[c].y * inv)),
                     h2_as_u32(__floats2half2_rn(acc[c].z * inv, acc[c].w * inv)));
    } else {
      const __nv_bfloat162 x = __floats2bfloat162_rn(acc[c].x * inv, acc[c].y * inv);
      const __nv_bfloat162 y = __floats2bfloat162_rn(acc[c].z * inv, acc[c].w * inv);
      o = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
    reinterpret_cast<uint2*>(out)[c] = o;
  }
}

template <int DT, int HD, int G, bool CUT>
int launch_one(const AttnArgs& a, dim3 grid, cudaStream_t st) {
  auto kern = kv4_prompt_kernel<DT, HD, G, CUT>;
  static int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    const int rc = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD, G>::kBytes),
                               "cudaFuncSetAttribute(kv4 prompt smem)");
    if (rc) return rc;
    configured_dev = dev;
  }
  kern<<<grid, kThreads, Smem<HD, G>::kBytes, st>>>(a);
  return cuda_status(cudaGetLastError(), "ql_kv4_attention (prompt) launch");
}

template <int DT, int HD, int G>
int launch(const AttnArgs& a, int ctas, cudaStream_t st) {
  const long items = ((long)a.T * (a.NH / a.NKV) / kRows + a.B) * a.NKV;
  const int splits = (int)max(1L, min(ctas / items, (long)kMostSplits));
  if (splits == 1) return launch_one<DT, HD, G, false>(a, dim3((unsigned)items), st);
  const int rc = launch_one<DT, HD, G, true>(a, dim3((unsigned)items, splits), st);
  if (rc) return rc;
  prompt_join_kernel<DT, HD><<<dim3((unsigned)items, HD / 32), kRows, 0, st>>>(a, splits);
  return cuda_status(cudaGetLastError(), "ql_kv4_attention (prompt join) launch");
}

template <int DT>
int launch_sizes(const AttnArgs& a, int HD, int group, int ctas, cudaStream_t st) {
  if (HD == 64) return group == 32 ? launch<DT, 64, 32>(a, ctas, st) : launch<DT, 64, 64>(a, ctas, st);
  return group == 32   ? launch<DT, 128, 32>(a, ctas, st)
         : group == 64 ? launch<DT, 128, 64>(a, ctas, st)
                       : launch<DT, 128, 128>(a, ctas, st);
}

}  // namespace

size_t kv4_prompt_bytes(int HD, int ctas) {
  return (size_t)ctas * (HD == 64 ? part_floats<64>() : HD == 128 ? part_floats<128>() : 0) * sizeof(float);
}

int kv4_prompt_attention(const AttnArgs& a, int dtype, int HD, int group, int ctas, cudaStream_t st) {
  return dtype == QL_F16 ? launch_sizes<QL_F16>(a, HD, group, ctas, st) : launch_sizes<QL_BF16>(a, HD, group, ctas, st);
}

int take_kv4_prompt_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kv4_prompt_status, sizeof(int)) != cudaSuccess) return 0;
  if (v) cudaMemcpyToSymbol(g_kv4_prompt_status, &zero, sizeof(int));
  return v;
}

}  // namespace ql
