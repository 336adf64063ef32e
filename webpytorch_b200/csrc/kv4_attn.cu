// Attention over the paged 4-bit cache: softmax(q K^T scale) V for ragged requests, causal from the
// end of each request (query i of a request is at position seq_len - q_len + i), with an optional
// sliding window, for one query token or many.
//
// Rows. The query heads that share a key/value head and the request's query tokens form one list of
// rows, r = i (NH / NKV) + head; a tile takes the next rows of it. The warp MMA (m16n8k16, fp16 in,
// fp32 out) has 16 of them. One-plane tiles use them for 16 rows; two-plane tiles hold 8 rows as
// fp16 high and low parts (22 bits), rows r and r + 8 of the MMA, whose results the same thread
// holds and adds: queries and probabilities keep 22 bits. Tiles of 8 rows or fewer take as many MMAs as one plane
// would; of 16-bit queries, which one plane holds exactly, the low parts are zeros.
// Keys. A lane owns HD / 4 consecutive elements of a position (a 16-byte load at HD = 128), all in
// one group of at least 32 elements, so a scale pair is loaded once per position. The order of the
// contraction is free, so the pairs the nibble masks give (element j with j + 4 of a word) are the
// MMA's k pairs and the queries are laid out to match.
// Values. P V contracts over positions. The C fragment of S gives lane t of a quad positions t,
// t + 4, t + 8, t + 12 of the block (the key rows are read in the order that makes it so); the words
// of two positions are interleaved by one byte permutation per half, after which the same masks give
// pairs of positions. Codes become the exact fp16 values they stand for: one fma each.
// Work. A unit is one block of 16 positions of one (request, key/value head, tile); the units of all
// requests form one line that is cut into equal pieces, one for each warp of a grid of one CTA an SM,
// so lengths as different as they come load the GPU evenly and the host needs to know none of them.
// A warp streams its blocks through a ring of bulk copies (one 2304-byte record a block at HD = 128, G =
// 64), keeps the running maximum and sum of the tile, writes a tile that it holds whole, and leaves a part of
// a tile to be joined: first with the parts of the CTA's other warps, then, for at most two tiles a
// CTA, with those of other CTAs by whichever of them finishes last, always in the same order.
// Bound. A position is NKV (HD + 8 HD / G) bytes, and each of its 4-bit codes is unpacked once by one lane: about
// 13 instructions for 8 codes, of which 5 are the ALU pipe's. Long ragged batches run at 42 % of the measured copy
// rate, and no pipe is full over the whole call (ALU 46 %, tensor 32 %, issue slots 57 %); fixed latencies and busy
// pipes are what warps wait for most: 96 requests of 200 to 12000 positions (8 heads of 128, 303 MB) 110 us, 2.75 TB/s;
// 131071 positions of one request (4 heads, 71 MB) 43 us. Short calls are the fixed chain: launch and first loads 8 us,
// the join in a CTA 3, across CTAs 3 (513 positions 15 us).
#include "kv4_attn.cuh"

namespace ql {

// set when a bounded wait of this file's kernel gave up (read by ql_device_status)
__device__ int g_kv4_status = 0;

namespace {

using namespace kv4;

constexpr int kMaxCtas = 512;   // counters in the workspace
static_assert(kMaxCtas * sizeof(unsigned int) == QL_KV4_COUNTER_BYTES, "the part of the workspace that callers zero");
// Rows of a request from which the prompt kernel takes it: where the GPU is full, its tile pair costs
// what 2.3 of the streaming kernel's 16-row tiles do. 200 requests of 3000 positions, 32 heads over 4: 48 rows 382 us
// there, 360 here; 64 rows 415 and 449.
constexpr int kPromptRows = 64;

// Warps of a CTA by the registers that a head's state takes, and ring stages by what they leave.
template <int HD>
struct Shape {
  static constexpr int kWarps = HD == 64 ? 16 : HD == 128 ? 12 : 8;
  static constexpr int kStages = 4;               // two pairs of blocks
  static constexpr int kThreads = kWarps * 32;
};

// A part of a tile: output fragments (planes summed), then m and l of 16 rows.
template <int HD, int PL>
struct Part {
  static constexpr int kVec = 4 / PL;                         // floats of a lane and fragment
  static constexpr int kStats = HD / 8 * 32 * kVec;
  static constexpr int kFloats = kStats + 32;
};
template <int N>
struct Vec;
template <>
struct Vec<2> { using T = float2; };
template <>
struct Vec<4> { using T = float4; };

template <int HD, int G>
struct Smem {
  static constexpr int kRing = 0;
  static constexpr int kQ = kRing + Shape<HD>::kWarps * Shape<HD>::kStages * block_bytes(HD, G);
  static constexpr int kBar = kQ + Shape<HD>::kWarps * HD / 16 * 512;
  static constexpr int kBytes = kBar + Shape<HD>::kWarps * Shape<HD>::kStages * 8;
};

struct Request {
  int q0, ql, seq;       // first query row, queries, length
  int tiles, blo, nblk;  // row tiles; first block that any query sees, and blocks from there
};

template <int ROWS>
__device__ __forceinline__ Request load_request(const AttnArgs& a, int b) {
  Request r;
  r.q0 = cu(a, b);
  r.ql = max(cu(a, b + 1) - r.q0, 0);
  r.seq = max(a.seq_lens[b], 0);
  const int end = min(r.seq, a.width << a.page_shift);
  const int rows = r.ql * (a.NH / a.NKV);
  r.tiles = a.prompt_rows && rows >= a.prompt_rows ? 0 : (rows + ROWS - 1) / ROWS;
  r.blo = a.window ? max(r.seq - r.ql - a.window + 1, 0) / kBlock : 0;
  r.nblk = max((end + kBlock - 1) / kBlock - r.blo, 1);
  return r;
}

__device__ __forceinline__ long long units_of(const Request& r, int nkv) { return (long long)r.tiles * nkv * r.nblk; }

// Two floats as fp16 pairs of high and low parts, x = hi + lo to 22 bits.
__device__ __forceinline__ void split_h2(float x, float y, __half2& hi, __half2& lo) {
  hi = __floats2half2_rn(x, y);
  const float2 h = __half22float2(hi);
  lo = __floats2half2_rn(x - h.x, y - h.y);
}

// 2^x; results below 2^-126 are zero.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int HD, int PL>
struct State {
  float o[HD / 8][4];   // C fragments of the output, tile i: elements (2t, 2t + 1) * HD / 8 + i
  float m[3 - PL];      // running maximum of rows g (and g + 8), in units of log2
  float l[3 - PL];      // sum of exponentials: this lane's part, the row's after reduce_rows
};

// Queries of the tile's rows as A fragments in shared memory, and coef >= 0: coef S is the score in
// units of log2. Rows are scaled by a power of two into fp16's range, and by the scale's sign. start()
// runs while the loads are under way.
template <int DT, int HD, int PL, class F>
__device__ __forceinline__ void load_queries(const AttnArgs& a, const Request& r, int kvh, int r0, int nrows, int grp,
                                             uint4* qf, float (&coef)[3 - PL], const F& start) {
  constexpr int WV = DT == QL_F32 ? 8 : 4;       // words of 8 elements
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t raw[3 - PL][HD / 32 * WV];
#pragma unroll
  for (int k = 0; k < 3 - PL; ++k) {
    const int i = r0 + min(g + 8 * k, nrows - 1);   // rows past the tile repeat its last one
    const long at = (long)(r.q0 + i / grp) * a.ldq + (long)(kvh * grp + i % grp) * HD + t * (HD / 4);
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.q) + at * (DT == QL_F32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < HD / 32 * WV / 4; ++j) {
      const uint4 u = p[j];
      raw[k][4 * j] = u.x; raw[k][4 * j + 1] = u.y; raw[k][4 * j + 2] = u.z; raw[k][4 * j + 3] = u.w;
    }
  }
  start();
  const auto element = [&](int k, int i) -> float {
    if (DT == QL_F32) return __int_as_float(raw[k][i]);
    const uint32_t u = raw[k][i / 2];
    if (DT == QL_F16) return i & 1 ? __high2float(u32_as_h2(u)) : __low2float(u32_as_h2(u));
    return __int_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  };
  float inv[3 - PL];
#pragma unroll
  for (int k = 0; k < 3 - PL; ++k) {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) mx = fmaxf(mx, fabsf(element(k, i)));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int e = stage_exponent(mx);
    inv[k] = copysignf(exp2i(-e), a.scale);
    coef[k] = exp2i(e) * (fabsf(a.scale) * 1.4426950408889634f);
  }
#pragma unroll
  for (int w = 0; w < HD / 32; ++w)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // the pairs that the nibble masks of a key word give: (0, 4), (1, 5) | (2, 6), (3, 7); row g (its
      // high part) and row g + 8 (row g's low part)
      __half2 f[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = 8 * w + 2 * h + j;
        if (PL == 2) {
          split_h2(element(0, i) * inv[0], element(0, i + 4) * inv[0], f[0][j], f[1][j]);
        } else {
#pragma unroll
          for (int k = 0; k < 3 - PL; ++k)
            f[k][j] = __floats2half2_rn(element(k, i) * inv[k], element(k, i + 4) * inv[k]);
        }
      }
      qf[(2 * w + h) * 32 + lane] = make_uint4(h2_as_u32(f[0][0]), h2_as_u32(f[1][0]), h2_as_u32(f[0][1]), h2_as_u32(f[1][1]));
    }
}

// The running maximum is moved (and the sums with it) when it grows by more than 2^kLazy, not each
// time: p' stays within fp16 and the ratio o / l does not depend on it. At 80 blocks a warp a row's
// maximum grows in about a third of them.
constexpr float kLazy = 6.f;
constexpr float kPShift = 9.f;   // p' = 2^9 p, up to 2^15: 11 bits of probabilities down to 2^-23

// O += P V of a block's values vc, for P's fragment p; any_lo / any_hi: the positions of the block that some row sees. In a
// masked block values that are not finite are looked for first: where there are any, true is returned and nothing is
// added. ODD: they count as zero.
template <int HD, int G, bool MASKED, bool ODD>
__device__ __forceinline__ bool add_values(float (&o)[HD / 8][4], const uint32_t (&p)[4], const uint8_t* vc, int any_lo,
                                           int any_hi) {
  constexpr int VW = HD / 64;               // words of a lane and position
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const __half2* vs = reinterpret_cast<const __half2*>(vc + code_bytes(HD));
  // words of positions t, t + 4 | t + 8, t + 12, elements g HD / 8 ...
  uint32_t w[4][VW];
  __half2 s2[2], m2[2], sm[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint8_t* from = vc + (t + 4 * k) * (HD / 2) + g * (HD / 16);
    if constexpr (VW == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(from);
      w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
    } else if constexpr (VW == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(from);
      w[k][0] = u.x; w[k][1] = u.y;
    } else {
      w[k][0] = *reinterpret_cast<const uint32_t*>(from);
    }
    sm[k] = vs[(t + 4 * k) * (HD / G) + g * (HD / 8) / G];
  }
  if (MASKED) {
    bool odd = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (t + 4 * k < any_lo || t + 4 * k >= any_hi) sm[k] = h2_const(0u);
      odd = odd || may_not_be_finite(sm[k]);
    }
    if (!ODD && __any_sync(0xffffffffu, odd)) return true;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    s2[k] = __lows2half2(sm[2 * k], sm[2 * k + 1]);
    m2[k] = __highs2half2(sm[2 * k], sm[2 * k + 1]);
  }
#pragma unroll
  for (int i = 0; i < VW; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t sel = h ? 0x7632u : 0x5410u;
      __half2 b0[4], b1[4];
      // nibbles 0..3 of the half words of two positions: codes_h2 reads the interleaved word as
      // (nibble j of one, nibble j of the other)
      codes_h2(__byte_perm(w[0][i], w[1][i], sel), b0);
      codes_h2(__byte_perm(w[2][i], w[3][i], sel), b1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        b0[k] = __hfma2(b0[k], s2[0], m2[0]);
        b1[k] = __hfma2(b1[k], s2[1], m2[1]);
        if (ODD) {
          b0[k] = finite_or_zero(b0[k]);
          b1[k] = finite_or_zero(b1[k]);
        }
        mma_16816_f16(o[8 * i + 4 * h + k], p[0], p[1], p[2], p[3], h2_as_u32(b0[k]), h2_as_u32(b1[k]));
      }
    }
  return false;
}

// The same for a masked block with values that are not finite: they count as zero in the product, whose rows share
// them, and 0 x, which is nan for them and 0 for all others, is added for the rows that see the position. lo / hi: of this
// lane's rows, relative to the block. Called, not inlined, so that it takes no registers from the loop.
template <int HD, int G, int PL>
__device__ __noinline__ void add_odd_values(float (&o)[HD / 8][4], uint32_t p0, uint32_t p1, uint32_t p2, uint32_t p3,
                                            const uint8_t* vc, int any_lo, int any_hi, int2 row0, int2 row1) {
  const uint32_t p[4] = {p0, p1, p2, p3};
  add_values<HD, G, true, true>(o, p, vc, any_lo, any_hi);
  const __half2* vs = reinterpret_cast<const __half2*>(vc + code_bytes(HD));
  const int t = threadIdx.x & 3;
#pragma unroll 1
  for (int at = 0; at < kBlock; ++at) {
    const bool sees[2] = {at >= row0.x && at < row0.y, at >= row1.x && at < row1.y};
    if (!sees[0] && !sees[1]) continue;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {           // the lane's elements t HD / 4 ...; element e is in tile e % (HD / 8)
      const __half2 sm = vs[at * (HD / G) + (t * (HD / 4) + 8 * j) / G];
      __half2 n[4];
      codes_h2(*reinterpret_cast<const uint32_t*>(vc + at * (HD / 2) + t * (HD / 8) + 4 * j), n);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 x = __half22float2(__hfma2(n[q], __low2half2(sm), __high2half2(sm)));
        const int i = (8 * j + q) % (HD / 8), k = 8 * j / (HD / 8);
#pragma unroll
        for (int r = 0; r < 3 - PL; ++r) {
          float &a = o[i][2 * r + k], &b = o[i + 4][2 * r + k];
          a = sees[r] ? fmaf(0.f, x.x, a) : a;
          b = sees[r] ? fmaf(0.f, x.y, b) : b;
        }
      }
    }
  }
  __syncwarp();
}

// Two blocks of 16 positions in shared memory: what there is once for a step of the loop (waits, the maximum's
// shuffles and vote) is once for 32 positions. MASKED: some of them are not seen by some row. lo / hi: visible
// positions of this lane's rows, relative to the first block; any_lo / any_hi: of any row. A masked position
// has p = 0, and where no row sees it its scales are dropped too, since memory that was never written may
// hold codes for nan. Where some rows see it and it is not finite, the product takes it as zero for all of them, and the
// rows that do see it are given nan after it.
template <int HD, int G, int PL, bool MASKED>
__device__ __forceinline__ void attend_blocks(State<HD, PL>& st, const uint8_t* const (&blk)[2], const uint4* qf,
                                              const float (&coef)[3 - PL], const int (&lo)[3 - PL],
                                              const int (&hi)[3 - PL], int any_lo, int any_hi) {
  constexpr int R = 3 - PL;                 // rows of a lane
  constexpr int KW = HD / 32;               // words of a lane and position
  constexpr int NG = HD / G, TWO = HD == 256 && G == 32 ? 2 : 1;   // groups that a lane's key elements are in
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float z[R][8];                            // S of positions 16 b + t + 4 k, at 4 b + k
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint8_t* ks = blk[b] + code_bytes(HD);
    float c[2][4] = {};                     // of positions t, t + 4 | t + 8, t + 12
    uint32_t w[2][KW];
    __half2 sm[2][TWO];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * j + (g >> 1) + 4 * (g & 1);
      const uint8_t* kp = blk[b] + row * (HD / 2) + t * (HD / 8);
      if constexpr (KW >= 4) {
#pragma unroll
        for (int i = 0; i < KW; i += 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(kp + 4 * i);
          w[j][i] = u.x; w[j][i + 1] = u.y; w[j][i + 2] = u.z; w[j][i + 3] = u.w;
        }
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(kp);
        w[j][0] = u.x; w[j][1] = u.y;
      }
#pragma unroll
      for (int i = 0; i < TWO; ++i) sm[j][i] = reinterpret_cast<const __half2*>(ks)[row * NG + (t * (HD / 4) + 32 * i) / G];
    }
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const uint4 a0 = qf[(2 * i) * 32 + lane], a1 = qf[(2 * i + 1) * 32 + lane];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const __half2 u = sm[j][TWO == 2 ? i / 4 : 0], s2 = __low2half2(u), m2 = __high2half2(u);
        __half2 n[4];
        codes_h2(w[j][i], n);
#pragma unroll
        for (int k = 0; k < 4; ++k) n[k] = __hfma2(n[k], s2, m2);
        mma_16816_f16(c[j], a0.x, a0.y, a0.z, a0.w, h2_as_u32(n[0]), h2_as_u32(n[1]));
        mma_16816_f16(c[j], a1.x, a1.y, a1.z, a1.w, h2_as_u32(n[2]), h2_as_u32(n[3]));
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (PL == 2) {
          z[0][4 * b + 2 * j + k] = c[j][k] + c[j][k + 2];
        } else {
          z[0][4 * b + 2 * j + k] = c[j][k];
          z[R - 1][4 * b + 2 * j + k] = c[j][k + 2];
        }
      }
  }
  if (MASKED) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (t + 4 * k < lo[r] || t + 4 * k >= hi[r]) z[r][k] = -INFINITY;
  }
  float mn[R];
  bool grows = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float x = fmaxf(fmaxf(z[r][0], z[r][1]), fmaxf(z[r][2], z[r][3]));
    x = fmaxf(x, fmaxf(fmaxf(z[r][4], z[r][5]), fmaxf(z[r][6], z[r][7])));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    mn[r] = MASKED && x == -INFINITY ? -INFINITY : x * coef[r];   // coef may be 0
    grows = grows || mn[r] > st.m[r] + kLazy;                     // st.m = -inf: the first one
  }
  if (__any_sync(0xffffffffu, grows)) {
    float f[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float top = fmaxf(st.m[r], mn[r]);
      f[r] = top > st.m[r] ? ex2(st.m[r] - top) : 1.f;
      st.m[r] = top;
      st.l[r] *= f[r];
    }
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      st.o[i][0] *= f[0];
      st.o[i][1] *= f[0];
      st.o[i][2] *= f[R - 1];
      st.o[i][3] *= f[R - 1];
    }
  }
  uint32_t a[2][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float base = kPShift - (MASKED && st.m[r] == -INFINITY ? 0.f : st.m[r]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float p[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        p[k] = ex2(fmaf(z[r][2 * j + k], coef[r], base));
        // a masked position, where coef is 0
        if (MASKED && z[r][2 * j + k] == -INFINITY) p[k] = 0.f;
        st.l[r] += p[k];
      }
      if (PL == 2) {
        __half2 h, l;
        split_h2(p[0], p[1], h, l);
        a[j >> 1][2 * (j & 1)] = h2_as_u32(h);
        a[j >> 1][2 * (j & 1) + 1] = h2_as_u32(l);
      } else {
        a[j >> 1][2 * (j & 1) + r] = h2_as_u32(__floats2half2_rn(p[0], p[1]));
      }
    }
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint8_t* vc = blk[b] + code_bytes(HD) + scale_bytes(HD, G);
    const bool odd = add_values<HD, G, MASKED, false>(st.o, a[b], vc, any_lo - 16 * b, any_hi - 16 * b);
    if (MASKED && odd) {
      float o[HD / 8][4];                       // a copy that has an address
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = st.o[i][j];
      add_odd_values<HD, G, PL>(o, a[b][0], a[b][1], a[b][2], a[b][3], vc, any_lo - 16 * b, any_hi - 16 * b,
                                make_int2(lo[0] - 16 * b, hi[0] - 16 * b), make_int2(lo[R - 1] - 16 * b, hi[R - 1] - 16 * b));
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) st.o[i][j] = o[i][j];
    }
  }
}

template <int HD, int PL>
__device__ __forceinline__ void store_part(const State<HD, PL>& st, float* part) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) {
    if (PL == 2)
      reinterpret_cast<float2*>(part)[i * 32 + lane] = make_float2(st.o[i][0] + st.o[i][2], st.o[i][1] + st.o[i][3]);
    else
      reinterpret_cast<float4*>(part)[i * 32 + lane] = make_float4(st.o[i][0], st.o[i][1], st.o[i][2], st.o[i][3]);
  }
  float* ml = part + Part<HD, PL>::kStats;
  if ((lane & 3) == 0)
#pragma unroll
    for (int r = 0; r < 3 - PL; ++r) {
      ml[(lane >> 2) + 8 * r] = st.m[r];
      ml[16 + (lane >> 2) + 8 * r] = st.l[r];
    }
}

template <int DT>
__device__ __forceinline__ void store2(void* out, long i, float x, float y) {
  if (DT == QL_F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(out) + i) = make_float2(x, y);
  else if (DT == QL_F16) *reinterpret_cast<__half2*>(reinterpret_cast<__half*>(out) + i) = __floats2half2_rn(x, y);
  else *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(out) + i) = __floats2bfloat162_rn(x, y);
}

// Output rows of a tile: row i is token q0 + i / grp, head kvh grp + i % grp.
__device__ __forceinline__ long out_row(const AttnArgs& a, int q0, int kvh, int row, int grp) {
  return (long)(q0 + row / grp) * a.NH + kvh * grp + row % grp;
}

template <int DT, int HD, int PL>
__device__ __forceinline__ void write_tile(const AttnArgs& a, const State<HD, PL>& st, int q0, int kvh, int r0,
                                           int nrows, int grp) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 3 - PL; ++r) {
    if (g + 8 * r >= nrows) continue;
    const float inv = st.l[r] == 0.f ? 0.f : 1.f / st.l[r];   // a row that sees nothing is zero
    const long at = out_row(a, q0, kvh, r0 + g + 8 * r, grp) * HD + t * (HD / 4);
    // the lane's HD / 4 elements are consecutive: tile i holds elements i and HD / 8 + i of them
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < HD / 8; i += 2) {
        const float x = (PL == 2 ? st.o[i][k] + st.o[i][k + 2] : st.o[i][2 * r + k]) * inv;
        const float y = (PL == 2 ? st.o[i + 1][k] + st.o[i + 1][k + 2] : st.o[i + 1][2 * r + k]) * inv;
        store2<DT>(a.out, at + k * (HD / 8) + i, x, y);
      }
  }
}

// The line of units cut for `warps` warps: the first `extra` of them take `each` + 1, the others `each`.
struct Split {
  long long warps, each, extra;
  __device__ __forceinline__ Split() {}
  __device__ __forceinline__ Split(long long units, int most) {
    warps = min(units, (long long)most);
    each = warps ? units / warps : 0;
    extra = units - warps * each;
  }
  __device__ __forceinline__ long long start(long long w) const { return w * each + min(w, extra); }
  __device__ __forceinline__ int warp_of(long long u) const {
    const long long big = extra * (each + 1);
    return (int)(u < big ? u / (each + 1) : extra + (u - big) / each);
  }
};

// A warp's piece of the line and the tile it is at: in shared memory, since the loop over a tile's blocks
// needs none of it and has no registers to spare.
struct Piece {
  long long u0, u1, u, us;      // the piece, the next tile in it, and where request b begins
  long long item0, item1;       // the tile
  Request r;
  int b, kvh, r0, nrows, lo_all, hi_all;
  int head, whole;              // its first tile began in an earlier warp; and goes on past this one
};

struct Cross {          // a tile that this CTA shares with others
  int valid, q0, kvh, r0, nrows, first, last, finish;
};

template <int DT, int HD, int G, int PL>
__global__ void __launch_bounds__(Shape<HD>::kThreads, 1) kv4_attention_kernel(AttnArgs a) {
  constexpr int R = 3 - PL, ROWS = 16 / PL, NW = Shape<HD>::kWarps, ST = Shape<HD>::kStages, NT = Shape<HD>::kThreads;
  constexpr int BB = block_bytes(HD, G);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_sums[NW], start_unit[NW];
  __shared__ int start_req[NW];
  __shared__ Piece pieces[NW];
  __shared__ Split sh_split;
  __shared__ Cross cross[2];
  __shared__ int abort_flag;
  using L = Smem<HD, G>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2;
  const int grp = a.NH / a.NKV;
  uint8_t* ring = smem + L::kRing + warp * ST * BB;
  uint4* qf = reinterpret_cast<uint4*>(smem + L::kQ) + warp * (HD / 16) * 32;
  const uint32_t ring_s = ptx::smem_addr(ring), bar = ptx::smem_addr(smem + L::kBar) + warp * ST * 8;
  if (lane == 0) {
    for (int s = 0; s < ST; ++s) ptx::mbar_init(bar + 8 * s, 1);
  }
  if (tid == 0) {
    abort_flag = 0;
    cross[0].valid = cross[1].valid = 0;
  }
  ptx::fence_mbar_init();
  __syncthreads();
  // rows of no request are zero
  const long used = (long)cu(a, a.B) * a.NH * HD, all = (long)a.T * a.NH * HD;
  for (long i = used + (long)blockIdx.x * NT + tid; i < all; i += (long)gridDim.x * NT)
    store_from_float(a.out, DT, i, 0.f);

  // The line of units: where this warp's piece begins. Up to 256 requests each warp finds it alone; for
  // more, every thread sums some requests and the block adds up (1 request of 64 positions: 10.9 us alone, 12.5 by
  // the block; 96 of 2000 44.2 and 46.2; 250 90.0 and 91.7; 1000 301.8 and 296.3).
  const long long w0 = (long long)blockIdx.x * NW;
  long long W = 0, us = 0;                     // units in all, and before request b
  int b = 0;
  Request r = {};
  Split split;
  if (a.B <= 256) {
    const int each = (a.B + 31) / 32, b0 = min(lane * each, a.B), b1 = min(b0 + each, a.B);
    long long mine = 0;
    for (int i = b0; i < b1; ++i) mine += units_of(load_request<ROWS>(a, i), a.NKV);
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    W = __shfl_sync(0xffffffffu, incl, 31);
    split = Split(W, gridDim.x * NW);
    if (w0 >= split.warps) return;
    if (w0 + warp < split.warps) {
      const long long u = split.start(w0 + warp);
      const int owner = __popc(__ballot_sync(0xffffffffu, incl <= u));   // the lane whose requests it is among
      us = __shfl_sync(0xffffffffu, incl - mine, owner);
      b = min(owner * each, a.B - 1);
      for (;; ++b) {
        r = load_request<ROWS>(a, b);
        if (u < us + units_of(r, a.NKV)) break;
        us += units_of(r, a.NKV);
      }
    }
  } else {
    const int each = (a.B + NT - 1) / NT, b0 = min(tid * each, a.B), b1 = min(b0 + each, a.B);
    long long mine = 0;
    for (int i = b0; i < b1; ++i) mine += units_of(load_request<ROWS>(a, i), a.NKV);
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    long long before = incl - mine;
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += warp_sums[w];
      W += warp_sums[w];
    }
    split = Split(W, gridDim.x * NW);
    if (w0 >= split.warps) return;
    if (mine > 0 && split.start(w0) < before + mine) {
      long long s = before, n = 0;
      int i = b0 - 1;
      for (int w = 0; w < NW && w0 + w < split.warps; ++w) {
        const long long u = split.start(w0 + w);
        if (u < before) continue;
        if (u >= before + mine) break;
        while (i < b0 || u >= s + n) {
          s += n;
          n = units_of(load_request<ROWS>(a, ++i), a.NKV);
        }
        start_req[w] = i;
        start_unit[w] = s;
      }
    }
    __syncthreads();
    if (w0 + warp < split.warps) {
      b = start_req[warp];
      us = start_unit[warp];
      r = load_request<ROWS>(a, b);
    }
  }
  const bool busy = w0 + warp < split.warps;
  float* parts = a.parts + (long)blockIdx.x * (2 + NW) * Part<HD, PL>::kFloats;
  Piece& c = pieces[warp];
  if (lane == 0) {
    c.r = r;
    c.b = b;
    c.us = us;
    c.u0 = c.u = split.start(w0 + warp);
    c.u1 = busy ? split.start(w0 + warp + 1) : c.u0;
    c.item0 = c.item1 = 0;
    c.head = c.whole = 0;
    if (warp == 0) sh_split = split;
  }
  __syncwarp();
  State<HD, PL> st;
  int s = 0, phase = 0;                        // stage of the next block in the ring, and its parity
  while (c.u < c.u1) {
    // open the next tile of the piece
    int blk0, n, first_masked, first_seen;
    uint32_t src;
    int pos[R];
    float coef[R];
    bool bad[R];                                // nan: for this lane's rows
    {
      Request r = c.r;
      int b = c.b;
      long long us = c.us, u = c.u;
      while (u >= us + units_of(r, a.NKV)) {
        us += units_of(r, a.NKV);
        r = load_request<ROWS>(a, ++b);
      }
      const int it = (int)((u - us) / r.nblk);
      const long long item0 = us + (long long)it * r.nblk, item1 = item0 + r.nblk, end = min(item1, c.u1);
      const int kvh = it / r.tiles, r0 = (it - kvh * r.tiles) * ROWS, nrows = min(ROWS, r.ql * grp - r0);
      const int table_end = a.width << a.page_shift;
      const int p_first = r.seq - r.ql + r0 / grp, p_last = r.seq - r.ql + (r0 + nrows - 1) / grp;
      const int lo_all = a.window ? max(p_first - a.window + 1, 0) : 0, hi_all = min(p_last + 1, table_end);
      // blocks of the piece that some row of the tile sees; all rows see those from first_seen to
      // before first_masked
      blk0 = max(r.blo + (int)(u - item0), lo_all / kBlock);
      n = max(min(r.blo + (int)(end - item0), (hi_all + kBlock - 1) / kBlock) - blk0, 0);
      first_masked = (p_first + 1) / kBlock - blk0;
      first_seen = a.window ? (max(p_last - a.window + 1, 0) + kBlock - 1) / kBlock - blk0 : 0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        pos[i] = r.seq - r.ql + (r0 + min(g + 8 * i, nrows - 1)) / grp;
        bad[i] = r.seq > table_end;             // a length past the table
      }
      __syncwarp();
      if (lane == 0) {
        c.r = r;
        c.b = b;
        c.us = us;
        c.item0 = item0;
        c.item1 = item1;
        c.u = end;
        c.kvh = kvh;
        c.r0 = r0;
        c.nrows = nrows;
        c.lo_all = lo_all;
        c.hi_all = hi_all;
      }
      src = source(a, b, kvh, blk0, lane, n);
      load_queries<DT, HD, PL>(a, r, kvh, r0, nrows, grp, qf, coef, [&]() {
        const int at = s + lane;
        if (lane < min(ST, n)) issue<BB>(a, src, at < ST ? at : at - ST, ring_s, bar);
      });
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      st.m[i] = -INFINITY;
      st.l[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] = 0.f;
    uint32_t next = kNoBlock, missing = 0;
    __syncwarp();
    for (int i = 0; i < n; i += 2) {
      if ((i & 31) == 0) {                        // lane j looks up block j of the 32 after these
        missing = __ballot_sync(0xffffffffu, src == kNoBlock);
        next = source(a, c.b, c.kvh, blk0, i + 32 + lane, n);
      }
      const bool both = i + 1 < n;
      const int s1 = s + 1 == ST ? 0 : s + 1;
      if (!warp_wait(bar + 8 * s, phase, &abort_flag) ||
          (both && !warp_wait(bar + 8 * s1, phase ^ (s1 == 0), &abort_flag))) {
        // gave up: nan for this tile, and no copy left in flight
#pragma unroll
        for (int j = 0; j < R; ++j) bad[j] = true;
        for (int j = i; j < min(i + ST, n); ++j) {
          ptx::mbar_wait_drain(bar + 8 * s, phase);
          if (++s == ST) s = 0, phase ^= 1;
        }
        __syncwarp();
        break;
      }
      const uint32_t gone = (missing >> (i & 31)) & (both ? 3u : 1u);   // blocks whose page is not one of the cache's
      const uint8_t* const blk[2] = {ring + s * BB, ring + s1 * BB};
      if (i >= first_seen && i + 1 < first_masked && both && !gone) {
        const int all[R] = {};
        attend_blocks<HD, G, PL, false>(st, blk, qf, coef, all, all, 0, 2 * kBlock);
      } else {
        // (of a second block past the last one nothing is seen, and nothing of one that is gone: the rows that would
        // see it are nan)
        const int p0 = (blk0 + i) * kBlock, from = gone & 1 ? kBlock : 0, to = both && !(gone & 2) ? 2 * kBlock : kBlock;
        int lo[R], hi[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
          lo[j] = (a.window ? max(pos[j] - a.window + 1, 0) : 0) - p0;
          hi[j] = pos[j] + 1 - p0;
          bad[j] = bad[j] || ((gone & 1) && lo[j] < kBlock && hi[j] > 0) || ((gone & 2) && lo[j] < 2 * kBlock && hi[j] > kBlock);
          lo[j] = max(lo[j], from);
          hi[j] = min(hi[j], to);
        }
        attend_blocks<HD, G, PL, true>(st, blk, qf, coef, lo, hi, max(c.lo_all - p0, from), min(c.hi_all - p0, to));
      }
      __syncwarp();
      // the stages are free: blocks i + ST and i + ST + 1 go there
      const int ahead = i + ST + (lane & 1);
      if (ahead < n && (ahead & 31) == lane) issue<BB>(a, (ahead ^ i) & 32 ? next : src, lane & 1 ? s1 : s, ring_s, bar);
      if ((i & 31) == 30) src = next;
      if ((s += both ? 2 : 1) >= ST) s -= ST, phase ^= 1;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 1);
      st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 2);
      if (bad[i]) st.l[i] = __int_as_float(0x7fc00000);
    }
    if (c.item0 >= c.u0 && c.item1 <= c.u1) {
      write_tile<DT, HD, PL>(a, st, c.r.q0, c.kvh, c.r0, c.nrows, grp);
    } else if (c.item0 < c.u0) {                 // began in an earlier warp
      if (c.u < c.u1) store_part<HD, PL>(st, parts + (2 + warp) * Part<HD, PL>::kFloats);
      if (lane == 0) {
        c.head = 1;
        c.whole = c.item1 > c.u1;
        if (warp == 0)
          cross[0] = {1, c.r.q0, c.kvh, c.r0, c.nrows, sh_split.warp_of(c.item0) / NW, sh_split.warp_of(c.item1 - 1) / NW, 0};
      }
    }
    __syncwarp();
  }
  __syncthreads();

  // Join the parts of this CTA's warps: a tile's parts are in consecutive warps, and the warp where it begins
  // (warp 0 for one that began in another CTA) adds them up in their order. A warp's last part goes to shared
  // memory, where the rings and queries are done with; an earlier one is in the workspace. Loops over
  // four floats at a time, not straight code over the state: it runs once, and its instructions have to be fetched.
  constexpr int SIZE = Part<HD, PL>::kFloats, STATS = Part<HD, PL>::kStats;
  float* shared_parts = reinterpret_cast<float*>(smem);
  static_assert(NW * SIZE * 4 <= L::kBar, "the parts of a CTA's warps fit where its rings were");
  if (c.u0 < c.u1 && (c.item0 < c.u0 || c.item1 > c.u1)) store_part<HD, PL>(st, shared_parts + warp * SIZE);
  __syncthreads();
  const auto head_part = [&](int w) {
    return pieces[w].item0 < pieces[w].u0 ? shared_parts + w * SIZE : parts + (2 + w) * SIZE;
  };
  // four floats i of a part are two neighbouring lanes of a fragment, or one lane's two rows: to the output, lane
  // (g, t) of tile k has elements 2t HD / 8 + k and HD / 8 past it
  const auto put = [&](const Cross& x, int i, float4 v, float f0, float f1) {
    const int ln = i * PL & 31, gg = ln >> 2, e = 2 * (ln & 3) * (HD / 8) + (i * PL >> 5);
    const float o[4] = {v.x * f0, v.y * f0, v.z * (PL == 2 ? f0 : f1), v.w * (PL == 2 ? f0 : f1)};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = PL == 2 ? gg : gg + 8 * h;
      if (row >= x.nrows) continue;
      const long at = out_row(a, x.q0, x.kvh, x.r0 + row, grp) * HD + (PL == 2 ? e + 2 * h * (HD / 8) : e);
      store_from_float(a.out, DT, at, o[2 * h]);
      store_from_float(a.out, DT, at + HD / 8, o[2 * h + 1]);
    }
  };
#pragma unroll 1
  for (int run = 0; run < 2; ++run) {
    // 0: the tile that began in an earlier CTA, 1: one that begins in this warp and goes on
    if (!(run == 0 ? warp == 0 && c.head : c.item1 > c.u1 && c.item0 >= c.u0)) continue;
    bool open = run ? true : c.whole;            // goes on past the parts so far
    int n = 1;
    for (int w = warp + 1; open && w < NW && pieces[w].head; ++w) {
      ++n;
      open = pieces[w].whole;
    }
    constexpr int CH = HD / 8 / PL;              // fours of a lane: all of one row, or of two
    const int row = (PL == 2 ? 2 * lane & 31 : lane) >> 2;
    float m[R], l[R] = {}, base[R];
    float4 acc[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto part = [&](int p) -> const float* {
      return p == 0 && run ? shared_parts + warp * SIZE : head_part(warp + p);
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      for (int p = 0; p < n; ++p) m[r] = fmaxf(m[r], part(p)[STATS + row + 8 * r]);
      base[r] = m[r] == -INFINITY ? 0.f : m[r];
    }
#pragma unroll 1
    for (int p = 0; p < n; ++p) {
      const float* from = part(p);
      float f[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        f[r] = ex2(from[STATS + row + 8 * r] - base[r]);
        l[r] = fmaf(f[r], from[STATS + 16 + row + 8 * r], l[r]);
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float4 v = reinterpret_cast<const float4*>(from)[i * 32 + lane];
        acc[i].x = fmaf(f[0], v.x, acc[i].x);
        acc[i].y = fmaf(f[0], v.y, acc[i].y);
        acc[i].z = fmaf(f[R - 1], v.z, acc[i].z);
        acc[i].w = fmaf(f[R - 1], v.w, acc[i].w);
      }
    }
    if (run && !open) {
      const Cross x = {1, c.r.q0, c.kvh, c.r0, c.nrows, 0, 0, 0};
      const float f0 = l[0] == 0.f ? 0.f : 1.f / l[0], f1 = l[R - 1] == 0.f ? 0.f : 1.f / l[R - 1];
#pragma unroll
      for (int i = 0; i < CH; ++i) put(x, i * 32 + lane, acc[i], f0, f1);
      continue;
    }
    float* to = parts + run * SIZE;
#pragma unroll
    for (int i = 0; i < CH; ++i) reinterpret_cast<float4*>(to)[i * 32 + lane] = acc[i];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      to[STATS + row + 8 * r] = m[r];
      to[STATS + 16 + row + 8 * r] = l[r];
    }
    if (run && lane == 0)
      cross[1] = {1, c.r.q0, c.kvh, c.r0, c.nrows, (int)blockIdx.x, sh_split.warp_of(c.item1 - 1) / NW, 0};
  }
  if (tid == 0 && abort_flag) atomicExch(&g_kv4_status, 1);
  __syncthreads();
  if (tid < 2 && cross[tid].valid) {
    // of the CTAs that share the tile, the last to arrive joins their parts (the fence covers what the
    // barrier has shown this thread of the other threads' stores)
    const Cross x = cross[tid];
    __threadfence();
    const bool done = atomicAdd(&a.counters[x.first], 1u) == (unsigned)(x.last - x.first);
    if (done) a.counters[x.first] = 0u;
    __threadfence();
    cross[tid].finish = done;
  }
  __syncthreads();
  float* stats = reinterpret_cast<float*>(smem);    // [parts][m of 16 rows, l of 16 rows]
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const Cross x = cross[k];
    if (!x.valid || !x.finish) continue;
    const int n = x.last - x.first + 1;
    const auto part = [&](int p) {
      return a.parts + ((long)(x.first + p) * (2 + NW) + (p == 0 ? 1 : 0)) * SIZE;
    };
    constexpr int NQ = HD / 4 * 16 / PL, AHEAD = 8;
    float4 v[AHEAD];                             // the first parts, under way with the stats
    if (tid < NQ)
#pragma unroll
      for (int p = 0; p < AHEAD; ++p)
        if (p < n) v[p] = __ldcg(reinterpret_cast<const float4*>(part(p)) + tid);
    for (int i = tid; i < n * 32; i += NT) stats[i] = __ldcg(part(i >> 5) + STATS + (i & 31));
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < NQ; i += NT) {
      const int row = (i * PL & 31) >> 2;
      float base[R], l[R] = {};
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float m = -INFINITY;
        for (int p = 0; p < n; ++p) m = fmaxf(m, stats[p * 32 + row + 8 * r]);
        base[r] = m == -INFINITY ? 0.f : m;
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int p0 = 0; p0 < n; p0 += AHEAD) {
        if (i != tid || p0)
#pragma unroll
          for (int p = 0; p < AHEAD; ++p)
            if (p0 + p < n) v[p] = __ldcg(reinterpret_cast<const float4*>(part(p0 + p)) + i);
#pragma unroll
        for (int p = 0; p < AHEAD; ++p)
          if (p0 + p < n) {
            float f[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
              f[r] = ex2(stats[(p0 + p) * 32 + row + 8 * r] - base[r]);
              l[r] = fmaf(f[r], stats[(p0 + p) * 32 + 16 + row + 8 * r], l[r]);
            }
            acc.x = fmaf(f[0], v[p].x, acc.x);
            acc.y = fmaf(f[0], v[p].y, acc.y);
            acc.z = fmaf(f[R - 1], v[p].z, acc.z);
            acc.w = fmaf(f[R - 1], v[p].w, acc.w);
          }
      }
      put(x, i, acc, l[0] == 0.f ? 0.f : 1.f / l[0], l[R - 1] == 0.f ? 0.f : 1.f / l[R - 1]);
    }
    __syncthreads();
  }
}

// Whether requests of kPromptRows rows or more are the prompt kernel's. It takes 16 positions of 16 rows in a
// fifth of the streaming kernel's time (0.16 against 0.8 ns over all SMs at HD = 128), and costs a join and another
// launch, so it pays from some rows on. The host knows the tokens past one a request, and not how they are spread.
// Measured, both sides, bf16: 32 heads of 128 over 4, 6000 positions, 64 tokens 36 us (streaming 56), 256 49 (152), 2000
// 211 (1039); 64 tokens over 64 positions 22 (18), over 1000 27 (29); 8 requests of 8 tokens 37 (39), of 32 49 (90); 16
// heads of 64, 3000 positions: 64 tokens 24 (24), 256 33 (37). Where no request has the rows after all, the launch costs 8
// to 16 us: 64 requests of 4000 positions, 2 tokens each 83 (70), 32 heads over 8 and 3 tokens 126 (110). The same tokens
// may be one chunk beside decoding requests, which wins more than that.
bool prompts_pay(int T, int B, int NH, int HD, int dtype) {
  return dtype != QL_F32 && HD <= 128 && (long)(T - B) * NH * HD >= 1l << 17;
}

int sm_count() {
  int sms = 148, dev = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms <= 0 ? 148 : sms < kMaxCtas ? sms : kMaxCtas;
}

template <int HD>
constexpr size_t part_floats() {
  return (size_t)(2 + Shape<HD>::kWarps) * Part<HD, 1>::kFloats;
}
// The two kernels run one after the other and share the memory.
size_t parts_bytes(int HD, int ctas) {
  const size_t own = (HD == 64 ? part_floats<64>() : HD == 128 ? part_floats<128>() : part_floats<256>()) * ctas * sizeof(float);
  return max(own, kv4_prompt_bytes(HD, ctas));
}

template <int DT, int HD, int G, int PL>
int launch_one(const AttnArgs& a, int ctas, cudaStream_t st) {
  auto kern = kv4_attention_kernel<DT, HD, G, PL>;
  static int configured_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_dev != dev) {
    const int rc = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD, G>::kBytes),
                               "cudaFuncSetAttribute(kv4 attention smem)");
    if (rc) return rc;
    configured_dev = dev;
  }
  kern<<<ctas, Shape<HD>::kThreads, Smem<HD, G>::kBytes, st>>>(a);
  return cuda_status(cudaGetLastError(), "ql_kv4_attention launch");
}

template <int DT, int HD, int G>
int launch(const AttnArgs& a, int ctas, cudaStream_t st) {
  // One plane where 16-bit inputs fill more than 8 rows of a tile: their outputs keep no more than the 11 bits of a
  // single fp16 probability. The host knows the mean only. Measured, 64 requests of 4000 positions, bf16, HD = 128,
  // one plane (two planes): 32 heads over 8, 1 token 103 us (98), 3 tokens 126 (189); over 4, 1 token 62 (59),
  // 2 tokens 83 (104). HD = 256, 32 requests: 32 over 4, 1 token 67 (67), 2 tokens 84 (103).
  constexpr bool can = DT != QL_F32;
  if (can && (long)a.T * (a.NH / a.NKV) > 8L * a.B) return launch_one<DT, HD, G, can ? 1 : 2>(a, ctas, st);
  return launch_one<DT, HD, G, 2>(a, ctas, st);
}

template <int DT>
int launch_sizes(const AttnArgs& a, int HD, int group, int ctas, cudaStream_t st) {
  if (HD == 64) return group == 32 ? launch<DT, 64, 32>(a, ctas, st) : launch<DT, 64, 64>(a, ctas, st);
  if (HD == 128)
    return group == 32   ? launch<DT, 128, 32>(a, ctas, st)
           : group == 64 ? launch<DT, 128, 64>(a, ctas, st)
                         : launch<DT, 128, 128>(a, ctas, st);
  return group == 32   ? launch<DT, 256, 32>(a, ctas, st)
         : group == 64 ? launch<DT, 256, 64>(a, ctas, st)
                       : launch<DT, 256, 128>(a, ctas, st);
}

}  // namespace

int take_kv4_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kv4_status, sizeof(int)) != cudaSuccess) return 0;
  if (v) cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int));
  return v | take_kv4_prompt_status();
}

}  // namespace ql

using namespace ql;

extern "C" size_t ql_kv4_attention_workspace(int NH, int NKV, int HD) {
  if (!kv4::sizes_ok(NKV, HD, 16, 32) || NH <= 0) return 0;
  return kMaxCtas * sizeof(unsigned int) + parts_bytes(HD, sm_count());
}

extern "C" int ql_kv4_attention(const void* q, int dtype, long ldq, int T, int NH, int NKV, int HD, const void* cache,
                                int num_pages, int page, int group, const int32_t* table, long table_stride,
                                int table_width, const int32_t* seq_lens, const int32_t* cu_q, int B, float scale,
                                int window, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (T == 0) return QL_OK;
  if (!q || !cache || !table || !seq_lens || !out || T < 0 || B <= 0 || NH <= 0 || NKV <= 0 || NH % NKV ||
      dtype < QL_F32 || dtype > QL_BF16 || ldq < (long)NH * HD || table_width <= 0 || table_stride < table_width ||
      window < 0 || (long)table_width * page > INT32_MAX || (!cu_q && T < B)) {
    set_error("ql_kv4_attention: bad arguments (T=%d B=%d NH=%d NKV=%d HD=%d ldq=%ld width=%d window=%d dtype=%d)", T, B,
              NH, NKV, HD, ldq, table_width, window, dtype);
    return QL_ERR_ARG;
  }
  if (!kv4::sizes_ok(NKV, HD, page, group) || num_pages <= 0 || (reinterpret_cast<uintptr_t>(cache) & 15)) {
    set_error("ql_kv4_attention: unsupported cache (pages=%d NKV=%d HD=%d page=%d group=%d; HD 64, 128 or 256, page a "
              "power of two 16 to 4096, group 32, 64 or 128 and at most HD, 16-byte aligned)", num_pages, NKV, HD, page,
              group);
    return QL_ERR_ARG;
  }
  const size_t need = ql_kv4_attention_workspace(NH, NKV, HD);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_error("ql_kv4_attention: workspace of %zu bytes (16-byte aligned, zeroed once) needed", need);
    return QL_ERR_ARG;
  }
  if ((long)num_pages * NKV * (page / kv4::kBlock) >= 0xffffffffl) {
    set_error("ql_kv4_attention: a cache of %ld blocks is past 32 bits", (long)num_pages * NKV * (page / kv4::kBlock));
    return QL_ERR_UNSUPPORTED;
  }
  const int ctas = sm_count();
  const size_t es = dtype == QL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % 8 || reinterpret_cast<uintptr_t>(q) % 16 || ldq * es % 16) {
    set_error("ql_kv4_attention: out must be 8-byte aligned, the tokens of q 16-byte aligned (ldq=%ld)", ldq);
    return QL_ERR_ALIGN;
  }
  AttnArgs a;
  a.q = q;
  a.ldq = ldq;
  a.T = T;
  a.NH = NH;
  a.NKV = NKV;
  a.cache = reinterpret_cast<const uint8_t*>(cache);
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctz((unsigned)page);
  a.table = table;
  a.table_stride = table_stride;
  a.width = table_width;
  a.seq_lens = seq_lens;
  a.cu_q = cu_q;
  a.B = B;
  a.scale = scale;
  a.window = window < table_width * page ? window : 0;   // one as long as the table hides nothing
  a.prompt_rows = prompts_pay(T, B, NH, HD, dtype) ? kPromptRows : 0;
  a.out = out;
  a.counters = reinterpret_cast<unsigned int*>(workspace);
  a.parts = reinterpret_cast<float*>(a.counters + kMaxCtas);
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.prompt_rows && cu_q) {
    const int rc = kv4_prompt_attention(a, dtype, HD, group, ctas, st);
    if (rc) return rc;
  } else {
    a.prompt_rows = 0;
  }
  return dtype == QL_F32   ? launch_sizes<QL_F32>(a, HD, group, ctas, st)
         : dtype == QL_F16 ? launch_sizes<QL_F16>(a, HD, group, ctas, st)
                           : launch_sizes<QL_BF16>(a, HD, group, ctas, st);
}
