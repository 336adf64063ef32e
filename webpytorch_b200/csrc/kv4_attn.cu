// Attention over the paged 4-bit cache: softmax(q K^T scale) V for ragged requests, causal from the
// end of each request (query i of a request is at position seq_len - q_len + i), with an optional
// sliding window, for one query token or many.
//
// Rows. The query heads that share a key/value head and the request's query tokens form one list of
// rows, r = i (NH / NKV) + head; a tile takes the next rows of it. The warp MMA (m16n8k16, fp16 in,
// fp32 out) has 16 of them. One-plane tiles use them for 16 rows; two-plane tiles hold 8 rows as
// fp16 high and low parts (22 bits), rows r and r + 8 of the MMA, whose results the same thread
// holds and adds: fp32 queries and probabilities keep fp32 accuracy, and tiles of 8 rows or fewer
// pay nothing for it.
// Keys. A lane owns HD / 4 consecutive elements of a position (a 16-byte load at HD = 128), all in
// one group of at least 32 elements, so a scale pair is loaded once per position. The order of the
// contraction is free, so the pairs the nibble masks give (element j with j + 4 of a word) are the
// MMA's k pairs and the queries are laid out to match.
// Values. P V contracts over positions. The C fragment of S gives lane t of a quad positions t,
// t + 4, t + 8, t + 12 of the block (the key rows are read in the order that makes it so); the words
// of two positions are interleaved by one byte permutation per half, after which the same masks give
// pairs of positions. Codes become the exact fp16 values they stand for: one fma each.
#include "kv4_common.cuh"

namespace ql {
namespace {

using namespace kv4;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct AttnArgs {
  const void* q;
  long ldq;
  int T, NH, NKV;
  const uint8_t* cache;
  int num_pages, page_shift, group;
  const int32_t* table;
  long table_stride;
  int width;
  const int32_t* seq_lens;
  const int32_t* cu_q;
  int B;
  float scale;
  int window;
  void* out;
};

__device__ __forceinline__ int cu(const AttnArgs& a, int b) { return a.cu_q ? min(max(a.cu_q[b], 0), a.T) : min(b, a.T); }

// Splits x into fp16 high and low parts, x = hi + lo to 22 bits.
__device__ __forceinline__ void split_h(float x, __half& hi, __half& lo) {
  hi = __float2half_rn(x);
  lo = __float2half_rn(x - __half2float(hi));
}

template <int HD, int PL>
struct State {
  float o[HD / 8][4];   // C fragments of the output, tile i: element (2t, 2t + 1) * HD / 8 + i
  float m[3 - PL];      // running maximum of rows g (and g + 8), in units of log2
  float l[3 - PL];      // this lane's part of the sum of exponentials
};

// One block of 16 positions. qf: the tile's A fragments [HD / 16][32] uint4 in shared memory.
// coef[r] * S is the score in units of log2; lo / hi: visible positions of this lane's rows, relative
// to the block. A masked position has p = 0, and its scales are dropped too, since memory that was
// never written may hold codes for nan.
template <int HD, int PL>
__device__ __forceinline__ void attend_block(State<HD, PL>& st, const uint8_t* blk, const uint4* qf, int group,
                                             const float (&coef)[3 - PL], bool masked, const int (&lo)[3 - PL],
                                             const int (&hi)[3 - PL], int any_lo, int any_hi) {
  constexpr int R = 3 - PL;                 // rows of a lane
  constexpr int KW = HD / 32, VW = HD / 64; // words of a lane: keys of one position, values of one
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ng = HD / group;
  const uint8_t* ks = blk + code_bytes(HD);
  const uint8_t* vc = ks + scale_bytes(HD, group);
  const uint8_t* vs = vc + code_bytes(HD);
  float z[R][4];                            // positions t, t + 4, t + 8, t + 12
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = 8 * j + (g >> 1) + 4 * (g & 1);
    uint32_t w[KW];
#pragma unroll
    for (int i = 0; i < KW; i += (KW >= 4 ? 4 : 2)) {
      if constexpr (KW >= 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(blk + row * (HD / 2) + t * (HD / 8) + i * 4);
        w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(blk + row * (HD / 2) + t * (HD / 8) + i * 4);
        w[i] = u.x; w[i + 1] = u.y;
      }
    }
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    __half2 s2, m2;
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      if (i == 0 || HD == 256) {            // at HD = 256 a lane's 64 elements may span two groups
        const __half2 sm = reinterpret_cast<const __half2*>(ks)[row * ng + (t * (HD / 4) + 8 * i) / group];
        s2 = __low2half2(sm);
        m2 = __high2half2(sm);
      }
      __half2 n[4];
      codes_h2(w[i], n);
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] = __hfma2(n[k], s2, m2);
      const uint4 a0 = qf[(2 * i) * 32 + lane], a1 = qf[(2 * i + 1) * 32 + lane];
      mma_16816_f16(c, a0.x, a0.y, a0.z, a0.w, h2_as_u32(n[0]), h2_as_u32(n[1]));
      mma_16816_f16(c, a1.x, a1.y, a1.z, a1.w, h2_as_u32(n[2]), h2_as_u32(n[3]));
    }
    if (PL == 2) {
      z[0][2 * j] = (c[0] + c[2]) * coef[0];
      z[0][2 * j + 1] = (c[1] + c[3]) * coef[0];
    } else {
      z[0][2 * j] = c[0] * coef[0];
      z[0][2 * j + 1] = c[1] * coef[0];
      z[R - 1][2 * j] = c[2] * coef[R - 1];
      z[R - 1][2 * j + 1] = c[3] * coef[R - 1];
    }
  }
  if (masked)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (t + 4 * k < lo[r] || t + 4 * k >= hi[r]) z[r][k] = -INFINITY;
  float mn[R];
  bool grows = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float x = fmaxf(fmaxf(z[r][0], z[r][1]), fmaxf(z[r][2], z[r][3]));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    mn[r] = fmaxf(st.m[r], x);
    grows = grows || mn[r] > st.m[r];
  }
  if (__any_sync(0xffffffffu, grows)) {
    float f[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f[r] = mn[r] > st.m[r] ? exp2f(st.m[r] - mn[r]) : 1.f;
      st.m[r] = mn[r];
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
  // p' = 2^11 p: fp16 keeps 11 bits of probabilities down to 2^-25
  uint32_t a[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float p[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float base = (st.m[r] == -INFINITY ? 0.f : st.m[r]) - 11.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        p[r][k] = exp2f(z[r][2 * j + k] - base);
        st.l[r] += p[r][k];
      }
    }
    if (PL == 2) {
      __half h0, l0, h1, l1;
      split_h(p[0][0], h0, l0);
      split_h(p[0][1], h1, l1);
      a[2 * j] = h2_as_u32(__halves2half2(h0, h1));
      a[2 * j + 1] = h2_as_u32(__halves2half2(l0, l1));
    } else {
      a[2 * j] = h2_as_u32(__floats2half2_rn(p[0][0], p[0][1]));
      a[2 * j + 1] = h2_as_u32(__floats2half2_rn(p[R - 1][0], p[R - 1][1]));
    }
  }
  // values: words of positions t, t + 4 | t + 8, t + 12, elements g HD / 8 ...
  uint32_t w[4][VW];
  __half2 s2[2], m2[2];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint8_t* p = vc + (t + 4 * k) * (HD / 2) + g * (HD / 16);
#pragma unroll
    for (int i = 0; i < VW; ++i) w[k][i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
  {
    __half2 sm[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sm[k] = reinterpret_cast<const __half2*>(vs)[(t + 4 * k) * ng + g * (HD / 8) / group];
      if (masked && (t + 4 * k < any_lo || t + 4 * k >= any_hi)) sm[k] = h2_const(0u);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      s2[k] = __lows2half2(sm[2 * k], sm[2 * k + 1]);
      m2[k] = __highs2half2(sm[2 * k], sm[2 * k + 1]);
    }
  }
#pragma unroll
  for (int i = 0; i < VW; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t sel = h ? 0x7632u : 0x5410u;
      __half2 b0[4], b1[4];
      // nibbles 0..3 of the half word: codes_h2 reads them as (nibble j, nibble j + 4) of the
      // interleaved word, which are the two positions
      codes_h2(__byte_perm(w[0][i], w[1][i], sel), b0);
      codes_h2(__byte_perm(w[2][i], w[3][i], sel), b1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        b0[k] = __hfma2(b0[k], s2[0], m2[0]);
        b1[k] = __hfma2(b1[k], s2[1], m2[1]);
        mma_16816_f16(st.o[8 * i + 4 * h + k], a[0], a[1], a[2], a[3], h2_as_u32(b0[k]), h2_as_u32(b1[k]));
      }
    }
}

// The request and the first row of tile x. Tiles of request b start at cu[b] grp / rows + b, which
// leaves room for ceil(rows of b / rows) of them wherever the division falls.
__device__ __forceinline__ int tile_start(const AttnArgs& a, int b, int grp, int rows) {
  return (int)((long)cu(a, b) * grp / rows) + b;
}

template <int DT, int HD, int PL>
__global__ void __launch_bounds__(kThreads) kv4_attention_kernel(AttnArgs a) {
  constexpr int R = 3 - PL, ROWS = 16 / PL;
  __shared__ uint4 qf[HD / 16][32];
  __shared__ float qexp[ROWS];
  __shared__ float red_m[kWarps][ROWS], red_l[kWarps][ROWS];
  __shared__ float red_o[kWarps][ROWS][HD];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int grp = a.NH / a.NKV, kvh = blockIdx.y, x = blockIdx.x;
  int b = 0;
  for (int hi = a.B - 1; b < hi;) {   // the last b whose first tile is at or before x
    const int mid = (b + hi + 1) >> 1;
    if (tile_start(a, mid, grp, ROWS) <= x) b = mid;
    else hi = mid - 1;
  }
  const int q0 = cu(a, b), ql = max(cu(a, b + 1) - q0, 0);
  const int r0 = (x - tile_start(a, b, grp, ROWS)) * ROWS;
  const int nrows = min(ROWS, ql * grp - r0);
  if (nrows <= 0) return;
  // queries: row r of the tile is token q0 + (r0 + r) / grp, head kvh grp + (r0 + r) % grp
  for (int r = warp; r < ROWS; r += kWarps) {
    float mx = 0.f;
    const int i = r0 + r;
    const long at = (long)(q0 + i / grp) * a.ldq + (long)(kvh * grp + i % grp) * HD;
    if (r < nrows)
      for (int d = lane; d < HD; d += 32) mx = fmaxf(mx, fabsf(load_as_float(a.q, DT, at + d)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const int e = stage_exponent(mx);
    if (lane == 0) qexp[r] = exp2i(e);
    const float inv = exp2i(-e);
    for (int d = lane; d < HD; d += 32) {
      const float v = r < nrows ? load_as_float(a.q, DT, at + d) * inv : 0.f;
      __half hi, lo;
      split_h(v, hi, lo);
      // element d: lane t = d / (HD / 4), word w, nibble j; fragment 2 w + (j & 2) / 2, registers
      // 0 / 1 (k pair 0) or 2 / 3 (k pair 1) by j & 1, half by j >> 2
      const int tt = d / (HD / 4), w = (d % (HD / 4)) / 8, j = d & 7;
      __half* f = reinterpret_cast<__half*>(&qf[2 * w + ((j >> 1) & 1)][(r & 7) * 4 + tt]);
      const int reg = 2 * (j & 1), half = j >> 2;
      if (PL == 2) {
        f[reg * 2 + half] = hi;
        f[(reg + 1) * 2 + half] = lo;
      } else {
        f[(reg + (r >> 3)) * 2 + half] = hi;
      }
    }
  }
  __syncthreads();
  const int table_end = a.width << a.page_shift;
  const int seq = max(a.seq_lens[b], 0);
  const int p_first = seq - ql + r0 / grp, p_last = seq - ql + (r0 + nrows - 1) / grp;
  const int lo_all = a.window ? max(p_first - a.window + 1, 0) : 0, hi_all = min(p_last + 1, table_end);
  State<HD, PL> st;
  float coef[R];
  int row_lo[R], row_hi[R];
  bool bad = seq > table_end;   // a length past the table: nan
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = g + 8 * r;
    coef[r] = qexp[row] * (a.scale * 1.4426950408889634f);
    const int p = seq - ql + (r0 + min(row, nrows - 1)) / grp;
    row_lo[r] = a.window ? max(p - a.window + 1, 0) : 0;
    row_hi[r] = p + 1;
    st.m[r] = -INFINITY;
    st.l[r] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) st.o[i][k] = 0.f;
  const int bb = block_bytes(HD, a.group);
  for (int blk = lo_all / kBlock + warp; blk * kBlock < hi_all; blk += kWarps) {
    const int p0 = blk * kBlock;
    const int page = a.table[b * a.table_stride + (p0 >> a.page_shift)];
    if (page < 0 || page >= a.num_pages) {
      bad = true;
      continue;
    }
    const uint8_t* src = a.cache + ((((long)page * a.NKV + kvh) << (a.page_shift - 4)) +
                                    ((p0 >> 4) & ((1 << (a.page_shift - 4)) - 1))) * bb;
    const bool masked = p0 + kBlock > p_first + 1 || (a.window && p0 < p_last - a.window + 1);
    int lo[R], hi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      lo[r] = row_lo[r] - p0;
      hi[r] = row_hi[r] - p0;
    }
    attend_block<HD, PL>(st, src, &qf[0][0], a.group, coef, masked, lo, hi, lo_all - p0, hi_all - p0);
  }
  // join the lanes of a row, then the warps
#pragma unroll
  for (int r = 0; r < R; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
    if (bad) st.l[r] = __int_as_float(0x7fc00000);
    if (t == 0) {
      red_m[warp][g + 8 * r] = st.m[r];
      red_l[warp][g + 8 * r] = st.l[r];
    }
  }
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int d = (2 * t + k) * (HD / 8) + i;
      if (PL == 2) {
        red_o[warp][g][d] = st.o[i][k] + st.o[i][k + 2];
      } else {
        red_o[warp][g][d] = st.o[i][k];
        red_o[warp][ROWS - 8 + g][d] = st.o[i][k + 2];
      }
    }
  __syncthreads();
  for (int i = tid; i < nrows * HD; i += kThreads) {
    const int r = i / HD, d = i - r * HD;
    float m = -INFINITY, l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red_m[w][r]);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(red_m[w][r] - base);
      l = fmaf(f, red_l[w][r], l);
      o = fmaf(f, red_o[w][r][d], o);
    }
    const int row = r0 + r;
    store_from_float(a.out, DT, ((long)(q0 + row / grp) * a.NH + kvh * grp + row % grp) * HD + d,
                     l == 0.f ? 0.f : o / l);     // a row that sees nothing is zero
  }
}

// Rows of q past the last request are padding: zero.
template <int DT>
__global__ void kv4_padding_kernel(AttnArgs a, long row) {
  const long used = (long)cu(a, a.B) * row;
  for (long i = used + (long)blockIdx.x * blockDim.x + threadIdx.x; i < a.T * row; i += (long)gridDim.x * blockDim.x)
    store_from_float(a.out, DT, i, 0.f);
}

template <int DT, int HD>
cudaError_t launch(const AttnArgs& a, cudaStream_t st) {
  const int grp = a.NH / a.NKV;
  // one plane where 16-bit inputs fill more than 8 rows: their outputs keep no more than the 11 bits
  // of a single fp16 probability (HD = 256 has no registers for 16 rows)
  constexpr bool can = DT != QL_F32 && HD != 256;
  const bool one_plane = can && (long)a.T * grp > 8L * a.B;
  const int rows = one_plane ? 16 : 8;
  const dim3 grid((unsigned)((long)a.T * grp / rows + a.B), a.NKV);
  if (one_plane) kv4_attention_kernel<DT, HD, (can ? 1 : 2)><<<grid, kThreads, 0, st>>>(a);
  else kv4_attention_kernel<DT, HD, 2><<<grid, kThreads, 0, st>>>(a);
  if (a.cu_q || a.T > a.B) kv4_padding_kernel<DT><<<64, 256, 0, st>>>(a, (long)a.NH * HD);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_hd(const AttnArgs& a, int HD, cudaStream_t st) {
  return HD == 64 ? launch<DT, 64>(a, st) : HD == 128 ? launch<DT, 128>(a, st) : launch<DT, 256>(a, st);
}

}  // namespace
}  // namespace ql

using namespace ql;

extern "C" size_t ql_kv4_attention_workspace(int NH, int NKV, int HD) {
  (void)NH;
  (void)NKV;
  (void)HD;
  return 0;
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
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("ql_kv4_attention: workspace of %zu bytes needed", need);
    return QL_ERR_ARG;
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
  a.group = group;
  a.table = table;
  a.table_stride = table_stride;
  a.width = table_width;
  a.seq_lens = seq_lens;
  a.cu_q = cu_q;
  a.B = B;
  a.scale = scale;
  a.window = window;
  a.out = out;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == QL_F32 ? launch_hd<QL_F32>(a, HD, st)
                        : dtype == QL_F16 ? launch_hd<QL_F16>(a, HD, st) : launch_hd<QL_BF16>(a, HD, st);
  return cuda_status(e, "ql_kv4_attention launch");
}
