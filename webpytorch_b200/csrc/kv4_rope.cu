// Norms of queries and keys for each head, the position rotation, and the write of keys and values
// into the paged 4-bit cache, in one pass over the QKV projection's rows.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = (x r) w                       (where the head has a norm)
//   z[i] = y[i] c_i - y[i + h] s_i,  z[i + h] = y[i + h] c_i + y[i] s_i   for i < h = rot / 2
// (rotate-half, as webtorch/lm_engine.py:66-74; elements past rot pass through). Codes of 4 bits
// have to come out the same wherever they are made, so every step is an IEEE operation without
// contraction and the mean's sum is a balanced tree of neighbours: x0 + x1, (x0 + x1) + (x2 + x3), ...
// which is what lanes that hold consecutive elements and a butterfly over the lanes add up.
//
// A call of many tokens has to read the rows and write q and the codes: 363 MB at 16384 tokens of 32 + 8 + 8 heads
// of 128 in bf16, 55 us at the measured copy rate. The kernel takes 112 us there, 3.2 TB/s: about 190
// instructions for 8 elements of a lane, many of them chains (the sum's tree and butterfly, square root and
// reciprocal, the group's minimum and range), fill 68 % of the issue slots. A call of a few tokens is one launch (6 us).
#include "kv4_common.cuh"

namespace ql {
namespace {

using namespace kv4;

constexpr int kThreads = 128;

struct RopeArgs {
  const void* qkv;
  long ld;
  int T, NH, NKV;
  const int32_t* positions;
  const float* cos;
  const float* sin;
  int lmax, half;          // half = rot / 2
  const float* qw;
  const float* kw;
  float eps;
  void* q_out;
  void* k_out;
  uint8_t* cache;
  long num_slots;
  int page_shift, group;
  const int64_t* slots;
};

template <int DT>
__device__ __forceinline__ float ld1(const void* p, long i) {
  return load_as_float(p, DT, i);
}

// Address of position `slot` of head g: codes of the keys (v = 0) or values (v = 1).
__device__ __forceinline__ uint8_t* block_of(const RopeArgs& a, long slot, int g, int HD) {
  const long page = slot >> a.page_shift;
  const int r = (int)(slot & ((1 << a.page_shift) - 1));
  return a.cache + ((page * a.NKV + g) << (a.page_shift - 4)) * block_bytes(HD, a.group) +
         (long)(r >> 4) * block_bytes(HD, a.group);
}

// Any row alignment and any rot: one warp per (token, head), lane l holds elements V l .. V l + V - 1.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  const int heads = a.NH + (a.cache || a.k_out ? (a.cache ? 2 : 1) * a.NKV : 0);
  const long item = (long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (item >= (long)a.T * heads) return;
  const long t = item / heads;
  const int h = (int)(item - t * heads);
  const bool is_q = h < a.NH, is_v = h >= a.NH + a.NKV;
  const int pos = a.positions[t];
  const long slot = a.cache ? a.slots[t] : -1;
  if (!is_q && a.cache && (slot < 0 || slot >= a.num_slots || pos < 0 || pos >= a.lmax)) return;
  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = ld1<DT>(a.qkv, t * a.ld + (long)h * HD + lane * V + i);
  if (!is_v) {
    const float* w = is_q ? a.qw : a.kw;
    if (w) {
      float s[V];
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = __fmul_rn(x[i], x[i]);
#pragma unroll
      for (int n = V; n > 1; n /= 2)
#pragma unroll
        for (int i = 0; i < n / 2; ++i) s[i] = __fadd_rn(s[2 * i], s[2 * i + 1]);
      float ss = s[0];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
      const float r = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.f / HD), a.eps)));
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[lane * V + i]);
    }
    const int hl = a.half / V;                       // lanes of a rotated half
    const bool first = lane < hl, second = lane >= hl && lane < 2 * hl;
    const int partner = first ? lane + hl : second ? lane - hl : lane;
    const bool in = pos >= 0 && pos < a.lmax;
    const long row = (long)(in ? pos : 0) * a.half + (second ? lane - hl : lane) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = __shfl_sync(0xffffffffu, x[i], partner);
      if (first || second) {
        const float c = a.cos[row + i], s = a.sin[row + i];
        x[i] = first ? __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y, s)) : __fadd_rn(__fmul_rn(x[i], c), __fmul_rn(y, s));
      }
    }
    // padding rows are zero; a position outside the tables gives nan
    if (!in)
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = pos < 0 ? 0.f : __int_as_float(0x7fc00000);
  }
  if (is_q || !a.cache) {
    void* out = is_q ? a.q_out : a.k_out;
    const long at = (t * (is_q ? a.NH : a.NKV) + (is_q ? h : h - a.NH)) * HD + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) store_from_float(out, DT, at + i, x[i]);
    return;
  }
  // 4 bits: minimum and range over the group's lanes
  const int gl = a.group / V;
  float lo = x[0], hi = x[0];
  bool ok = true;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    ok = ok && fabsf(x[i]) <= 65504.f;               // false for nan
  }
  for (int o = 1; o < gl; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    ok = __shfl_xor_sync(0xffffffffu, (int)ok, o) && ok;
  }
  __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)), m = __float2half_rn(lo);
  if (!ok) s = m = __ushort_as_half((unsigned short)0x7fff);
  const float sf = __half2float(s), mf = __half2float(m);
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float n = !ok || sf == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], mf), sf)), 0.f), 15.f);
    code |= (uint32_t)n << (4 * i);
  }
  const int r = (int)(slot & 15);
  uint8_t* blk = block_of(a, slot, is_v ? h - a.NH - a.NKV : h - a.NH, HD) +
                 (is_v ? code_bytes(HD) + scale_bytes(HD, a.group) : 0);
  uint8_t* cp = blk + r * (HD / 2) + lane * (V / 2);
  if (V == 2) *cp = (uint8_t)code;
  if (V == 4) *reinterpret_cast<uint16_t*>(cp) = (uint16_t)code;
  if (V == 8) *reinterpret_cast<uint32_t*>(cp) = code;
  if (lane % gl == 0)
    reinterpret_cast<__half2*>(blk + code_bytes(HD))[r * (HD / a.group) + lane / gl] = __halves2half2(s, m);
}

// Two IEEE fp32 products in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// rint(d / s) for 0 <= d <= 15 s and s a half, as IEEE division rounds it, packed 4 bits each. The product with
// 1 / s is off by a rounding or two, which matters next to k + 1/2 only, and there the comparison is exact:
// (k + 1/2) s and d - n s are fp32 numbers, and no d other than (k + 1/2) s itself has a quotient that rounds to
// k + 1/2 (a neighbour of d is further off, relatively, than half a step of the quotient). All elements are
// looked at at once whether one is that near; an integer is the low bits of the sum with 1.5 * 2^23.
template <int E>
__device__ __forceinline__ uint32_t round_quotients(const float (&d)[E], float s, float inv) {
  constexpr float kMagic = 12582912.f;
  constexpr uint32_t kBits = 0x4B400000u;
  const float half = 0.5f * s;
  float t[E], near = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    t[j] = __fadd_rn(__fmul_rn(d[j], inv), kMagic);             // ties to even
    near = fmaxf(near, fabsf(fmaf(-__fsub_rn(t[j], kMagic), s, d[j])));
  }
  if (near >= half) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float rest = fmaf(-__fsub_rn(t[j], kMagic), s, d[j]);
      if (fabsf(rest) > half || (fabsf(rest) == half && (__float_as_uint(t[j]) & 1u))) t[j] += rest > 0.f ? 1.f : -1.f;
    }
  }
  uint32_t code = 0u, offset = 0u;
#pragma unroll
  for (int j = E - 1; j >= 0; --j) {                            // (code << 4) + n, with the bits of 1.5 * 2^23 in it
    code = code * 16u + __float_as_uint(t[j]);
    offset = offset * 16u + kBits;
  }
  return code - offset;
}

// Rows of 16-byte aligned heads whose rotated halves are whole 16-byte pieces: a lane holds E consecutive
// elements (16 bytes; 8 fp32 elements at HD = 256), so 16 bytes a lane are read and written, a warp takes
// 32 E / HD heads at a time, and one token's cos, sin and slot serve all of its heads. `split` warps share a
// token, so that few tokens still fill the GPU; with many tokens each warp takes a whole one, since what it does
// once (position, cos, sin) is 4 us of its 27 (16384 tokens with the read of what was written, 1 / 2 / 4 warps a token:
// 135 / 147 / 177 us). kAhead loads are under way at once. All other rows take the kernel above: 297 us there, the
// same time up to 16 tokens.
constexpr int kVecThreads = 256;
constexpr int kAhead = 4;

template <int DT, int HD>
struct Lanes {
  static constexpr int SIZE = DT == QL_F32 ? 4 : 2;
  static constexpr int E = 16 / SIZE > HD / 32 ? 16 / SIZE : HD / 32;
  static constexpr int LPH = HD / E, HPW = 32 / LPH, NV = E * SIZE / 16;
};

template <int DT, int HD>
struct Token {
  long t;
  int pos;
  bool in;                       // a position of the tables
  const uint8_t* row;
  float c[Lanes<DT, HD>::E], s[Lanes<DT, HD>::E];   // of this lane's elements; s with the sign of its half
  int partner;                   // the lane with the other half's elements
  bool turns;                    // this lane's elements are rotated
  uint8_t* blk;                  // head 0's block in the cache
  long head_bytes;
  int r;                         // row in the block
};

template <int DT, int HD>
__device__ __forceinline__ void unpack(const uint4 (&raw)[Lanes<DT, HD>::NV], float (&x)[Lanes<DT, HD>::E]) {
#pragma unroll
  for (int v = 0; v < Lanes<DT, HD>::NV; ++v) {
    const uint32_t w[4] = {raw[v].x, raw[v].y, raw[v].z, raw[v].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == QL_F32) {
        x[4 * v + j] = __int_as_float(w[j]);
      } else {
        const float2 f = DT == QL_F16 ? __half22float2(u32_as_h2(w[j]))
                                      : make_float2(__int_as_float(w[j] << 16), __int_as_float(w[j] & 0xffff0000u));
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    }
  }
}

template <int DT, int HD>
__device__ __forceinline__ void store_head(void* out, long at, const float (&x)[Lanes<DT, HD>::E]) {
  uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(out) + at * Lanes<DT, HD>::SIZE);
#pragma unroll
  for (int v = 0; v < Lanes<DT, HD>::NV; ++v) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == QL_F32) {
        w[j] = __float_as_uint(x[4 * v + j]);
      } else if (DT == QL_F16) {
        w[j] = h2_as_u32(__floats2half2_rn(x[2 * j], x[2 * j + 1]));
      } else {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    p[v] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A head's elements in 4 bits: minimum and range over the group's lanes; an element that no half holds
// makes the maximum infinite.
template <int DT, int HD>
__device__ __forceinline__ void store_codes(const RopeArgs& a, const Token<DT, HD>& k, int h, bool is_v, int l,
                                            const float (&x)[Lanes<DT, HD>::E]) {
  constexpr int E = Lanes<DT, HD>::E;
  const int gl = a.group / E;
  float lo = x[0], hi = x[0], zero = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
    zero = fmaf(x[j], 0.f, zero);                    // nan where an element is not finite
  }
  if (!(zero == 0.f)) hi = INFINITY;
  for (int o = 1; o < gl; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const bool ok = hi <= 65504.f && lo >= -65504.f;
  __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f)), m = __float2half_rn(lo);
  if (!ok) s = m = __ushort_as_half((unsigned short)0x7fff);
  const float sf = __half2float(s), mf = __half2float(m);
  const bool flat = !(sf > 0.f);                     // constant, or not finite: codes 0
  const float inv = flat ? 0.f : __frcp_rn(sf), step = flat ? 1.f : sf;
  float d[E];
  // below zero by the minimum's rounding, above 15 steps by that and the scale's
#pragma unroll
  for (int j = 0; j < E; ++j) d[j] = fminf(fmaxf(__fsub_rn(x[j], mf), 0.f), flat ? 0.f : 15.f * step);
  const uint32_t code = round_quotients<E>(d, step, inv);
  if (h < 0) return;
  uint8_t* to = k.blk + h * k.head_bytes + (is_v ? code_bytes(HD) + scale_bytes(HD, a.group) : 0);
  uint8_t* cp = to + k.r * (HD / 2) + l * (E / 2);
  if (E == 4) *reinterpret_cast<uint16_t*>(cp) = (uint16_t)code;
  else *reinterpret_cast<uint32_t*>(cp) = code;
  if ((l & (gl - 1)) == 0)
    reinterpret_cast<__half2*>(to + code_bytes(HD))[k.r * (HD / a.group) + l / gl] = __halves2half2(s, m);
}

enum { kQuery, kKey, kValue };

// Steps i0 .. i1 - 1 of one kind of heads, HPW heads a step.
template <int DT, int HD, bool CACHE, bool FULL, int KIND>
__device__ __forceinline__ void heads(const RopeArgs& a, const Token<DT, HD>& k, int i0, int i1) {
  using L = Lanes<DT, HD>;
  constexpr int E = L::E;
  const int lane = threadIdx.x & 31, l = lane % L::LPH, sub = lane / L::LPH;
  const int count = KIND == kQuery ? a.NH : a.NKV, first = KIND == kQuery ? 0 : KIND == kKey ? a.NH : a.NH + a.NKV;
  const float* w = KIND == kQuery ? a.qw : KIND == kKey ? a.kw : nullptr;
  const uint8_t* from = k.row + ((long)first * HD + l * E) * L::SIZE;
  float g[E];
  if (w)
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(w + l * E + j));
      g[j] = u.x; g[j + 1] = u.y; g[j + 2] = u.z; g[j + 3] = u.w;
    }
  for (; i0 < i1; i0 += kAhead) {
    uint4 raw[kAhead][L::NV];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = min((i0 + u) * L::HPW + sub, count - 1);   // past the last head: it again, not stored
      const uint4* p = reinterpret_cast<const uint4*>(from + (long)h * (HD * L::SIZE));
#pragma unroll
      for (int v = 0; v < L::NV; ++v) raw[u][v] = __ldg(p + v);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i0 + u >= i1) break;
      const int h = (i0 + u) * L::HPW + sub < count ? (i0 + u) * L::HPW + sub : -1;
      float x[E];
      unpack<DT, HD>(raw[u], x);
      if (KIND != kValue) {
        if (w) {
          float s[E];
#pragma unroll
          for (int j = 0; j < E; j += 2) {
            const float2 v = mul2(make_float2(x[j], x[j + 1]), make_float2(x[j], x[j + 1]));
            s[j] = v.x;
            s[j + 1] = v.y;
          }
#pragma unroll
          for (int n = E; n > 1; n /= 2)
#pragma unroll
            for (int j = 0; j < n / 2; ++j) s[j] = __fadd_rn(s[2 * j], s[2 * j + 1]);
          float ss = s[0];
#pragma unroll
          for (int o = 1; o < L::LPH; o <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
          const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.f / HD), a.eps)));
#pragma unroll
          for (int j = 0; j < E; j += 2) {
            const float2 v = mul2(mul2(make_float2(x[j], x[j + 1]), make_float2(inv, inv)), make_float2(g[j], g[j + 1]));
            x[j] = v.x;
            x[j + 1] = v.y;
          }
        }
#pragma unroll
        for (int j = 0; j < E; j += 2) {
          // x c - y s is x c + y (-s) to the bit. The sums are not packed: ptxas fuses a packed product with a packed
          // sum, their .rn notwithstanding.
          const float2 y = make_float2(__shfl_sync(0xffffffffu, x[j], k.partner), __shfl_sync(0xffffffffu, x[j + 1], k.partner));
          const float2 xc = mul2(make_float2(x[j], x[j + 1]), make_float2(k.c[j], k.c[j + 1]));
          const float2 ys = mul2(y, make_float2(k.s[j], k.s[j + 1]));
          const float2 z = make_float2(__fadd_rn(xc.x, ys.x), __fadd_rn(xc.y, ys.y));
          x[j] = FULL || k.turns ? z.x : x[j];
          x[j + 1] = FULL || k.turns ? z.y : x[j + 1];
        }
        if (!k.in)
#pragma unroll
          for (int j = 0; j < E; ++j) x[j] = k.pos < 0 ? 0.f : __int_as_float(0x7fc00000);
      }
      if (KIND == kQuery || !CACHE) {
        if (h >= 0) store_head<DT, HD>(KIND == kQuery ? a.q_out : a.k_out, (k.t * count + h) * HD + l * E, x);
      } else {
        store_codes<DT, HD>(a, k, h, KIND == kValue, l, x);
      }
    }
  }
}

template <int DT, int HD, bool CACHE, bool FULL>
__global__ void __launch_bounds__(kVecThreads) qk_norm_rope_vec_kernel(RopeArgs a, int split) {
  using L = Lanes<DT, HD>;
  constexpr int E = L::E;
  const int lane = threadIdx.x & 31, l = lane % L::LPH;
  const unsigned warp = blockIdx.x * (kVecThreads / 32) + (threadIdx.x >> 5);
  const unsigned t = warp / (unsigned)split, part = warp - t * (unsigned)split;
  if (t >= (unsigned)a.T) return;
  Token<DT, HD> k;
  k.t = t;
  k.pos = a.positions[t];
  k.in = k.pos >= 0 && k.pos < a.lmax;
  k.row = reinterpret_cast<const uint8_t*>(a.qkv) + t * a.ld * L::SIZE;
  const int hl = a.half / E;                           // lanes of a rotated half
  const bool first = l < hl;
  k.turns = l < 2 * hl;
  k.partner = lane - l + (first ? l + hl : k.turns ? l - hl : l);
#pragma unroll
  for (int j = 0; j < E; ++j) k.c[j] = k.s[j] = 0.f;
  if (k.turns && k.in) {
    const long row = (long)k.pos * a.half + (first ? l : l - hl) * E;
    const float sign = first ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(a.cos + row + j));
      const float4 v = __ldg(reinterpret_cast<const float4*>(a.sin + row + j));
      k.c[j] = u.x; k.c[j + 1] = u.y; k.c[j + 2] = u.z; k.c[j + 3] = u.w;
      k.s[j] = sign * v.x; k.s[j + 1] = sign * v.y; k.s[j + 2] = sign * v.z; k.s[j + 3] = sign * v.w;
    }
  }
  const int iq = (a.NH + L::HPW - 1) / L::HPW, ik = (a.NKV + L::HPW - 1) / L::HPW, steps = iq + (CACHE ? 2 : 1) * ik;
  const int i0 = (int)(part * steps / split), i1 = (int)((part + 1) * steps / split);
  if (i0 < iq) heads<DT, HD, CACHE, FULL, kQuery>(a, k, i0, min(i1, iq));
  if (i1 <= iq) return;
  if (CACHE) {
    const long slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots || !k.in) return;   // not cached
    k.blk = block_of(a, slot, 0, HD);
    k.head_bytes = (long)block_bytes(HD, a.group) << (a.page_shift - 4);
    k.r = (int)(slot & 15);
  }
  if (i0 < iq + ik) heads<DT, HD, CACHE, FULL, kKey>(a, k, max(i0 - iq, 0), min(i1 - iq, ik));
  if (CACHE && i1 > iq + ik) heads<DT, HD, CACHE, FULL, kValue>(a, k, max(i0 - iq - ik, 0), i1 - iq - ik);
}

// The values that slots stand for: a warp takes a token, a lane decodes words of 8 codes into 16 bytes.
template <int HD>
__global__ void __launch_bounds__(kVecThreads) kv4_read_kernel(RopeArgs a, __half* k_out, __half* v_out) {
  constexpr int W = HD / 8;
  const long t = (long)blockIdx.x * (kVecThreads / 32) + (threadIdx.x >> 5);
  if (t >= a.T) return;
  const long slot = a.slots[t];
  const bool in = slot >= 0 && slot < a.num_slots;
  const int r = (int)(slot & 15);
  const uint8_t* blk = in ? block_of(a, slot, 0, HD) : nullptr;
  const long head_bytes = (long)block_bytes(HD, a.group) << (a.page_shift - 4);
#pragma unroll 2
  for (int i = threadIdx.x & 31; i < 2 * a.NKV * W; i += 32) {
    const int h = i / W, w = i % W;
    const bool is_v = h >= a.NKV;
    const int g = is_v ? h - a.NKV : h;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (in) {
      const uint8_t* p = blk + g * head_bytes + (is_v ? code_bytes(HD) + scale_bytes(HD, a.group) : 0);
      const uint32_t code = *reinterpret_cast<const uint32_t*>(p + r * (HD / 2) + 4 * w);
      const __half2 sm = reinterpret_cast<const __half2*>(p + code_bytes(HD))[r * (HD / a.group) + 8 * w / a.group];
      __half2 n[4];                                       // (element j, element j + 4)
      codes_h2(code, n);
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = h2_as_u32(__hfma2(n[j], __low2half2(sm), __high2half2(sm)));
      o = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                     __byte_perm(v[2], v[3], 0x7632));
    }
    reinterpret_cast<uint4*>((is_v ? v_out : k_out) + (t * a.NKV + g) * HD)[w] = o;
  }
}

bool cache_args(const char* who, const void* cache, int num_pages, int NKV, int HD, int page, int group) {
  if (!sizes_ok(NKV, HD, page, group) || num_pages <= 0 || (reinterpret_cast<uintptr_t>(cache) & 15)) {
    set_error("%s: unsupported cache (pages=%d NKV=%d HD=%d page=%d group=%d; HD 64, 128 or 256, page a power of two "
              "16 to 4096, group 32, 64 or 128 and at most HD, 16-byte aligned)", who, num_pages, NKV, HD, page, group);
    return false;
  }
  return true;
}

template <int DT, int HD>
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
  constexpr int SIZE = Lanes<DT, HD>::SIZE, E = Lanes<DT, HD>::E, HPW = Lanes<DT, HD>::HPW;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.q_out) |
                       reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.cos) |
                       reinterpret_cast<uintptr_t>(a.sin) | reinterpret_cast<uintptr_t>(a.qw) |
                       reinterpret_cast<uintptr_t>(a.kw) | (uintptr_t)(a.ld * SIZE);
  if (at % 16 == 0 && a.half % E == 0) {
    const int steps = (a.NH + HPW - 1) / HPW + (a.cache ? 2 : 1) * ((a.NKV + HPW - 1) / HPW);
    // at least 16 warps an SM, as far as there are steps for them
    const int split = (int)max(1L, min((long)steps, 148L * 16 / a.T));
    const long blocks = ((long)a.T * split + kVecThreads / 32 - 1) / (kVecThreads / 32);
    auto kern = a.half * 2 == HD ? (a.cache ? qk_norm_rope_vec_kernel<DT, HD, true, true> : qk_norm_rope_vec_kernel<DT, HD, false, true>)
                                 : (a.cache ? qk_norm_rope_vec_kernel<DT, HD, true, false> : qk_norm_rope_vec_kernel<DT, HD, false, false>);
    kern<<<(unsigned)blocks, kVecThreads, 0, st>>>(a, split);
    return cudaGetLastError();
  }
  const long items = (long)a.T * (a.NH + (a.cache ? 2 * a.NKV : a.NKV));
  qk_norm_rope_kernel<DT, HD><<<(unsigned)((items + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_rope_hd(const RopeArgs& a, int HD, cudaStream_t st) {
  return HD == 64 ? launch_rope<DT, 64>(a, st) : HD == 128 ? launch_rope<DT, 128>(a, st) : launch_rope<DT, 256>(a, st);
}

}  // namespace
}  // namespace ql

using namespace ql;

extern "C" size_t ql_kv4_block_bytes(int HD, int group) {
  return kv4::sizes_ok(1, HD, 16, group) ? (size_t)kv4::block_bytes(HD, group) : 0;
}

extern "C" int ql_qk_norm_rope(const void* qkv, int dtype, long ld, int T, int NH, int NKV, int HD,
                               const int32_t* positions, const float* rope_cos, const float* rope_sin, int lmax, int rot,
                               const float* q_weight, const float* k_weight, float eps, void* q_out, void* k_out,
                               void* cache, int num_pages, int page, int group, const int64_t* slots, void* stream) {
  if (T == 0) return QL_OK;
  const int V = HD / 32;
  if (!qkv || !positions || (rot && (!rope_cos || !rope_sin)) || !q_out || (!cache) == (!k_out) || (cache && !slots) || T < 0 ||
      NH <= 0 || NKV <= 0 || dtype < QL_F32 || dtype > QL_BF16 || (HD != 64 && HD != 128 && HD != 256) ||
      ld < (long)(NH + 2 * NKV) * HD || lmax <= 0 || rot < 0 || rot > HD || rot % (2 * V)) {
    set_error("ql_qk_norm_rope: bad arguments (T=%d NH=%d NKV=%d HD=%d ld=%ld lmax=%d rot=%d dtype=%d; HD 64, 128 or "
              "256, rot a multiple of HD / 16, either a cache with slots or k_out)", T, NH, NKV, HD, ld, lmax, rot, dtype);
    return QL_ERR_ARG;
  }
  if (cache && !cache_args("ql_qk_norm_rope", cache, num_pages, NKV, HD, page, group)) return QL_ERR_ARG;
  RopeArgs a;
  a.qkv = qkv;
  a.ld = ld;
  a.T = T;
  a.NH = NH;
  a.NKV = NKV;
  a.positions = positions;
  a.cos = rope_cos;
  a.sin = rope_sin;
  a.lmax = lmax;
  a.half = rot / 2;
  a.qw = q_weight;
  a.kw = k_weight;
  a.eps = eps;
  a.q_out = q_out;
  a.k_out = k_out;
  a.cache = reinterpret_cast<uint8_t*>(cache);
  a.num_slots = cache ? (long)num_pages * page : 0;
  a.page_shift = cache ? __builtin_ctz((unsigned)page) : 0;
  a.group = group;
  a.slots = slots;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == QL_F32 ? launch_rope_hd<QL_F32>(a, HD, st)
                        : dtype == QL_F16 ? launch_rope_hd<QL_F16>(a, HD, st) : launch_rope_hd<QL_BF16>(a, HD, st);
  return cuda_status(e, "ql_qk_norm_rope launch");
}

extern "C" int ql_kv4_read(const void* cache, int num_pages, int NKV, int HD, int page, int group, const int64_t* slots,
                           int T, void* k_out, void* v_out, void* stream) {
  if (T == 0) return QL_OK;
  if (!cache || !slots || !k_out || !v_out || T < 0 ||
      ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)) {
    set_error("ql_kv4_read: bad arguments (T=%d; outputs 16-byte aligned)", T);
    return QL_ERR_ARG;
  }
  if (!cache_args("ql_kv4_read", cache, num_pages, NKV, HD, page, group)) return QL_ERR_ARG;
  RopeArgs a = {};
  a.T = T;
  a.NKV = NKV;
  a.cache = reinterpret_cast<uint8_t*>(const_cast<void*>(cache));
  a.num_slots = (long)num_pages * page;
  a.page_shift = __builtin_ctz((unsigned)page);
  a.group = group;
  a.slots = slots;
  const unsigned blocks = (unsigned)(((long)T + kVecThreads / 32 - 1) / (kVecThreads / 32));
  const cudaStream_t st = (cudaStream_t)stream;
  __half* k = reinterpret_cast<__half*>(k_out);
  __half* v = reinterpret_cast<__half*>(v_out);
  if (HD == 64) kv4_read_kernel<64><<<blocks, kVecThreads, 0, st>>>(a, k, v);
  else if (HD == 128) kv4_read_kernel<128><<<blocks, kVecThreads, 0, st>>>(a, k, v);
  else kv4_read_kernel<256><<<blocks, kVecThreads, 0, st>>>(a, k, v);
  return cuda_status(cudaGetLastError(), "ql_kv4_read launch");
}
