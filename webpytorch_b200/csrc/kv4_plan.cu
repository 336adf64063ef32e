// Block tables and slot maps of a serving step, built on the GPU from request lengths.
//
// Request b holds ceil(prev_b / page) pages and asks for new_b tokens, or ends (new_b < 0) and gives
// its pages back. First come first served: with need_b = ceil((prev_b + new_b) / page) - held_b,
//   served_b  iff  sum_{c <= b} new_c <= max_tokens  and  (need_b = 0 or sum_{c <= b} need_c <= avail),
// sums over the requests that fit their table row, avail = free pages + pages given back. Both sums
// grow with b, so the served requests that need pages are the first ones that do, and the pages
// taken are a contiguous piece of the stack, from its top.
//
// The work is a launch and two dependent block scans; the bytes (4.3 MB of maps at 262144 tokens) are under a
// microsecond. 8 requests take 5 us, 1000 with 20000 tokens 9, 6000 with 262144 tokens 18 (lengths staged in
// shared memory first: the same).
#include "ql_common.cuh"

namespace ql {
namespace {

constexpr int kThreads = 1024;
// Requests whose sums fit in shared memory (16384 requests 68 us there, 16385 in the workspace 79).
constexpr int kMost = 16384;

struct PlanArgs {
  const int32_t* prev;
  const int32_t* fresh;   // new tokens of each request, negative: the request ends
  int32_t* table;
  long table_stride;
  int n, width;
  int32_t* free_pages;
  int free_capacity;
  const int32_t* n_free_in;
  int page_shift, max_tokens;
  int32_t* seq_lens;
  int32_t* cu_new;
  int64_t* slots;
  int32_t* positions;
  int32_t* requests;
  int32_t* n_free_out;
  int32_t* sums;          // workspace for more than kMost requests: three arrays of n + 1
};

struct Request {
  int back, need;
  long long tok;
  int len;
  bool fits, over;
};

__device__ __forceinline__ int pages_of(long long len, int shift) {
  return (int)((len + (1ll << shift) - 1) >> shift);
}

__device__ __forceinline__ Request load_request(const PlanArgs& a, int b) {
  Request r = {};
  const long long prev = max(a.prev[b], 0);
  const long long fresh = a.fresh[b];
  r.len = (int)prev;
  const int held = pages_of(prev, a.page_shift);
  r.over = fresh < 0;
  if (r.over) {
    r.back = min(held, a.width);
  } else {
    const int pages = pages_of(prev + fresh, a.page_shift);
    r.fits = pages <= a.width;
    if (r.fits) {
      r.need = pages - held;
      r.tok = fresh;
    }
  }
  return r;
}

// Sums over the threads before this one, and over all of them.
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long (&total)[N], long long (*warps)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    incl[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, incl[k], o);
      if (lane >= o) incl[k] += u;
    }
  }
  __syncthreads();
  if (lane == 31)
#pragma unroll
    for (int k = 0; k < N; ++k) warps[warp][k] = incl[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const long long own = warps[lane][k];      // kThreads / 32 = 32 warps
    long long all = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, all, o);
      if (lane >= o) all += u;
    }
    total[k] = __shfl_sync(0xffffffffu, all, 31);
    v[k] = incl[k] - v[k] + __shfl_sync(0xffffffffu, all - own, warp);
  }
}

// The first b with end[b] > i.
__device__ __forceinline__ int find(const int32_t* end, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (end[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Entry i of the stack of free pages after the returned ones are pushed. The pushes are made by
// other threads of the same launch, so entries above the old top come from the rows they leave.
__device__ __forceinline__ int32_t stack_entry(const PlanArgs& a, const int32_t* back_end, int n_free, int i) {
  if (i < n_free) return a.free_pages[i];
  const int k = i - n_free;
  const int b = find(back_end, a.n, k);
  return a.table[b * a.table_stride + k - (b ? back_end[b - 1] : 0)];
}

// Every CTA sums over all requests (8 bytes a request from L2, two block scans), so that one launch does
// without any exchange between CTAs, then writes its share of the tokens and pages. SHARED: the sums are in
// its shared memory, where the binary searches run; for more requests than fit, in a workspace that every
// CTA fills alike.
template <bool SHARED>
__global__ void __launch_bounds__(kThreads) plan_kernel(PlanArgs a) {
  extern __shared__ int32_t shared_sums[];
  __shared__ long long warps3[kThreads / 32][3], warps2[kThreads / 32][2];
  int32_t* cu = SHARED ? shared_sums : a.sums + (long)blockIdx.x * 3 * (a.n + 1);
  int32_t* need_end = cu + a.n + 1;       // inclusive sums of pages taken
  int32_t* back_end = need_end + a.n;     // and of pages given back
  const int tid = threadIdx.x;
  const int each = (a.n + kThreads - 1) / kThreads, b0 = min(tid * each, a.n), b1 = min(b0 + each, a.n);
  long long v[3] = {}, all[3];
  for (int b = b0; b < b1; ++b) {
    const Request r = load_request(a, b);
    v[0] += r.back;
    v[1] += r.need;
    v[2] += r.tok;
  }
  block_scan<3>(v, all, warps3);
  const int n_free = min(max(*a.n_free_in, 0), a.free_capacity);
  const int avail = (int)min(n_free + all[0], (long long)a.free_capacity);
  long long w[2] = {}, sums[2];
  {
    long long need = v[1], tok = v[2];
    for (int b = b0; b < b1; ++b) {
      const Request r = load_request(a, b);
      need += r.need;
      tok += r.tok;
      if (r.fits && tok <= a.max_tokens && (r.need == 0 || need <= avail)) {
        w[0] += r.tok;
        w[1] += r.need;
      }
    }
  }
  block_scan<2>(w, sums, warps2);
  const int total = (int)sums[0], taken = (int)sums[1];
  for (int b = b0; b < b1; ++b) {
    const Request r = load_request(a, b);
    v[0] += r.back;
    v[1] += r.need;
    v[2] += r.tok;
    const bool served = r.fits && v[2] <= a.max_tokens && (r.need == 0 || v[1] <= avail);
    cu[b] = (int32_t)w[0];
    if (blockIdx.x == 0) {
      a.cu_new[b] = (int32_t)w[0];
      a.seq_lens[b] = r.over ? 0 : r.len + (served ? (int)r.tok : 0);
    }
    if (served) {
      w[0] += r.tok;
      w[1] += r.need;
    }
    need_end[b] = (int32_t)w[1];
    back_end[b] = (int32_t)v[0];
  }
  if (tid == 0) {
    cu[a.n] = total;
    if (blockIdx.x == 0) {
      a.cu_new[a.n] = total;
      a.n_free_out[0] = avail - taken;
    }
  }
  __syncthreads();

  const int t0 = blockIdx.x * kThreads + tid, step = gridDim.x * kThreads, page = 1 << a.page_shift;
  for (int t = t0; t < a.max_tokens; t += step) {
    int64_t slot = -1;
    int pos = -1, b = -1;
    if (t < total) {
      b = find(cu + 1, a.n, t);
      const int prev = max(a.prev[b], 0);
      const int held = pages_of(prev, a.page_shift);
      pos = prev + t - cu[b];
      const int i = pos >> a.page_shift;
      const int32_t p = i < held ? a.table[b * a.table_stride + i]
                                 : stack_entry(a, back_end, n_free, avail - 1 - ((b ? need_end[b - 1] : 0) + i - held));
      slot = (int64_t)p * page + (pos & (page - 1));
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.requests[t] = b;
  }
  for (int k = t0; k < taken; k += step) {   // pages taken: table entries past the held ones
    const int b = find(need_end, a.n, k);
    const int held = pages_of(max(a.prev[b], 0), a.page_shift);
    a.table[b * a.table_stride + held + k - (b ? need_end[b - 1] : 0)] = stack_entry(a, back_end, n_free, avail - 1 - k);
  }
  for (int k = n_free + t0; k < avail; k += step)   // pages given back
    a.free_pages[k] = stack_entry(a, back_end, n_free, k);
}

int ctas_for(int n, int max_tokens) {
  return max(1, min(n <= kMost ? 148 : 16, (max(max_tokens, n) + kThreads - 1) / kThreads));
}

}  // namespace
}  // namespace ql

using namespace ql;

extern "C" size_t ql_kv_plan_workspace(int n) {
  return n <= kMost ? 0 : (size_t)16 * 3 * (n + 1) * sizeof(int32_t);
}

extern "C" int ql_kv_plan(const int32_t* prev_lens, const int32_t* new_lens, int n, int32_t* table, long table_stride,
                          int table_width, int32_t* free_pages, int free_capacity, const int32_t* n_free, int page,
                          int max_tokens, int32_t* seq_lens, int32_t* cu_new, int64_t* slots, int32_t* positions,
                          int32_t* requests, int32_t* n_free_out, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (!prev_lens || !new_lens || !table || !free_pages || !n_free || !seq_lens || !cu_new || !n_free_out || n <= 0 ||
      table_width <= 0 || table_stride < table_width || free_capacity <= 0 || max_tokens < 0 ||
      (max_tokens > 0 && (!slots || !positions || !requests)) || page < 16 || page > 4096 || (page & (page - 1))) {
    set_error("ql_kv_plan: bad arguments (n=%d width=%d stride=%ld capacity=%d max_tokens=%d page=%d; page a power of "
              "two, 16 to 4096)", n, table_width, table_stride, free_capacity, max_tokens, page);
    return QL_ERR_ARG;
  }
  if ((long)table_width * page > INT32_MAX || (long)n * table_width > INT32_MAX) {
    set_error("ql_kv_plan: a row of %d pages of %d tokens, or %d rows of it, is past 32 bits", table_width, page, n);
    return QL_ERR_UNSUPPORTED;
  }
  if (prev_lens == seq_lens || n_free == n_free_out) {
    set_error("ql_kv_plan: seq_lens and n_free_out may not be prev_lens and n_free");
    return QL_ERR_ARG;
  }
  if (ql_kv_plan_workspace(n) > 0 && (!workspace || workspace_bytes < ql_kv_plan_workspace(n))) {
    set_error("ql_kv_plan: workspace of %zu bytes needed", ql_kv_plan_workspace(n));
    return QL_ERR_ARG;
  }
  PlanArgs a;
  a.prev = prev_lens;
  a.fresh = new_lens;
  a.table = table;
  a.table_stride = table_stride;
  a.n = n;
  a.width = table_width;
  a.free_pages = free_pages;
  a.free_capacity = free_capacity;
  a.n_free_in = n_free;
  a.page_shift = __builtin_ctz((unsigned)page);
  a.max_tokens = max_tokens;
  a.seq_lens = seq_lens;
  a.cu_new = cu_new;
  a.slots = slots;
  a.positions = positions;
  a.requests = requests;
  a.n_free_out = n_free_out;
  a.sums = reinterpret_cast<int32_t*>(workspace);
  const cudaStream_t st = (cudaStream_t)stream;
  const int ctas = ctas_for(n, max_tokens);
  if (n > kMost) {
    plan_kernel<false><<<ctas, kThreads, 0, st>>>(a);
  } else {
    static int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
      const int rc = cuda_status(cudaFuncSetAttribute(plan_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                      3 * (kMost + 1) * (int)sizeof(int32_t)),
                                 "cudaFuncSetAttribute(plan smem)");
      if (rc) return rc;
      configured_dev = dev;
    }
    plan_kernel<true><<<ctas, kThreads, 3 * (size_t)(n + 1) * sizeof(int32_t), st>>>(a);
  }
  return cuda_status(cudaGetLastError(), "ql_kv_plan launch");
}
