// Block tables and slot maps of a serving step, built on the GPU from request lengths.
//
// Request b holds ceil(prev_b / page) pages and asks for new_b tokens, or ends (new_b < 0) and gives
// its pages back. First come first served: with need_b = ceil((prev_b + new_b) / page) - held_b,
//   served_b  iff  sum_{c <= b} new_c <= max_tokens  and  (need_b = 0 or sum_{c <= b} need_c <= avail),
// sums over the requests that fit their table row, avail = free pages + pages given back. Both sums
// grow with b, so the served requests that need pages are the first ones that do, and the pages
// taken are a contiguous piece of the stack, from its top.
#include "ql_common.cuh"

namespace ql {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kFillThreads = 256;

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
  int32_t* need_end;   // [n] workspace: inclusive sums of pages taken
  int32_t* back_end;   // [n] workspace: inclusive sums of pages given back
  int32_t* totals;     // [2] workspace: avail, pages taken
};

struct Request {
  long long back, need, tok;
  bool fits, over;
};

__device__ __forceinline__ int pages_of(long long len, int shift) {
  return (int)((len + (1ll << shift) - 1) >> shift);
}

__device__ __forceinline__ Request load_request(const PlanArgs& a, int b) {
  Request r = {0, 0, 0, false, false};
  if (b >= a.n) return r;
  const long long prev = max(a.prev[b], 0);
  const long long fresh = a.fresh[b];
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

// Inclusive sum over the block; *total receives the block's sum.
__device__ __forceinline__ long long block_scan(long long v, long long* warps, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  long long before = 0, all = 0;
  for (int w = 0; w < kScanThreads / 32; ++w) {
    const long long x = warps[w];
    if (w < warp) before += x;
    all += x;
  }
  *total = all;
  return v + before;
}

__global__ void __launch_bounds__(kScanThreads) plan_scan_kernel(PlanArgs a) {
  __shared__ long long warps[kScanThreads / 32];
  const int tid = threadIdx.x;
  long long total, back_all = 0;
  for (int b0 = 0; b0 < a.n; b0 += kScanThreads) {
    const Request r = load_request(a, b0 + tid);
    const long long end = back_all + block_scan(r.back, warps, &total);
    if (b0 + tid < a.n) a.back_end[b0 + tid] = (int32_t)min(end, (long long)INT32_MAX);
    back_all += total;
  }
  const long long n_free = min(max(*a.n_free_in, 0), a.free_capacity);
  const long long avail = min(n_free + back_all, (long long)a.free_capacity);
  long long need0 = 0, tok0 = 0, put0 = 0, taken = 0;
  for (int b0 = 0; b0 < a.n; b0 += kScanThreads) {
    const int b = b0 + tid;
    const Request r = load_request(a, b);
    const long long need_end = need0 + block_scan(r.need, warps, &total);
    need0 += total;
    const long long tok_end = tok0 + block_scan(r.tok, warps, &total);
    tok0 += total;
    const bool served = r.fits && tok_end <= a.max_tokens && (r.need == 0 || need_end <= avail);
    const long long put = served ? r.tok : 0;
    const long long put_end = put0 + block_scan(put, warps, &total);
    put0 += total;
    const long long taken_end = taken + block_scan(served ? r.need : 0, warps, &total);
    taken += total;
    if (b < a.n) {
      a.cu_new[b] = (int32_t)(put_end - put);
      a.seq_lens[b] = r.over ? 0 : max(a.prev[b], 0) + (int32_t)put;
      a.need_end[b] = (int32_t)taken_end;
    }
  }
  if (tid == 0) {
    a.cu_new[a.n] = (int32_t)put0;
    a.n_free_out[0] = (int32_t)(avail - taken);
    a.totals[0] = (int32_t)avail;
    a.totals[1] = (int32_t)taken;
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
__device__ __forceinline__ int32_t stack_entry(const PlanArgs& a, int n_free, int i) {
  if (i < n_free) return a.free_pages[i];
  const int k = i - n_free;
  const int b = find(a.back_end, a.n, k);
  return a.table[b * a.table_stride + k - (b ? a.back_end[b - 1] : 0)];
}

__global__ void __launch_bounds__(kFillThreads) plan_fill_kernel(PlanArgs a) {
  const int t0 = blockIdx.x * kFillThreads + threadIdx.x, step = gridDim.x * kFillThreads;
  const int n_free = min(max(*a.n_free_in, 0), a.free_capacity);
  const int avail = a.totals[0], taken = a.totals[1], total = a.cu_new[a.n];
  const int page = 1 << a.page_shift;
  for (int t = t0; t < a.max_tokens; t += step) {
    int64_t slot = -1;
    int pos = -1, b = -1;
    if (t < total) {
      b = find(a.cu_new + 1, a.n, t);
      const int prev = max(a.prev[b], 0);
      const int held = pages_of(prev, a.page_shift);
      pos = prev + t - a.cu_new[b];
      const int i = pos >> a.page_shift;
      const int32_t p = i < held ? a.table[b * a.table_stride + i]
                                 : stack_entry(a, n_free, avail - 1 - ((b ? a.need_end[b - 1] : 0) + i - held));
      slot = (int64_t)p * page + (pos & (page - 1));
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.requests[t] = b;
  }
  for (int k = t0; k < taken; k += step) {   // pages taken: table entries past the held ones
    const int b = find(a.need_end, a.n, k);
    const int held = pages_of(max(a.prev[b], 0), a.page_shift);
    a.table[b * a.table_stride + held + k - (b ? a.need_end[b - 1] : 0)] = stack_entry(a, n_free, avail - 1 - k);
  }
  for (int k = n_free + t0; k < avail; k += step)   // pages given back
    a.free_pages[k] = stack_entry(a, n_free, k);
}

}  // namespace
}  // namespace ql

using namespace ql;

extern "C" size_t ql_kv_plan_workspace(int n) { return n <= 0 ? 0 : ((size_t)2 * n + 2) * sizeof(int32_t); }

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
  if (!workspace || workspace_bytes < ql_kv_plan_workspace(n)) {
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
  a.need_end = reinterpret_cast<int32_t*>(workspace);
  a.back_end = a.need_end + n;
  a.totals = a.back_end + n;
  const cudaStream_t st = (cudaStream_t)stream;
  plan_scan_kernel<<<1, kScanThreads, 0, st>>>(a);
  const int blocks = max(1, min(148 * 8, (max(max_tokens, n) + kFillThreads - 1) / kFillThreads));
  plan_fill_kernel<<<blocks, kFillThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError(), "ql_kv_plan launch");
}
