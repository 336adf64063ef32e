// What the two attention kernels over the paged 4-bit cache share: the call's arguments, and the lookup and
// copy of a block.
#pragma once

#include "kv4_common.cuh"
#include "sm100_ptx.cuh"

namespace ql {
namespace kv4 {

struct AttnArgs {
  const void* q;
  long ldq;
  int T, NH, NKV;
  const uint8_t* cache;
  int num_pages, page_shift;
  const int32_t* table;
  long table_stride;
  int width;
  const int32_t* seq_lens;
  const int32_t* cu_q;
  int B;
  float scale;
  int window;
  int prompt_rows;          // requests of so many rows or more are the prompt kernel's
  void* out;
  unsigned int* counters;   // [kMaxCtas], zero between launches
  float* parts;             // [ctas][2 + warps] partial results
};

__device__ __forceinline__ int cu(const AttnArgs& a, int b) { return a.cu_q ? min(max(a.cu_q[b], 0), a.T) : min(b, a.T); }

// A wait by a whole warp. The lanes leave the polling loop at different times, and one may give up on what another
// still saw complete: the vote brings the warp together, as the tensor-core instructions that follow want it, and
// makes the answer the same for all lanes.
template <bool SLEEP = false>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, SLEEP ? ptx::mbar_wait_sleep(bar, parity, abort_flag) : ptx::mbar_wait(bar, parity, abort_flag));
}

constexpr uint32_t kNoBlock = 0xffffffffu;

// Block i of n from blk0 of request b, as its index in the cache; kNoBlock past the end or for a page
// that is not one of the cache's.
__device__ __forceinline__ uint32_t source(const AttnArgs& a, int b, int kvh, int blk0, int i, int n) {
  const int shift = a.page_shift - 4;
  if (i >= n) return kNoBlock;
  const int page = a.table[b * a.table_stride + ((blk0 + i) >> shift)];
  if (page < 0 || page >= a.num_pages) return kNoBlock;
  return (((uint32_t)page * a.NKV + kvh) << shift) + ((blk0 + i) & ((1 << shift) - 1));
}

// A lane's block into a stage of the ring.
template <int BB>
__device__ __forceinline__ void issue(const AttnArgs& a, uint32_t src, int stage, uint32_t ring, uint32_t bar) {
  if (src != kNoBlock) {
    ptx::mbar_arrive_expect_tx(bar + 8 * stage, BB);
    ptx::bulk_load(ring + stage * BB, a.cache + (size_t)src * BB, BB, bar + 8 * stage);
  } else {
    ptx::mbar_arrive(bar + 8 * stage);
  }
}

}  // namespace kv4

// Requests of kPromptRows rows or more, 16-bit types, HD 64 or 128 (kv4_prompt.cu).
// Calls of few rows leave parts in a.parts, kv4_prompt_bytes of it, for a GPU of `ctas` SMs.
int kv4_prompt_attention(const kv4::AttnArgs& a, int dtype, int HD, int group, int ctas, cudaStream_t st);
size_t kv4_prompt_bytes(int HD, int ctas);
int take_kv4_prompt_status();

}  // namespace ql
