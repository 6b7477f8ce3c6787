// 8-bit paged key/value cache: append, gather, attention over the cache, page copies.
//
// Layout of one layer's cache (K and V alike): e4m3 codes [pages, heads, page_size, d] and fp32 scales
// [pages, heads, page_size / 16]: every 16 tokens of a head share a power-of-two scale.  Head-major pages keep the 16 x d
// codes of a block contiguous, which is what one warp of every kernel here reads or writes.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace teb200 {

constexpr int kKvBlock = 16;         // tokens that share a scale
constexpr int kKvStatusPages = 31;   // status code: page table, lengths and cache do not fit each other

struct Fp8CacheView {
  uint8_t* k = nullptr;
  uint8_t* v = nullptr;
  float* k_scale = nullptr;
  float* v_scale = nullptr;
  int pages = 0, heads = 0, page_size = 0, d = 0;
  const int* table = nullptr;  // [n, width] page of every page_size tokens, negative: not held
  int width = 0;
  int n = 0;                   // sequences
  const int* kv_lens = nullptr;  // [n] tokens held (the new ones included)
  int* status = nullptr;
};

struct Fp8AppendArgs {
  Fp8CacheView c;
  const void* new_k = nullptr;  // [t, heads, d] views, element strides below, d contiguous
  const void* new_v = nullptr;
  long long k_st = 0, k_sh = 0, v_st = 0, v_sh = 0;
  const int* cu_new = nullptr;  // [n + 1]
  int t = 0;
  int dtype = 0;                // DType of new_k / new_v
  int max_new = 0;              // longest run of new tokens (sizes the grid, longer runs are handled)
};
cudaError_t fp8_cache_append(const Fp8AppendArgs& a, cudaStream_t stream);

struct Fp8GatherArgs {
  Fp8CacheView c;
  void* out_k = nullptr;        // [rows, heads, d] contiguous
  void* out_v = nullptr;
  const int* off = nullptr;     // [n] first row of every sequence (nullptr: expansion, below)
  int rows = 0;
  int max_kv = 0;               // longest sequence (sizes the grid, longer ones are handled; an expansion cuts them there)
  int dtype = 0;
  // Expansion for the packed attention kernel: sequence i starts at row i * pitch and is followed by zeros up to the next
  // multiple of 128 rows; 128-row blocks that no query of the step sees are left out.  The launch also writes what that
  // kernel needs beside it: cumulative lengths and first rows of keys and queries, cut to what the buffers hold (that
  // kernel does not check them), and zeros in the output rows that no query claims.
  int pitch = 0;
  const int* cu_q = nullptr;    // [n + 1]
  int max_q = 0;
  int window_left = -1, sinks = 0;
  int* cu_k = nullptr;          // [n + 1]
  int* first_row = nullptr;     // [n + 1]
  int* cut_q = nullptr;         // [n + 1] cumulative queries
  int* first_q = nullptr;       // [n + 1]
  void* out = nullptr;          // [tq, row_bytes]
  int tq = 0;
  bool last = true;             // the rows of `out` behind the last sequence are nobody's
  long long row_bytes = 0;      // multiple of 4
};
cudaError_t fp8_cache_gather(const Fp8GatherArgs& a, cudaStream_t stream);

struct Fp8AttendArgs {
  Fp8CacheView c;
  const void* q = nullptr;      // [tq, hq, d] view, d contiguous
  long long q_st = 0, q_sh = 0;
  void* out = nullptr;          // [tq, hq, d] contiguous
  const int* cu_q = nullptr;    // [n + 1]
  int tq = 0, hq = 0;
  int is_bf16 = 1;
  int max_q = 0, max_kv = 0;
  int causal = 1, window_left = -1, sinks = 0;
  float scale = 1.f;
  float* part = nullptr;        // workspace of fp8_attend_workspace() floats, nullptr if that is 0
};
long long fp8_attend_workspace(const Fp8AttendArgs& a);
cudaError_t fp8_attend(const Fp8AttendArgs& a, cudaStream_t stream);

struct PageCopyTensor {
  void* base;
  long long page_bytes;
};
// pages[dst[i]] = pages[src[i]] of every tensor; src / dst are HOST arrays (they travel in the launch parameters), every
// id is below the tensors' page count, no page is written twice and none that is written is read.
cudaError_t copy_pages(const PageCopyTensor* tensors, int num_tensors, const int* src, const int* dst, int pairs,
                       cudaStream_t stream);

}  // namespace teb200
