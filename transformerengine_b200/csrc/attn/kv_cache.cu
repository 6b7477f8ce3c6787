// 8-bit paged key/value cache: quantizing append, dequantizing gather, page copies.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "fp8_cache.cuh"
#include "teb200/api.h"
#include "teb200/kv_cache.h"

namespace teb200 {
namespace {

using namespace kvc;

// 8 consecutive values of a row, as they are loaded and as fp32
template <typename T>
struct Raw8 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  // larger of `top` and the magnitudes' bits, two 16-bit numbers at a time (their order is that of the values)
  __device__ __forceinline__ uint32_t top_bits(uint32_t top) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
    return top;
  }
  static __device__ __forceinline__ bool finite(uint32_t top) {
    constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    return (top & 0xffffu) < kInf && (top >> 16) < kInf;
  }
  static __device__ __forceinline__ float value(uint32_t top) {
    const uint16_t b = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    return std::is_same<T, __nv_bfloat16>::value ? __uint_as_float(static_cast<uint32_t>(b) << 16) : __half2float(__ushort_as_half(b));
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ uint32_t top_bits(uint32_t top) const {
    float x[8];
    get(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    return top;
  }
  static __device__ __forceinline__ bool finite(uint32_t top) { return top < 0x7f800000u; }
  static __device__ __forceinline__ float value(uint32_t top) { return __uint_as_float(top); }
};

// One warp per (sequence, 16-token block, K or V, head); the four warps of a CTA take neighbouring heads, whose rows
// adjoin in memory.  A lane owns 8 consecutive dims of the rows lane / (d / 8), + 32 / (d / 8), ...  The block's largest
// finite magnitude sets the scale, and rows that were there before are rounded again when it rises.  A power-of-two scale
// makes that second rounding exact except where a code becomes subnormal.  Reading 16-bit rows and writing codes bounds
// long runs (29000 tokens of 8 heads, d 128: 178 MB in 38 us); a single token per sequence is one chain of dependent loads
// (lengths, then page and row, then scale: 4.3 us).
template <typename T, int D>
__global__ void __launch_bounds__(128, D == 256 ? (sizeof(T) == 4 ? 2 : 4) : (sizeof(T) == 4 ? 4 : 8)) append_kernel(const Fp8AppendArgs a) {
  constexpr int kLanesPerRow = D / 8;
  constexpr int kRows = 32 / kLanesPerRow;   // rows per pass
  constexpr int kPasses = kKvBlock / kRows;
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= 2 * a.c.heads) return;
  const bool is_v = unit >= a.c.heads;
  const int head = is_v ? unit - a.c.heads : unit;
  const int seq = blockIdx.z;
  const int per = a.c.page_size / kKvBlock;
  const int src0 = a.cu_new[seq];
  const int n_new = a.cu_new[seq + 1] - src0;
  const int len = a.c.kv_lens[seq];
  const int old = len - n_new;
  if (n_new <= 0) return;
  if (old < 0 || src0 < 0 || src0 + n_new > a.t) {
    if (lane == 0) atomicCAS(a.c.status, 0, kKvStatusPages);
    return;
  }
  const T* src = static_cast<const T*>(is_v ? a.new_v : a.new_k) + head * (is_v ? a.v_sh : a.k_sh) +
                 (lane % kLanesPerRow) * 8;
  const long long st = is_v ? a.v_st : a.k_st;
  for (int blk = old / kKvBlock + blockIdx.y; blk * kKvBlock < len; blk += gridDim.y) {
    const int slot = blk / per;
    const int page = slot < a.c.width ? a.c.table[static_cast<long long>(seq) * a.c.width + slot] : -1;
    const int first = max(old - blk * kKvBlock, 0);             // rows [first, end) are new
    const int end = min(len - blk * kKvBlock, kKvBlock);
    const T* rows = src + (src0 + blk * kKvBlock - old) * st;
    Raw8<T> raw[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int r = p * kRows + lane / kLanesPerRow;
      if (r >= first && r < end) raw[p].load(rows + r * st);
    }
    if (page < 0 || page >= a.c.pages) {
      if (lane == 0) atomicCAS(a.c.status, 0, kKvStatusPages);
      continue;
    }
    const long long idx = (static_cast<long long>(page) * a.c.heads + head) * per + blk % per;
    uint8_t* codes = (is_v ? a.c.v : a.c.k) + idx * (kKvBlock * D) + lane * 8;
    float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + idx;
    float was = first > 0 ? *scale : 0.f;
    uint32_t bits = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int r = p * kRows + lane / kLanesPerRow;
      if (r >= first && r < end) bits = raw[p].top_bits(bits);
    }
    float top = Raw8<T>::value(bits);
    if (!Raw8<T>::finite(bits)) {
      // NaN and infinities do not set the scale: once more, without them
      top = 0.f;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int r = p * kRows + lane / kLanesPerRow;
        if (r >= first && r < end) {
          float x[8];
          raw[p].get(x);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (fabsf(x[i]) < INFINITY) top = fmaxf(top, fabsf(x[i]));
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float now = fmaxf(scale_for(top), was);
    if (first == 0) was = now;
    const float inv = inverse_of_power(now);
    const float again = was * inv;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int r = p * kRows + lane / kLanesPerRow;
      uint2* dst = reinterpret_cast<uint2*>(codes + p * 256);
      if (r >= first && r < end) {
        float x[8];
        raw[p].get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= inv;
        *dst = make_uint2(to_e4m3x4(x[0], x[1], x[2], x[3]), to_e4m3x4(x[4], x[5], x[6], x[7]));
      } else if (r < first && now != was) {
        const uint2 old8 = *dst;
        float y[8];
        from_e4m3x4(old8.x, y);
        from_e4m3x4(old8.y, y + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= again;
        *dst = make_uint2(to_e4m3x4(y[0], y[1], y[2], y[3]), to_e4m3x4(y[4], y[5], y[6], y[7]));
      }
    }
    if (lane == 0) *scale = now;   // every lane has read it: the maximum above is a warp-wide exchange
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&y)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&y)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(y[4], y[5], y[6], y[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&y)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<true>(y[0], y[1]), pack2<true>(y[2], y[3]), pack2<true>(y[4], y[5]),
                                            pack2<true>(y[6], y[7]));
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const float (&y)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<false>(y[0], y[1]), pack2<false>(y[2], y[3]),
                                            pack2<false>(y[4], y[5]), pack2<false>(y[6], y[7]));
}

// What the packed attention kernel needs beside the expanded keys and values (CTA 0), and zeros in the rows without a query.
__device__ __forceinline__ void expansion_extras(const Fp8GatherArgs& a) {
  const long long cta = (static_cast<long long>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const long long ctas = static_cast<long long>(gridDim.x) * gridDim.y * gridDim.z;
  zero_unclaimed(static_cast<uint32_t*>(a.out), a.row_bytes / 4, a.cu_q, a.c.n, a.tq, a.max_q, a.last, cta, ctas);
  if (cta != 0 || threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  int base = 0, base_q = 0;
  if (lane == 0) a.cu_k[0] = a.cut_q[0] = 0;
  for (int i0 = 0; i0 <= a.c.n; i0 += 32) {
    const int i = i0 + lane;
    SeqFit f = {0, 0, 0, false};
    if (i < a.c.n) f = fit_sequence(a.cu_q, a.c.kv_lens, i, a.tq, a.max_q, a.max_kv);
    if (f.bad) atomicCAS(a.c.status, 0, kKvStatusPages);
    int x = f.len, q = f.qlen;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o), z = __shfl_up_sync(0xffffffffu, q, o);
      if (lane >= o) {
        x += y;
        q += z;
      }
    }
    if (i < a.c.n) {
      a.cu_k[i + 1] = base + x;
      a.cut_q[i + 1] = base_q + q;
    }
    if (i <= a.c.n) {
      a.first_row[i] = i * a.pitch;
      a.first_q[i] = f.q_row0;
    }
    base += __shfl_sync(0xffffffffu, x, 31);
    base_q += __shfl_sync(0xffffffffu, q, 31);
  }
}

// One warp per (sequence, 16-token block, K or V, head): codes * scale into a token-major buffer.  Blocks whose page is
// not held, and the rows from a sequence's end to the next multiple of 128 (expansion), become zeros.  An expansion reports
// pages that are not held where a query sees them, as attention in place does.
template <typename T, int D>
__global__ void __launch_bounds__(128) gather_kernel(const Fp8GatherArgs a) {
  constexpr int kLanesPerRow = D / 8;
  constexpr int kRows = 32 / kLanesPerRow;
  constexpr int kPasses = kKvBlock / kRows;
  const int lane = threadIdx.x & 31;
  if (a.off == nullptr) expansion_extras(a);
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= 2 * a.c.heads) return;
  const bool is_v = unit >= a.c.heads;
  const int head = is_v ? unit - a.c.heads : unit;
  const int seq = blockIdx.z;
  const int per = a.c.page_size / kKvBlock;
  int len, first_q = 0;
  if (a.off != nullptr) {
    len = a.c.kv_lens[seq];
  } else {
    const SeqFit f = fit_sequence(a.cu_q, a.c.kv_lens, seq, a.tq, a.max_q, a.max_kv);
    len = f.len;                // a longer sequence is cut, as where the codes are read in place
    first_q = f.len - f.qlen;
    if (f.qlen == 0) len = 0;   // nobody looks
  }
  const int off = a.off != nullptr ? a.off[seq] : seq * a.pitch;
  const int stop = a.off == nullptr ? (len + 127) / 128 * 128 : len;
  if (len < 0 || off < 0 || stop > (a.off == nullptr ? a.pitch : a.rows - off)) {   // (never in an expansion)
    if (lane == 0) atomicCAS(a.c.status, 0, kKvStatusPages);
    return;
  }
  int unseen_from = 0, unseen_to = 0;   // rows that nobody looks at
  int seen_from = 0;                    // first row in a window
  if (a.off == nullptr && a.window_left >= 0) {
    seen_from = max(first_q - a.window_left, 0);
    unseen_to = seen_from / 128 * 128;
    unseen_from = min(a.sinks, 0x7fffff00) / 128 * 128 + (a.sinks % 128 != 0 ? 128 : 0);
  }
  T* out = static_cast<T*>(is_v ? a.out_v : a.out_k) + static_cast<long long>(off) * a.c.heads * D + head * D +
           (lane % kLanesPerRow) * 8;
  for (int blk = blockIdx.y; blk * kKvBlock < stop; blk += gridDim.y) {
    if (blk * kKvBlock >= unseen_from && blk * kKvBlock < unseen_to) continue;
    const int slot = blk / per;
    int page = -1;
    if (blk * kKvBlock < len) {
      page = slot < a.c.width ? a.c.table[static_cast<long long>(seq) * a.c.width + slot] : a.c.pages;
      const bool wanted = blk * kKvBlock + kKvBlock > seen_from || blk * kKvBlock < a.sinks;   // by the step's queries
      if (a.off != nullptr ? page >= a.c.pages : wanted && (page < 0 || page >= a.c.pages)) {
        if (lane == 0) atomicCAS(a.c.status, 0, kKvStatusPages);
      }
      if (page >= a.c.pages) page = -1;
    }
    const long long idx = page < 0 ? 0 : (static_cast<long long>(page) * a.c.heads + head) * per + blk % per;
    const uint8_t* codes = (is_v ? a.c.v : a.c.k) + idx * (kKvBlock * D) + lane * 8;
    const float scale = page < 0 ? 0.f : (is_v ? a.c.v_scale : a.c.k_scale)[idx];
    uint2 w[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = blk * kKvBlock + p * kRows + lane / kLanesPerRow;
      w[p] = make_uint2(0u, 0u);
      if (page >= 0 && row < len) w[p] = *reinterpret_cast<const uint2*>(codes + p * 256);
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = blk * kKvBlock + p * kRows + lane / kLanesPerRow;
      if (row >= stop) continue;
      float y[8];
      from_e4m3x4(w[p].x, y);
      from_e4m3x4(w[p].y, y + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = w[p].x == 0u && w[p].y == 0u ? 0.f : y[i] * scale;
      store8<T>(out + static_cast<long long>(row) * a.c.heads * D, y);
    }
  }
}

// ---------------------------------------------------------------------------------------------------- page copies
constexpr int kCopyTensors = 128;
constexpr int kCopyChunk = 16384;  // bytes per CTA step (3.4 GB of pages in 572 us; the table travels in the launch parameters)

template <int PAIRS>
struct CopyTable {
  uint8_t* base[kCopyTensors];
  long long page_bytes[kCopyTensors];
  int chunk_start[kCopyTensors + 1];  // cumulative chunks (pairs * chunks per page)
  int pairs, tensors;
  int src[PAIRS], dst[PAIRS];
};

template <typename V>
__device__ __forceinline__ void copy_range(uint8_t* dst, const uint8_t* src, int bytes) {
  const int n = bytes / static_cast<int>(sizeof(V));
  const V* s = reinterpret_cast<const V*>(src);
  V* d = reinterpret_cast<V*>(dst);
  int i = threadIdx.x;
  for (; i + 3 * static_cast<int>(blockDim.x) < n; i += 4 * blockDim.x) {
    V v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = s[i + u * blockDim.x];
#pragma unroll
    for (int u = 0; u < 4; ++u) d[i + u * blockDim.x] = v[u];
  }
  for (; i < n; i += blockDim.x) d[i] = s[i];
}

template <int PAIRS>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyTable<PAIRS> t) {
  const int total = t.chunk_start[t.tensors];
  for (int c = blockIdx.x; c < total; c += gridDim.x) {
    int lo = 0, hi = t.tensors - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (t.chunk_start[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const long long pb = t.page_bytes[lo];
    const int per = static_cast<int>((pb + kCopyChunk - 1) / kCopyChunk);
    const int rel = c - t.chunk_start[lo];
    const int pair = rel / per;
    const long long at = static_cast<long long>(rel % per) * kCopyChunk;
    const int bytes = static_cast<int>(pb - at < kCopyChunk ? pb - at : kCopyChunk);
    const uint8_t* s = t.base[lo] + t.src[pair] * pb + at;
    uint8_t* d = t.base[lo] + t.dst[pair] * pb + at;
    const uint64_t align = reinterpret_cast<uint64_t>(t.base[lo]) | static_cast<uint64_t>(pb);
    if (align % 16 == 0) copy_range<uint4>(d, s, bytes);
    else if (align % 4 == 0) copy_range<uint32_t>(d, s, bytes);
    else copy_range<uint8_t>(d, s, bytes);
  }
}

template <int PAIRS>
cudaError_t launch_copy(const PageCopyTensor* tensors, int num_tensors, const int* src, const int* dst, int pairs,
                        cudaStream_t stream) {
  CopyTable<PAIRS> t;
  t.pairs = pairs;
  t.tensors = num_tensors;
  long long chunks = 0;
  for (int i = 0; i < num_tensors; ++i) {
    t.base[i] = static_cast<uint8_t*>(tensors[i].base);
    t.page_bytes[i] = tensors[i].page_bytes;
    t.chunk_start[i] = static_cast<int>(chunks);
    chunks += (tensors[i].page_bytes + kCopyChunk - 1) / kCopyChunk * pairs;
    if (chunks > 0x7fffffff) return cudaErrorInvalidValue;
  }
  t.chunk_start[num_tensors] = static_cast<int>(chunks);
  for (int i = 0; i < pairs; ++i) {
    t.src[i] = src[i];
    t.dst[i] = dst[i];
  }
  if (chunks == 0) return cudaSuccess;
  const int grid = static_cast<int>(chunks < 148 * 8 ? chunks : 148 * 8);
  copy_pages_kernel<PAIRS><<<grid, 256, 0, stream>>>(t);
  return cudaGetLastError();
}

template <typename T>
cudaError_t append_d(const Fp8AppendArgs& a, dim3 grid, cudaStream_t s) {
  if (a.c.d == 64) append_kernel<T, 64><<<grid, 128, 0, s>>>(a);
  else if (a.c.d == 128) append_kernel<T, 128><<<grid, 128, 0, s>>>(a);
  else if (a.c.d == 256) append_kernel<T, 256><<<grid, 128, 0, s>>>(a);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

template <typename T>
cudaError_t gather_d(const Fp8GatherArgs& a, dim3 grid, cudaStream_t s) {
  if (a.c.d == 64) gather_kernel<T, 64><<<grid, 128, 0, s>>>(a);
  else if (a.c.d == 128) gather_kernel<T, 128><<<grid, 128, 0, s>>>(a);
  else if (a.c.d == 256) gather_kernel<T, 256><<<grid, 128, 0, s>>>(a);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

// CTAs along a sequence's 16-token blocks: those of the longest one, but no millions in all where that is a loose bound
// or few sequences are long (the kernels walk on by the grid's height)
int blocks_of(long long blocks, const Fp8CacheView& c) {
  const long long most = 262144 / (static_cast<long long>((2 * c.heads + 3) / 4) * c.n) + 1;
  blocks = blocks < 1 ? 1 : (blocks < most ? blocks : most);
  return static_cast<int>(blocks < 65535 ? blocks : 65535);
}

bool view_ok(const Fp8CacheView& c) {
  return c.pages > 0 && c.heads > 0 && c.page_size >= kKvBlock && c.page_size % kKvBlock == 0 && c.n <= 65535 &&
         c.width > 0;
}

}  // namespace

cudaError_t fp8_cache_append(const Fp8AppendArgs& a, cudaStream_t s) {
  if (!view_ok(a.c)) return cudaErrorInvalidValue;
  if (a.c.n == 0 || a.t == 0) return cudaSuccess;
  const long long blocks = (static_cast<long long>(a.max_new) + kKvBlock - 2) / kKvBlock + 1;  // a run may start on a block's last row
  const dim3 grid((2 * a.c.heads + 3) / 4, blocks_of(blocks, a.c), a.c.n);
  if (a.dtype == kFloat32) return append_d<float>(a, grid, s);
  if (a.dtype == kFloat16) return append_d<__half>(a, grid, s);
  if (a.dtype == kBFloat16) return append_d<__nv_bfloat16>(a, grid, s);
  return cudaErrorInvalidValue;
}

cudaError_t fp8_cache_gather(const Fp8GatherArgs& a, cudaStream_t s) {
  if (!view_ok(a.c)) return cudaErrorInvalidValue;
  if (a.c.n == 0 || (a.rows == 0 && a.off != nullptr)) return cudaSuccess;
  if (a.off == nullptr && (a.cu_q == nullptr || a.cu_k == nullptr || a.first_row == nullptr || a.cut_q == nullptr || a.first_q == nullptr ||
                           a.out == nullptr || a.row_bytes % 4 != 0 || static_cast<long long>(a.pitch) * a.c.n > a.rows))
    return cudaErrorInvalidValue;
  const dim3 grid((2 * a.c.heads + 3) / 4, blocks_of((static_cast<long long>(a.max_kv) + 127) / 128 * 8, a.c), a.c.n);
  if (a.dtype == kFloat32) return gather_d<float>(a, grid, s);
  if (a.dtype == kFloat16) return gather_d<__half>(a, grid, s);
  if (a.dtype == kBFloat16) return gather_d<__nv_bfloat16>(a, grid, s);
  return cudaErrorInvalidValue;
}

cudaError_t copy_pages(const PageCopyTensor* tensors, int num_tensors, const int* src, const int* dst, int pairs,
                       cudaStream_t stream) {
  // the table travels in the launch parameters: a small one for a fork, a large one for a compaction
  for (int t0 = 0; t0 < num_tensors; t0 += kCopyTensors) {
    const int nt = num_tensors - t0 < kCopyTensors ? num_tensors - t0 : kCopyTensors;
    for (int p0 = 0; p0 < pairs; p0 += 1024) {
      const int np = pairs - p0 < 1024 ? pairs - p0 : 1024;
      const cudaError_t e = np <= 64 ? launch_copy<64>(tensors + t0, nt, src + p0, dst + p0, np, stream)
                                     : launch_copy<1024>(tensors + t0, nt, src + p0, dst + p0, np, stream);
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

}  // namespace teb200
