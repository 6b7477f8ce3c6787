// Code conversions shared by the kernels of the 8-bit key/value cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "teb200/kv_cache.h"

namespace teb200 {
namespace kvc {

// A sequence's queries within the packed rows and the tokens it holds; `bad`: the given numbers do not fit and were cut.
struct SeqFit {
  int q_row0, qlen, len;
  bool bad;
};

__device__ __forceinline__ SeqFit fit_sequence(const int* cu_q, const int* kv_lens, int seq, int tq, int max_q, int max_kv) {
  SeqFit f;
  f.q_row0 = cu_q[seq];
  f.qlen = cu_q[seq + 1] - f.q_row0;
  f.len = kv_lens[seq];
  f.bad = f.q_row0 < 0 || f.q_row0 > tq || f.qlen < 0 || f.qlen > max_q || f.qlen > tq - f.q_row0 || f.len < 0 || f.len > max_kv;
  if (f.bad) {
    f.q_row0 = min(max(f.q_row0, 0), tq);
    f.qlen = min(min(max(f.qlen, 0), max_q), tq - f.q_row0);
    f.len = min(max(f.len, 0), max_kv);
  }
  return f;
}

// Zeros in the output rows (of `words` 32-bit words) that no query claims: behind the last sequence (if `last`), and,
// reported by fit_sequence, those of a sequence beyond max_q.  All threads of `ctas` CTAs take part.
__device__ __forceinline__ void zero_unclaimed(uint32_t* out, long long words, const int* cu_q, int n, int tq, int max_q,
                                               bool last, long long cta, long long ctas) {
  const int end = last ? cu_q[n] : tq;
  int q0 = cta < n ? cu_q[cta] : 0, q1 = cta < n ? cu_q[cta + 1] : 0;   // the first (mostly the only) turn of the loop below
  for (long long i = max(end, 0) * words + cta * blockDim.x + threadIdx.x; i < tq * words; i += ctas * blockDim.x) out[i] = 0u;
  for (long long seq = cta; seq < n;) {
    const int from = min(max(q0, 0), tq);
    const int claimed = min(min(max(q1 - q0, 0), max_q), tq - from);
    for (long long i = (from + claimed) * words + threadIdx.x; i < min(q1, tq) * words; i += blockDim.x) out[i] = 0u;
    seq += ctas;
    if (seq < n) {
      q0 = cu_q[seq];
      q1 = cu_q[seq + 1];
    }
  }
}

// The smallest power of two s with top <= 448 s, kept within 2^-60 .. 2^60.  With top = f 2^e, 1 <= f < 2, and
// 448 = 1.75 2^8, that is 2^(e - 8) for f <= 1.75 and 2^(e - 7) above.
__device__ __forceinline__ float scale_for(float top) {
  const uint32_t bits = __float_as_uint(top);
  int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -60 ? -60 : (e > 60 ? 60 : e);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// 1 / s of a power of two by its exponent bits (a fast-math division need not be exact)
__device__ __forceinline__ float inverse_of_power(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }

// to e4m3, nearest even; beyond 448 saturates, NaN stays NaN
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// two e4m3 codes (low half of w) as two fp16 values, exact
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
  return r;
}

__device__ __forceinline__ void from_e4m3x4(uint32_t w, float* y) {
  const uint32_t a = e4m3x2_to_f16x2(static_cast<uint16_t>(w)), b = e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16));
  const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
  y[0] = fa.x; y[1] = fa.y; y[2] = fb.x; y[3] = fb.y;
}

// Two fp32 values rounded to 16 bits.  A code may round an fp16 value up past fp16's largest: that one saturates.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  if (fabsf(a) > 65504.f) a = copysignf(65504.f, a);
  if (fabsf(b) > 65504.f) b = copysignf(65504.f, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace kvc
}  // namespace teb200
