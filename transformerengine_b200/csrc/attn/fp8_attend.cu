// Attention over the 8-bit paged key/value cache: few queries per sequence against long caches.
//
// The codes are read once per group of query heads, so the bytes of the cache bound the work: per token and head 2 d
// bytes against 4 d flop per query row.  A warp takes whole steps of tokens and works on transposed products,
//   S^T[token, row] = K[token, :] . Q^T        (m16n8k16: 16 tokens x 8 query rows)
//   O^T[dim, row]  += V^T[dim, token] . P^T    (m16n8k16: 16 dims x 8 query rows)
// because the query rows of one key head (heads per group x queries) are few: 8 fill the narrow side of the
// instruction, where 16 rows of Q as its wide side would be half empty.  Every operand comes straight from global memory
// into the registers that the instruction wants: the 16-byte pieces of K and V that a lane loads are whole fragments once
// the order of d (for K) and of the output dims (for V) is chosen to fit, so nothing passes through shared memory.
// Codes become fp16 exactly.  Q is scaled per row by a power of two into fp16's range (bf16 has fewer bits than fp16, so
// only values 2^-29 below the row's largest lose any).  A block's K scale multiplies its scores, its V scale s multiplies
// the probabilities: with the running maximum m taken over score + log2 s, exp2(score - m) * s stays within 1 and fits
// fp16 whatever the scales (kept within 2^-60 .. 2^60); sums and accumulators are fp32.
// Long caches are split over CTAs by equal runs of steps; a second kernel joins the parts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fp8_cache.cuh"
#include "teb200/api.h"
#include "teb200/kv_cache.h"

namespace teb200 {
namespace {

using namespace kvc;

constexpr int kWarps = 4;
constexpr int kLookahead = 16;  // steps whose pages and scales a warp looks up at once

struct AttendParams {
  Fp8AttendArgs a;
  int chunk;       // steps per CTA
  int splits;      // CTAs along the tokens
  int row_tiles;   // tiles of query rows per (sequence, key head)
  int group;       // query heads per key head
  float scale_log2;
};

template <int D>
struct Cfg {
  static constexpr int kStep = D == 256 ? 16 : 32;   // tokens per step and warp
  static constexpr int kBlocks = kStep / kKvBlock;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream2(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Where the rows [r0, r1) of a sequence's tile look: positions and the steps of tokens to walk.
struct Walk {
  int len, qlen;       // tokens held, queries
  int q_row0;          // first query token of the sequence in the packed queries
  int sink_steps;      // steps 0 .. sink_steps - 1 come before the gap
  int gap;             // tokens skipped after them
  int steps;           // total
};

template <int STEP>
__device__ __forceinline__ Walk walk_of(const Fp8AttendArgs& a, int seq, int r0, int r1, int group, bool report) {
  Walk w;
  w.q_row0 = a.cu_q[seq];
  w.qlen = a.cu_q[seq + 1] - w.q_row0;
  w.len = a.c.kv_lens[seq];
  bool bad = w.q_row0 < 0 || w.q_row0 > a.tq || w.qlen < 0 || w.qlen > a.max_q || w.qlen > a.tq - w.q_row0 || w.len < 0 ||
             w.len > a.max_kv;
  if (bad) {
    if (report) atomicCAS(a.c.status, 0, kKvStatusPages);
    w.q_row0 = min(max(w.q_row0, 0), a.tq);
    w.qlen = min(min(max(w.qlen, 0), a.max_q), a.tq - w.q_row0);
    w.len = min(max(w.len, 0), a.max_kv);
  }
  w.sink_steps = 0;
  w.gap = 0;
  const int rows = min(r1, w.qlen * group);
  if (rows <= r0 || w.len == 0) {
    w.steps = 0;
    return w;
  }
  int end = w.len;  // exclusive
  if (a.causal) end = w.len - w.qlen + (rows - 1) / group + 1;
  if (end <= 0) {
    w.steps = 0;
    return w;
  }
  int begin = 0;
  if (a.window_left >= 0) begin = max(w.len - w.qlen + r0 / group - a.window_left, 0) / STEP * STEP;
  const int sinks = (min(a.sinks, end) + STEP - 1) / STEP;
  if (begin > sinks * STEP) {
    w.sink_steps = sinks;
    w.gap = begin - sinks * STEP;
  }
  w.steps = (end - w.gap + STEP - 1) / STEP;
  return w;
}

template <int D, int NT, bool BF>
__global__ void __launch_bounds__(kWarps * 32, D == 64 ? 4 : (NT == 1 && D == 128 ? 3 : 2))
attend_kernel(const AttendParams p) {
  using C = Cfg<D>;
  constexpr int STEP = C::kStep;
  constexpr int NB = C::kBlocks;       // 16-token blocks per step
  constexpr int R = NT * 8;            // query rows of the tile
  constexpr int KC = D / 64;           // 16-byte pieces of a key row per lane
  constexpr int MT = D / 16;           // 16-dim tiles of the output
  const Fp8AttendArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int g8 = lane >> 2, c4 = lane & 3;
  const int seq = blockIdx.z;
  if (seq == a.c.n) {
    // queries behind the last sequence: zeros
    if (blockIdx.x != 0) return;
    const long long first = static_cast<long long>(max(a.cu_q[a.c.n], 0)) * a.hq * D;
    const long long last = static_cast<long long>(a.tq) * a.hq * D;
    uint32_t* o = reinterpret_cast<uint32_t*>(a.out);
    for (long long i = first / 2 + blockIdx.y * blockDim.x + threadIdx.x; i < last / 2; i += gridDim.y * blockDim.x) o[i] = 0u;
    return;
  }
  const int head = blockIdx.y / p.row_tiles;
  const int r0 = blockIdx.y % p.row_tiles * R;
  const Walk w = walk_of<STEP>(a, seq, r0, r0 + R, p.group, threadIdx.x == 0);
  const int rows = min(w.qlen * p.group - r0, R);   // rows of this tile
  if (rows <= 0) return;
  const int s_begin = blockIdx.x * p.chunk;
  const int s_end = min(s_begin + p.chunk, w.steps);
  if (s_begin >= s_end && blockIdx.x > 0) return;
  const int active = (w.steps + p.chunk - 1) / p.chunk;

  __shared__ float sm_o[kWarps][R][D + 4];
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];

  // ---- queries: fp16 fragments of row g8 of every 8-row tile, scaled by a power of two
  uint32_t qf[NT][KC * 4][2];
  float row_scale[NT][2];             // of columns 2 c4, 2 c4 + 1: score units (log2)
  int hi[NT][2], lo[NT][2];           // visible tokens of those columns: lo <= j <= hi, or j < sinks
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = min(t * 8 + g8, rows - 1) + r0;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (w.q_row0 + r / p.group) * a.q_st +
                        (head * p.group + r % p.group) * a.q_sh;
    float x[KC][16];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const uint4* src = reinterpret_cast<const uint4*>(q + i * 64 + c4 * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v = src[h];
        const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float f0, f1;
          if (BF) {
            f0 = __uint_as_float(ww[e] << 16);
            f1 = __uint_as_float(ww[e] & 0xffff0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ww[e]));
            f0 = f.x;
            f1 = f.y;
          }
          x[i][h * 8 + e * 2] = f0;
          x[i][h * 8 + e * 2 + 1] = f1;
          top = fmaxf(top, fmaxf(fabsf(f0), fabsf(f1)));
        }
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // top * 2^-e in [2^14, 2^15); e is kept where 2^-e is a finite number
    const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -100);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < KC; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const __half2 v = __floats2half2_rn(x[i][k * 4 + h * 2] * down, x[i][k * 4 + h * 2 + 1] * down);
          qf[t][i * 4 + k][h] = *reinterpret_cast<const uint32_t*>(&v);
        }
#pragma unroll
    for (int e2 = 0; e2 < 2; ++e2) {
      row_scale[t][e2] = __shfl_sync(0xffffffffu, up, (c4 * 2 + e2) * 4) * p.scale_log2;
      const int rr = min(t * 8 + c4 * 2 + e2, rows - 1) + r0;
      const int pos = w.len - w.qlen + rr / p.group;
      hi[t][e2] = a.causal ? min(pos, w.len - 1) : w.len - 1;
      lo[t][e2] = a.window_left >= 0 ? pos - a.window_left : 0;
    }
  }
  // limits over the whole tile: steps inside need no mask
  const int pos_first = w.len - w.qlen + r0 / p.group;
  const int pos_last = w.len - w.qlen + (r0 + rows - 1) / p.group;
  const int hi_min = a.causal ? min(pos_first, w.len - 1) : w.len - 1;
  const int hi_max = a.causal ? min(pos_last, w.len - 1) : w.len - 1;
  const int lo_min = a.window_left >= 0 ? pos_first - a.window_left : 0;
  const int lo_max = a.window_left >= 0 ? pos_last - a.window_left : 0;

  float o[NT][MT][4];
  float m_run[NT][2], l_run[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][j][e] = 0.f;
    m_run[t][0] = m_run[t][1] = -INFINITY;
    l_run[t][0] = l_run[t][1] = 0.f;
  }

  const int per = a.c.page_size / kKvBlock;
  const int* table = a.c.table + static_cast<long long>(seq) * a.c.width;

  uint4 kr[NB][2][KC];
  uint4 vr[NB][4][D >= 128 ? D / 128 : 1];

  // pages and scales of the warp's next kLookahead steps, one block per lane
  int look_idx = -1;
  float look_k = 0.f, look_v = 0.f;
  auto look_up = [&](int step0) {
    const int st = step0 + (lane / NB) * kWarps;
    look_idx = -1;
    look_k = 0.f;
    look_v = 1.f;
    if (lane < kLookahead * NB && st < s_end) {
      const int tok = st * STEP + (st >= w.sink_steps ? w.gap : 0) + (lane % NB) * kKvBlock;
      if (tok < w.len) {
        const int blk = tok / kKvBlock;
        const int slot = blk / per;
        const int page = slot < a.c.width ? table[slot] : -1;
        if (page >= 0 && page < a.c.pages) {
          look_idx = (page * a.c.heads + head) * per + blk % per;
          look_k = a.c.k_scale[look_idx];
          look_v = a.c.v_scale[look_idx];
        } else {
          // a page that is not held may lie outside what the tile sees; inside, its tokens count as hidden
          if (tok <= hi_max && (tok + kKvBlock > lo_min || tok < a.sinks)) atomicCAS(a.c.status, 0, kKvStatusPages);
        }
      }
    }
  };
  auto load_k = [&](int j) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int idx = __shfl_sync(0xffffffffu, look_idx, j * NB + b);
      const uint8_t* base = a.c.k + static_cast<long long>(max(idx, 0)) * (kKvBlock * D) + g8 * D + c4 * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < KC; ++i) kr[b][h][i] = ld_stream(base + h * 8 * D + i * 64);
    }
  };
  auto load_v = [&](int j) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int idx = __shfl_sync(0xffffffffu, look_idx, j * NB + b);
      const uint8_t* base = a.c.v + static_cast<long long>(max(idx, 0)) * (kKvBlock * D) + c4 * 2 * D;
#pragma unroll
      for (int t = 0; t < 4; ++t) {   // tokens 2c, 2c + 1, 2c + 8, 2c + 9
        const uint8_t* row = base + ((t & 1) + (t >> 1) * 8) * D;
        if (D == 64) {
          const uint2 x = ld_stream2(row + g8 * 8);
          vr[b][t][0].x = x.x;
          vr[b][t][0].y = x.y;
        } else {
#pragma unroll
          for (int i = 0; i < D / 128; ++i) vr[b][t][i] = ld_stream(row + i * 128 + g8 * 16);
        }
      }
    }
  };

  int look_base = s_begin + warp;
  if (look_base < s_end) {
    look_up(look_base);
    load_k(0);
    load_v(0);
  }
  int j = 0;
  for (int st = s_begin + warp; st < s_end; st += kWarps, ++j) {
    const int tok0 = st * STEP + (st >= w.sink_steps ? w.gap : 0);
    // ---- S^T = K Q^T
    float s[NT][NB][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][b][e] = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint32_t wa[4] = {kr[b][0][i].x, kr[b][0][i].y, kr[b][0][i].z, kr[b][0][i].w};
        const uint32_t wb[4] = {kr[b][1][i].x, kr[b][1][i].y, kr[b][1][i].z, kr[b][1][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(wa[k]));
          const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(wa[k] >> 16));
          const uint32_t a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(wb[k]));
          const uint32_t a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(wb[k] >> 16));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(s[t][b], a0, a1, a2, a3, qf[t][i * 4 + k][0], qf[t][i * 4 + k][1]);
        }
      }
    float ks[NB], vs[NB];
    bool held[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      ks[b] = __shfl_sync(0xffffffffu, look_k, j * NB + b);
      vs[b] = __shfl_sync(0xffffffffu, look_v, j * NB + b);
      held[b] = __shfl_sync(0xffffffffu, look_idx, j * NB + b) >= 0;
    }
    // ---- the next step's keys
    const bool more = st + kWarps < s_end;
    const bool turn = j + 1 == kLookahead;
    if (more && !turn) load_k(j + 1);
    // ---- softmax
    bool all_held = true;
#pragma unroll
    for (int b = 0; b < NB; ++b) all_held = all_held && held[b];
    const bool need_mask = !all_held || tok0 + STEP - 1 > hi_min || (tok0 < lo_max && tok0 + STEP > a.sinks);
    uint32_t pf[NT][NB][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        // log2 of the block's V scale, from its exponent
        const float lv = static_cast<float>(static_cast<int>(__float_as_uint(vs[b]) >> 23) - 127);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[t][b][e] * (row_scale[t][e & 1] * ks[b]);
          if (need_mask) {
            const int tok = tok0 + b * kKvBlock + g8 + (e >> 1) * 8;
            const bool seen = held[b] && tok <= hi[t][e & 1] && (tok >= lo[t][e & 1] || tok < a.sinks);
            if (!seen) x = -INFINITY;
          }
          s[t][b][e] = x;
          mx[e & 1] = fmaxf(mx[e & 1], x + lv);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], off));
      }
      float alpha[2], m_use[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m_new = fmaxf(m_run[t][e], mx[e]);
        m_use[e] = m_new == -INFINITY ? 0.f : m_new;
        alpha[e] = ex2(m_run[t][e] - m_use[e]);
        m_run[t][e] = m_new;
        l_run[t][e] *= alpha[e];
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float pv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = ex2(s[t][b][e] - m_use[e & 1]);
          l_run[t][e & 1] += x;
          pv[e] = x * vs[b];
        }
        const __half2 h0 = __floats2half2_rn(pv[0], pv[1]), h1 = __floats2half2_rn(pv[2], pv[3]);
        pf[t][b][0] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&h0));
        pf[t][b][1] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&h1));
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int jt = 0; jt < MT; ++jt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][jt][e] *= alpha[e & 1];
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (need_mask) {
        // hidden tokens meet probability 0, but what their slots hold may be NaN
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int tok = tok0 + b * kKvBlock + c4 * 2 + (t & 1) + (t >> 1) * 8;
          if (!held[b] || tok > hi_max || (tok < lo_min && tok >= a.sinks)) {
#pragma unroll
            for (int i = 0; i < (D >= 128 ? D / 128 : 1); ++i) vr[b][t][i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < (D >= 128 ? D / 128 : 1); ++i) {
        constexpr int kWords = D == 64 ? 2 : 4;
        const uint32_t w0[4] = {vr[b][0][i].x, vr[b][0][i].y, vr[b][0][i].z, vr[b][0][i].w};
        const uint32_t w1[4] = {vr[b][1][i].x, vr[b][1][i].y, vr[b][1][i].z, vr[b][1][i].w};
        const uint32_t w2[4] = {vr[b][2][i].x, vr[b][2][i].y, vr[b][2][i].z, vr[b][2][i].w};
        const uint32_t w3[4] = {vr[b][3][i].x, vr[b][3][i].y, vr[b][3][i].z, vr[b][3][i].w};
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {   // dims 4k + 2u, 4k + 2u + 1 of the lane's piece
            const uint32_t x = __byte_perm(w0[k], w1[k], u == 0 ? 0x5140 : 0x7362);
            const uint32_t y = __byte_perm(w2[k], w3[k], u == 0 ? 0x5140 : 0x7362);
            const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(x));
            const uint32_t a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(x >> 16));
            const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(y));
            const uint32_t a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(y >> 16));
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16(o[t][(i * 4 + k) * 2 + u], a0, a1, a2, a3, pf[t][b][0], pf[t][b][1]);
          }
        }
      }
    }
    // ---- the next step's values
    if (more) {
      if (turn) {
        look_up(st + kWarps);
        load_k(0);
        load_v(0);
        j = -1;
      } else {
        load_v(j + 1);
      }
    }
  }

  // ---- join the warps
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[t][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      const int r = t * 8 + c4 * 2 + e;
      if (g8 == 0) {
        sm_m[warp][r] = m_run[t][e];
        sm_l[warp][r] = l;
      }
#pragma unroll
      for (int jt = 0; jt < MT; ++jt) {
        const int dim = D == 64 ? g8 * 8 + jt * 2 : (jt / 8) * 128 + g8 * 16 + (jt % 8) * 2;
        *reinterpret_cast<float2*>(&sm_o[warp][r][dim]) = make_float2(o[t][jt][e], o[t][jt][e + 2]);
      }
    }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * (D / 2); x += kWarps * 32) {
    const int r = x / (D / 2), d = x % (D / 2) * 2;
    float m = sm_m[0][r];
#pragma unroll
    for (int v = 1; v < kWarps; ++v) m = fmaxf(m, sm_m[v][r]);
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      const float f = ex2(sm_m[v][r] - m_use);
      l += sm_l[v][r] * f;
      const float2 y = *reinterpret_cast<const float2*>(&sm_o[v][r][d]);
      x0 += y.x * f;
      x1 += y.y * f;
    }
    const int rr = r0 + r;
    const long long row = static_cast<long long>(w.q_row0 + rr / p.group) * a.hq + head * p.group + rr % p.group;
    if (active <= 1) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // NaN stays NaN
      *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + row * D + d) = pack2<BF>(x0 * inv, x1 * inv);
    } else {
      const long long part = static_cast<long long>(blockIdx.x) * a.tq * a.hq + row;
      float* po = a.part + static_cast<long long>(p.splits) * a.tq * a.hq * 2;
      *reinterpret_cast<float2*>(po + part * D + d) = make_float2(x0, x1);
      if (d == 0) *reinterpret_cast<float2*>(a.part + part * 2) = make_float2(m, l);
    }
  }
}

// One warp per query row: joins the parts of its sequence's steps.
template <int D, bool BF>
__global__ void __launch_bounds__(128) join_kernel(const AttendParams p, int rows_per_tile) {
  const Fp8AttendArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int seq = blockIdx.y;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 5);      // query row: token, then head
  const int qi = r / a.hq, hq = r % a.hq;
  const int rr = qi * p.group + hq % p.group;             // row within the key head
  const int r0 = rr / rows_per_tile * rows_per_tile;
  const Walk w = walk_of<Cfg<D>::kStep>(a, seq, r0, r0 + rows_per_tile, p.group, false);
  if (qi >= w.qlen) return;
  const int active = (w.steps + p.chunk - 1) / p.chunk;
  if (active <= 1) return;
  const long long rows = static_cast<long long>(a.tq) * a.hq;
  const long long row = static_cast<long long>(w.q_row0 + qi) * a.hq + hq;
  const float* ml = a.part;
  const float* po = a.part + p.splits * rows * 2;
  float m = -INFINITY;
  for (int s = lane; s < active; s += 32) m = fmaxf(m, ml[(s * rows + row) * 2]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int s = 0; s < active; ++s) {
    const float2 v = *reinterpret_cast<const float2*>(ml + (s * rows + row) * 2);
    const float f = ex2(v.x - m_use);
    l += v.y * f;
    const float* src = po + (s * rows + row) * D + lane * 2;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float2 y = *reinterpret_cast<const float2*>(src + i * 64);
      acc[2 * i] += y.x * f;
      acc[2 * i + 1] += y.y * f;
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + row * D);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) out[lane + i * 32] = pack2<BF>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
}

int rows_per_tile(const Fp8AttendArgs& a) {
  const int rows = a.hq / a.c.heads * a.max_q;
  return rows <= 8 || a.c.d == 256 ? 8 : 16;   // d 256: the accumulators of 16 rows do not fit the registers
}

// Equal runs of steps per CTA: enough CTAs to fill the SMs a few times over when every sequence were as long as the
// longest, but at least 4 steps per warp, so that writing and joining the fp32 parts stays small beside reading the codes.
AttendParams plan(const Fp8AttendArgs& a) {
  AttendParams p;
  p.a = a;
  p.group = a.hq / a.c.heads;
  const int R = rows_per_tile(a);
  p.row_tiles = (p.group * a.max_q + R - 1) / R;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  const int step = a.c.d == 256 ? 16 : 32;
  long long tokens = a.max_kv;
  if (a.window_left >= 0) {
    const long long seen = static_cast<long long>(a.window_left) + R + 2 * step + (a.sinks + step - 1) / step * step;
    tokens = seen < tokens ? seen : tokens;
  }
  const int steps = static_cast<int>((tokens + step - 1) / step) + 1;
  const long long tiles = static_cast<long long>(a.c.n) * a.c.heads * p.row_tiles;
  const long long want = 148 * 3 * 4;
  long long splits = (want + tiles - 1) / (tiles > 0 ? tiles : 1);
  int chunk = static_cast<int>((steps + splits - 1) / splits);
  chunk = chunk < 4 * kWarps ? 4 * kWarps : (chunk + kWarps - 1) / kWarps * kWarps;
  p.chunk = chunk;
  p.splits = (steps + chunk - 1) / chunk;
  return p;
}

template <int D, int NT, bool BF>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  const dim3 grid(p.splits, p.a.c.heads * p.row_tiles, p.a.c.n + 1);
  attend_kernel<D, NT, BF><<<grid, kWarps * 32, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  const dim3 jgrid((p.a.max_q * p.a.hq + 3) / 4, p.a.c.n);
  join_kernel<D, BF><<<jgrid, 128, 0, s>>>(p, NT * 8);
  return cudaGetLastError();
}

template <int D, int NT>
cudaError_t launch_t(const AttendParams& p, cudaStream_t s) {
  return p.a.is_bf16 ? launch<D, NT, true>(p, s) : launch<D, NT, false>(p, s);
}

bool attend_ok(const Fp8AttendArgs& a) {
  const Fp8CacheView& c = a.c;
  return c.pages > 0 && c.heads > 0 && c.page_size >= kKvBlock && c.page_size % kKvBlock == 0 && c.n >= 0 &&
         c.n < 65535 && c.width > 0 && a.hq % c.heads == 0 && a.max_q >= 0 && a.max_kv >= 0 &&
         static_cast<long long>(c.pages) * c.heads * (c.page_size / kKvBlock) <= 0x7fffffff &&
         (c.d == 64 || c.d == 128 || c.d == 256);
}

}  // namespace

long long fp8_attend_workspace(const Fp8AttendArgs& a) {
  if (!attend_ok(a) || a.tq == 0 || a.max_q == 0) return 0;
  const AttendParams p = plan(a);
  return p.splits == 1 ? 0 : static_cast<long long>(p.splits) * a.tq * a.hq * (a.c.d + 2);
}

cudaError_t fp8_attend(const Fp8AttendArgs& a, cudaStream_t s) {
  if (!attend_ok(a)) return cudaErrorInvalidValue;
  if (a.tq == 0) return cudaSuccess;
  const AttendParams p = plan(a);
  if (static_cast<long long>(a.c.heads) * p.row_tiles > 65535 || (p.splits > 1 && a.part == nullptr)) return cudaErrorInvalidValue;
  if (a.c.d == 64) return p.group * a.max_q <= 8 ? launch_t<64, 1>(p, s) : launch_t<64, 2>(p, s);
  if (a.c.d == 128) return p.group * a.max_q <= 8 ? launch_t<128, 1>(p, s) : launch_t<128, 2>(p, s);
  return launch_t<256, 1>(p, s);
}

}  // namespace teb200
