// Attention over the 8-bit paged key/value cache: few queries per sequence against long caches.
//
// The codes are read once per group of query heads, so the bytes of the cache bound the work: per token and head 2 d
// bytes against 4 d flop per query row.  A warp takes whole steps of tokens and works on transposed products,
//   S^T[token, row] = K[token, :] . Q^T        (m16n8k16: 16 tokens x 8 query rows)
//   O^T[dim, row]  += V^T[dim, token] . P^T    (m16n8k16: 16 dims x 8 query rows)
// because the query rows of one key head (heads per group x queries) are few: 8 fill the narrow side of the
// instruction, where 16 rows of Q as its wide side would be half empty.  Each warp keeps a ring of kStages steps of 8 KB
// in flight with cp.async (its own ring: no warp waits for another), 192 KB per SM.  A lane's 16-byte pieces of K and V
// are whole fragments once the order of d (for K) and of the output dims (for V) is chosen to fit; the pieces of a row are
// permuted in shared memory so that both reads are free of bank conflicts.
// Codes become fp16 exactly.  Q is scaled per row by a power of two into fp16's range (bf16 has fewer bits than fp16, so
// only values 2^-29 below the row's largest lose any).  A block's K scale multiplies its scores, its V scale s multiplies
// the probabilities: with the running maximum m taken over score + log2 s, exp2(score + log2 s - m + 15) stays within 2^15
// and fits fp16 whatever the scales (kept within 2^-60 .. 2^60); sums and accumulators are fp32.  The 15 bits keep what the
// others add up to beside a token that takes nearly everything: without them codes below 2^-25 of the largest were zero in
// the products but not in the row sum (8000 tokens beside a first one with 99.99 % of the mass: 13 % off, now 2^-11).
// The steps of all sequences and heads form one line that the resident CTAs share equally, whatever the lengths: a CTA
// walks the end of one sequence, whole ones, and the beginning of another, and a second kernel joins the sequences that
// were cut.  Where no sequence is long (kDirectSteps), or a window makes them alike, a CTA per sequence and head takes it
// whole.  64 sequences of up to 8000 tokens, 32 / 8 heads, d 128: 0.56 GB of codes in 99 - 112 us; 4 of up to 130000, 64 / 8
// heads: 0.78 GB in 134 - 157 us (a copy moves 6.5 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "fp8_cache.cuh"
#include "teb200/api.h"
#include "teb200/kv_cache.h"
#include "teb200/ptx.cuh"

namespace teb200 {
namespace {

using namespace kvc;

constexpr int kWarps = 4;

// A CTA per sequence and head, without cutting and joining, is faster up to kDirectSteps steps, and up to twice as many
// where there are CTAs for half the SMs or more (us whole / cut, 32 / 8 heads: 700 tokens 8.1 / 11.9 for 1 sequence, 11.0 /
// 18.3 for 32; 2000 tokens 16.8 / 12.7 and 25.4 / 32.2).  Fewer than kMinShare steps are not worth a CTA of their own
// (4, 8 and 16 differ by less than 1 us from 1000 to 8000 tokens).
constexpr int kDirectSteps = 32;
constexpr int kMinShare = 8;

// Softmax offset of a row that has seen nothing: finite, so that differences with it are no NaN.
constexpr float kNothingSeen = -3.4e38f;

// What a row subtracts from its scores (log2) before the exponential: their maximum less 15.  Beyond 2^20, where the
// subtraction would be rounded and exp2 might leave fp16's range, the maximum itself.
__device__ __forceinline__ float softmax_offset(float top) { return fabsf(top) < 1048576.f ? top - 15.f : top; }

struct AttendParams {
  Fp8AttendArgs a;
  int ctas;        // 0: one CTA per (sequence, key head, tile of rows); else they share the line of steps
  int row_tiles;   // tiles of query rows per (sequence, key head)
  int group;       // query heads per key head
  float scale_log2;
  // workspace of the cut sequences: two slots per CTA (its first run of steps, and a later one)
  float2* part_ml;   // [2 ctas][R] softmax offset and row sum
  float* part_o;     // [2 ctas][R][d]
  int4* cuts;        // [ctas] the cut sequence that the CTA begins: sequence, first row, slot, last CTA; slot < 0: none
};

template <int D>
struct Cfg {
  static constexpr int kStep = D == 256 ? 16 : 32;      // tokens per step and warp
  static constexpr int kStepBytes = kStep * D;          // of K, and of V
  static constexpr int kBlocks = kStep / kKvBlock;
  static constexpr int kLookahead = 32 / kBlocks;       // steps whose pages and scales a warp looks up at once
};
// Steps in flight per warp and CTAs per SM: about 192 KB of rings per SM either way.  At d 128 two CTAs with three steps and
// three with two are alike (64 sequences of up to 8000 tokens: 104 and 107 us, 4 of up to 130000: 145 and 153), steps of
// 16 tokens are slower (109 - 121 us: the exchanges per step double).  At d 64 a step is half as many bytes.
template <int D, int NT>
struct Tune {
  static constexpr int kStages = D == 64 && NT == 2 ? 4 : 3;
  static constexpr int kCtas = D == 64 ? (NT == 1 ? 4 : 3) : 2;
  // 16 rows at d 256: the accumulators leave no registers for the queries' fragments
  static constexpr bool kQueriesInSmem = D == 256 && NT == 2;
  static constexpr int kRing = kWarps * kStages * 2 * Cfg<D>::kStepBytes;
  static constexpr int kParts = kWarps * NT * 8 * (D + 4) * 4;   // the warps' outputs, over the rings
  static constexpr int kRings = kRing > kParts ? kRing : kParts;
  static constexpr int kSmem = kRings + (kQueriesInSmem ? NT * (D / 16) * 256 : 0) + 128;   // to start on a 128-byte line
};

// Byte of 16-byte piece `piece` of row `row` within a step.  A K read takes pieces 4i .. 4i + 3 of rows 2j and 2j + 1 at
// once, a V read pieces 2j and 2j + 1 of rows 0, 2, 4, 6 (or 1, 3, 5, 7): with the pieces of a 128-byte line exchanged by
// ((row & 1) << 2) ^ (row & 6) both touch all 32 banks.  Rows of 64 bytes share a line in pairs.
template <int D>
__device__ __forceinline__ int place(int row, int piece) {
  if (D == 64) return (row >> 1) * 128 + ((((row & 1) << 2) | piece) ^ (((row >> 1) & 3) << 1)) * 16;
  return row * D + (piece ^ (((row & 1) << 2) ^ (row & 6))) * 16;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ void sts16_zero(uint32_t p) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(p), "r"(0) : "memory");
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}

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

// Where the rows [r0, r1) of a sequence's tile look: positions and the steps of tokens to walk.
struct Walk {
  int len, qlen;       // tokens held, queries
  int q_row0;          // first query token of the sequence in the packed queries
  int sink_steps;      // steps 0 .. sink_steps - 1 come before the gap
  int gap;             // tokens skipped after them
  int steps;           // total
  int rows;            // query rows of the tile (0: nothing to do); a tile with rows has at least one (hidden) step
};

template <int STEP>
__device__ __forceinline__ Walk walk_of(const Fp8AttendArgs& a, int seq, int r0, int r1, int group, bool report) {
  const SeqFit f = fit_sequence(a.cu_q, a.c.kv_lens, seq, a.tq, a.max_q, a.max_kv);
  if (f.bad && report) atomicCAS(a.c.status, 0, kKvStatusPages);
  Walk w;
  w.q_row0 = f.q_row0;
  w.qlen = f.qlen;
  w.len = f.len;
  w.sink_steps = 0;
  w.gap = 0;
  const int rows = min(r1, w.qlen * group);
  w.rows = max(rows - r0, 0);
  w.steps = w.rows > 0 ? 1 : 0;
  if (w.rows == 0 || w.len == 0) return w;
  int end = w.len;  // exclusive
  if (a.causal) end = w.len - w.qlen + (rows - 1) / group + 1;
  if (end <= 0) return w;
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

// What a CTA needs to know of its run of steps [s_begin, s_end) of one (sequence, key head, tile of rows).
struct Run {
  int seq, head, tile;
  int s_begin, s_end;
  int slot;            // >= 0: the run is part of a cut sequence and goes to this slot; else to the output
};

template <int D, int NT, bool BF>
__device__ __forceinline__ void attend_run(const AttendParams& p, const Walk& w, const Run& run, uint8_t* smem,
                                           float (*sm_m)[NT * 8], float (*sm_l)[NT * 8],
                                           float4 (*sm_meta)[Tune<D, NT>::kStages][Cfg<D>::kBlocks]) {
  using C = Cfg<D>;
  constexpr int STEP = C::kStep;
  constexpr int kStages = Tune<D, NT>::kStages;
  constexpr int kStepBytes = C::kStepBytes, kStageBytes = 2 * kStepBytes;
  constexpr int NB = C::kBlocks;       // 16-token blocks per step
  constexpr int R = NT * 8;            // query rows of the tile
  constexpr int KC = D / 64;           // 16-byte pieces of a key row per lane
  constexpr int MT = D / 16;           // 16-dim tiles of the output
  const Fp8AttendArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int g8 = lane >> 2, c4 = lane & 3;
  const int head = run.head;
  const int r0 = run.tile * R;
  const int rows = w.rows;
  const int s_begin = run.s_begin, s_end = run.s_end;
  // Addresses within a step, as place() gives them: a lane's first 16-byte piece to copy, of its key row and of its value
  // row.  The other pieces lie a constant further on, with bits 5 and 6 (the exchange within a line) flipped by a constant;
  // steps start on 128-byte lines, so the flips work on the full shared-memory address.
  const uint32_t ring = smem_u32(smem) + warp * (kStages * kStageBytes);
  const uint32_t copy_at = place<D>(lane / (D / 16), lane % (D / 16));
  const uint32_t key_at = place<D>(g8, c4);
  const uint32_t value_at = D == 64 ? place<D>(c4 * 2, g8 >> 1) + (g8 & 1) * 8 : place<D>(c4 * 2, g8);

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
    m_run[t][0] = m_run[t][1] = kNothingSeen;
    l_run[t][0] = l_run[t][1] = 0.f;
  }

  const int per = a.c.page_size / kKvBlock;
  const int* table = a.c.table + static_cast<long long>(run.seq) * a.c.width;

  // pages and scales of the warp's next kLookahead steps, one block per lane
  int look_idx = -1;
  float look_k = 0.f, look_v = 1.f;
  auto look_up = [&](int step0) {
    const int st = step0 + (lane / NB) * kWarps;
    look_idx = -1;
    look_k = 0.f;
    look_v = 1.f;
    if (st < s_end) {
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
          // a page that is not held may lie outside what the tile sees; inside, it is reported and its tokens are zeros
          if (tok <= hi_max && (tok + kKvBlock > lo_min || tok < a.sinks)) atomicCAS(a.c.status, 0, kKvStatusPages);
        }
      }
    }
  };
  // start the copies of the keys (values) of the warp's n-th step; blocks that are not held: block 0, whose codes nobody
  // uses.  One group each, in the order k0 v0 k1 v1 ...
  auto fetch = [&](int n, bool values) {
    const int st = s_begin + warp + n * kWarps;
    if (st < s_end) {
      const int at = n % C::kLookahead;
      if (!values && at == 0) look_up(st);
      const uint32_t to = ring + n % kStages * kStageBytes + (values ? kStepBytes : 0) + copy_at;
      const uint8_t* from = (values ? a.c.v : a.c.k) + lane * 16;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int idx = __shfl_sync(0xffffffffu, look_idx, at * NB + b);
        const uint8_t* src = from + static_cast<long long>(max(idx, 0)) * (kKvBlock * D);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {                // 512 bytes further: rows that exchange differently
          constexpr uint32_t kFlip[4] = {0u, D == 64 ? 0u : (D == 128 ? 64u : 32u), D == 256 ? 64u : 0u, D == 64 ? 0u : (D == 128 ? 64u : 96u)};
          cp_async16((to ^ kFlip[i % 4]) + b * (kKvBlock * D) + i * 512, src + i * 512);
        }
      }
      if (!values && lane / NB == at)
        sm_meta[warp][n % kStages][lane % NB] = make_float4(look_k, look_v, look_idx >= 0 ? 1.f : 0.f, 0.f);
    }
    cp_async_commit();
  };

#pragma unroll
  for (int n = 0; n < kStages; ++n) {
    fetch(n, false);
    fetch(n, true);
  }

  // ---- queries: fp16 fragments of row g8 of every 8-row tile, scaled by a power of two
  constexpr bool kQS = Tune<D, NT>::kQueriesInSmem;
  uint32_t qf[kQS ? 1 : NT][kQS ? 1 : KC * 4][2];
  uint2* q_smem = reinterpret_cast<uint2*>(smem + Tune<D, NT>::kRings);   // [NT][KC * 4][32]
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
          const uint32_t bits = *reinterpret_cast<const uint32_t*>(&v);
          if (!kQS) qf[kQS ? 0 : t][kQS ? 0 : i * 4 + k][h] = bits;
          else if (warp == t) reinterpret_cast<uint32_t*>(q_smem + (t * KC * 4 + i * 4 + k) * 32 + lane)[h] = bits;
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

  if (kQS) __syncthreads();      // every warp has written its fragments of the queries

  int n = 0;
  for (int st = s_begin + warp; st < s_end; st += kWarps, ++n) {
    const int tok0 = st * STEP + (st >= w.sink_steps ? w.gap : 0);
    cp_async_wait<2 * kStages - 1>();
    __syncwarp();
    const uint32_t keys = ring + n % kStages * kStageBytes + key_at;
    const uint32_t values = ring + n % kStages * kStageBytes + kStepBytes + value_at;
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
        const uint32_t from = (keys ^ (i & 1) * 64) + b * (kKvBlock * D) + (i >> 1) * 128;   // pieces 4 i + c4
        const uint4 ka = lds16(from), kb = lds16(from + 8 * D);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w};
        const uint32_t wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(wa[k]));
          const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(wa[k] >> 16));
          const uint32_t a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(wb[k]));
          const uint32_t a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(wb[k] >> 16));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint2 q;
            if (kQS) q = lds8(smem_u32(q_smem + (t * KC * 4 + i * 4 + k) * 32 + lane));
            else q = make_uint2(qf[kQS ? 0 : t][kQS ? 0 : i * 4 + k][0], qf[kQS ? 0 : t][kQS ? 0 : i * 4 + k][1]);
            mma_f16(s[t][b], a0, a1, a2, a3, q.x, q.y);
          }
        }
      }
    float ks[NB], vs[NB];
    bool held[NB];
    bool all_held = true;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float4 meta = sm_meta[warp][n % kStages][b];
      ks[b] = meta.x;
      vs[b] = meta.y;
      held[b] = meta.z != 0.f;
      all_held = all_held && held[b];
    }
    __syncwarp();                 // every lane has read the keys
    fetch(n + kStages, false);
    // ---- softmax of x = score + log2(V scale); exp2(x - offset) is what multiplies the V codes, and divided by the scale
    // it is the term of the row sum
    const bool need_mask = !all_held || tok0 + STEP - 1 > hi_min || (tok0 < lo_max && tok0 + STEP > a.sinks);
    uint32_t pf[NT][NB][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float lv = static_cast<float>(static_cast<int>(__float_as_uint(vs[b]) >> 23) - 127);  // log2 by the exponent
        const float c[2] = {row_scale[t][0] * ks[b], row_scale[t][1] * ks[b]};
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][b][e] = fmaf(s[t][b][e], c[e & 1], lv);
      }
    if (!all_held) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (!held[b]) {
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][b][0] = s[t][b][1] = s[t][b][2] = s[t][b][3] = 0.f;   // zero keys (V scale: 1)
        }
    }
    if (need_mask) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = tok0 + b * kKvBlock + g8 + (e >> 1) * 8;
            const bool seen = tok <= hi[t][e & 1] && (tok >= lo[t][e & 1] || tok < a.sinks);
            if (!seen) s[t][b][e] = -INFINITY;
          }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e & 1] = fmaxf(mx[e & 1], s[t][b][e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], off));
      }
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m_new = fmaxf(m_run[t][e], softmax_offset(mx[e]));
        alpha[e] = ex2(m_run[t][e] - m_new);
        m_run[t][e] = m_new;
        l_run[t][e] *= alpha[e];
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float inv = inverse_of_power(vs[b]);
        float pv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[e] = ex2(s[t][b][e] - m_run[t][e & 1]);
          l_run[t][e & 1] = fmaf(pv[e], inv, l_run[t][e & 1]);
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
    cp_async_wait<2 * kStages - 1>();
    __syncwarp();
    if (need_mask) {
      // tokens hidden from all rows meet probability 0, but what their slots hold may be NaN: zeros in their place, and in
      // that of tokens whose page is not held
      const uint32_t stage = ring + n % kStages * kStageBytes + kStepBytes;
      for (int x = lane; x < STEP * (D / 16); x += 32) {
        const int row = x / (D / 16), tok = tok0 + row;
        const bool there = NB == 1 ? held[0] : (row < kKvBlock ? held[0] : held[NB - 1]);
        if (!there || tok > hi_max || (tok < lo_min && tok >= a.sinks)) sts16_zero(stage + place<D>(row, x % (D / 16)));
      }
      __syncwarp();
    }
    constexpr int VP = D >= 128 ? D / 128 : 1;   // pieces of a value row per lane
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        constexpr int kWords = D == 64 ? 2 : 4;
        uint32_t wv[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          // rows 2c, 2c + 1 (exchanged by 64 bytes more; two 64-byte rows share a line), 2c + 8, 2c + 9
          const uint32_t from = (values ^ (t & 1) * 64) + b * (kKvBlock * D) + (t >> 1) * 8 * D + (D == 64 ? 0 : (t & 1) * D) + i * 128;
          if (D == 64) {
            const uint2 x = lds8(from);
            wv[t][0] = x.x;
            wv[t][1] = x.y;
          } else {
            const uint4 x = lds16(from);
            wv[t][0] = x.x; wv[t][1] = x.y; wv[t][2] = x.z; wv[t][3] = x.w;
          }
        }
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {   // dims 4k + 2u, 4k + 2u + 1 of the lane's piece
            const uint32_t x = __byte_perm(wv[0][k], wv[1][k], u == 0 ? 0x5140 : 0x7362);
            const uint32_t y = __byte_perm(wv[2][k], wv[3][k], u == 0 ? 0x5140 : 0x7362);
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
    __syncwarp();                 // every lane has read the values
    fetch(n + kStages, true);
  }
  cp_async_wait<0>();
  __syncthreads();   // every warp is done with its ring
  float* sm_o = reinterpret_cast<float*>(smem);   // [kWarps][R][D + 4]

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
        *reinterpret_cast<float2*>(sm_o + (warp * R + r) * (D + 4) + dim) = make_float2(o[t][jt][e], o[t][jt][e + 2]);
      }
    }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * (D / 4); x += kWarps * 32) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    float m = sm_m[0][r];
#pragma unroll
    for (int v = 1; v < kWarps; ++v) m = fmaxf(m, sm_m[v][r]);
    float l = 0.f, x0 = 0.f, x1 = 0.f, x2 = 0.f, x3 = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      const float f = ex2(sm_m[v][r] - m);
      l += sm_l[v][r] * f;
      const float4 y = *reinterpret_cast<const float4*>(sm_o + (v * R + r) * (D + 4) + d);
      x0 += y.x * f;
      x1 += y.y * f;
      x2 += y.z * f;
      x3 += y.w * f;
    }
    if (run.slot < 0) {
      const int rr = r0 + r;
      const long long row = static_cast<long long>(w.q_row0 + rr / p.group) * a.hq + head * p.group + rr % p.group;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // NaN stays NaN
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + row * D + d) =
          make_uint2(pack2<BF>(x0 * inv, x1 * inv), pack2<BF>(x2 * inv, x3 * inv));
    } else {
      const int part = run.slot * R + r;
      *reinterpret_cast<float4*>(p.part_o + static_cast<long long>(part) * D + d) = make_float4(x0, x1, x2, x3);
      if (d == 0) p.part_ml[part] = make_float2(m, l);
    }
  }
}

// Inclusive sum over the CTA's threads; sm holds kWarps values.
__device__ __forceinline__ int block_scan(int x, int* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  for (int v = 0; v < warp; ++v) x += sm[v];
  return x;
}

template <int D, int NT, bool BF>
__global__ void __launch_bounds__(kWarps * 32, (Tune<D, NT>::kCtas)) attend_kernel(const AttendParams p) {
  constexpr int STEP = Cfg<D>::kStep;
  constexpr int R = NT * 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);  // the warps' rings; then their parts of the output
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];
  __shared__ float4 sm_meta[kWarps][Tune<D, NT>::kStages][Cfg<D>::kBlocks];   // of a block: K scale, V scale, held
  __shared__ int sm_scan[kWarps], sm_at[2], sm_total;
  const Fp8AttendArgs& a = p.a;
  cudaTriggerProgrammaticLaunchCompletion();   // the joining kernel may be launched (it waits for this one's end)
  zero_unclaimed(reinterpret_cast<uint32_t*>(a.out), static_cast<long long>(a.hq) * (D / 2), a.cu_q, a.c.n, a.tq, a.max_q, true,
                 static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x, static_cast<long long>(gridDim.x) * gridDim.y);
  if (a.c.n == 0) return;
  Run run;
  if (p.ctas == 0) {
    run.seq = blockIdx.y;
    run.head = blockIdx.x / p.row_tiles;
    run.tile = blockIdx.x % p.row_tiles;
    const Walk w = walk_of<STEP>(a, run.seq, run.tile * R, run.tile * R + R, p.group, threadIdx.x == 0);
    run.s_begin = 0;
    run.s_end = w.steps;
    run.slot = -1;
    if (w.rows > 0) attend_run<D, NT, BF>(p, w, run, smem, sm_m, sm_l, sm_meta);
    return;
  }
  // ---- the line of steps: key heads, in each the tiles, in each the sequences
  const int entries = p.row_tiles * a.c.n;
  const auto entry = [&](int e) {
    const int tile = e / a.c.n;
    return walk_of<STEP>(a, e % a.c.n, tile * R, tile * R + R, p.group, blockIdx.x == 0);
  };
  int mine = static_cast<int>(threadIdx.x) < entries ? entry(threadIdx.x).steps : 0;
  const int own = mine;                        // of the first kWarps * 32 entries
  for (int e = threadIdx.x + kWarps * 32; e < entries; e += kWarps * 32) mine += entry(e).steps;
  const int upto = block_scan(mine, sm_scan);
  if (threadIdx.x == kWarps * 32 - 1) sm_total = upto;
  __syncthreads();
  const int per_head = sm_total;               // steps of one key head
  const long long total = static_cast<long long>(per_head) * a.c.heads;
  const long long even = (total + p.ctas - 1) / p.ctas;
  const long long share = (max(even, static_cast<long long>(kMinShare)) + kWarps - 1) / kWarps * kWarps;
  long long pos = share * blockIdx.x;
  const long long stop = min(pos + share, total);
  if (pos >= stop) {
    if (threadIdx.x == 0) p.cuts[blockIdx.x] = make_int4(0, 0, -1, 0);
    return;
  }
  run.head = static_cast<int>(pos / per_head);
  int rem = static_cast<int>(pos - static_cast<long long>(run.head) * per_head);
  // the entry that holds step `rem` of the head
  int e = 0, base = 0;
  for (int e0 = 0; e0 < entries; e0 += kWarps * 32) {
    int x = own, incl = upto;
    if (entries > kWarps * 32) {               // else the sum above was this scan
      if (e0 > 0) x = e0 + static_cast<int>(threadIdx.x) < entries ? entry(e0 + threadIdx.x).steps : 0;
      incl = block_scan(x, sm_scan) + base;
    }
    if (rem >= incl - x && rem < incl) {
      sm_at[0] = e0 + threadIdx.x;
      sm_at[1] = rem - (incl - x);
    }
    const bool found = __syncthreads_or(rem >= incl - x && rem < incl);
    if (found) break;
    if (threadIdx.x == kWarps * 32 - 1) sm_at[0] = incl;
    __syncthreads();
    base = sm_at[0];
  }
  e = sm_at[0];
  run.s_begin = sm_at[1];
  int4 begun = make_int4(0, 0, -1, 0);
  for (bool first = true; pos < stop; first = false) {
    const Walk w = entry(e);
    if (w.steps > 0) {
      run.tile = e / a.c.n;
      run.seq = e % a.c.n;
      run.s_end = static_cast<int>(min(static_cast<long long>(w.steps), run.s_begin + (stop - pos)));
      const bool cut = run.s_begin > 0 || run.s_end < w.steps;
      run.slot = cut ? static_cast<int>(blockIdx.x) * 2 + (first ? 0 : 1) : -1;
      if (run.s_begin == 0 && cut)                 // whoever begins a cut sequence says where its parts are
        begun = make_int4(run.seq, run.head * p.row_tiles + run.tile, run.slot, static_cast<int>((pos + w.steps - 1) / share));
      __syncthreads();                            // the last run's parts have been read
      attend_run<D, NT, BF>(p, w, run, smem, sm_m, sm_l, sm_meta);
      pos += run.s_end - run.s_begin;
    }
    run.s_begin = 0;
    if (++e == entries) {
      e = 0;
      ++run.head;
    }
  }
  if (threadIdx.x == 0) p.cuts[blockIdx.x] = begun;   // at most one: it runs past the CTA's end
}

// Joins the parts of cut sequences: CTA (x, y) row y of the one that CTA x began.  The warps take parts in turn, a lane D / 32
// dims; launched while the last parts are still being computed, it waits for them at its start.
template <int D, int R, bool BF>
__global__ void __launch_bounds__(128) join_kernel(const AttendParams p) {
  constexpr int kW = 4;
  const Fp8AttendArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cudaGridDependencySynchronize();
  const int4 cut = p.cuts[blockIdx.x];                     // sequence, key head and tile, first slot, last CTA
  if (cut.z < 0) return;
  const int head = cut.y / p.row_tiles;
  const int rr = cut.y % p.row_tiles * R + blockIdx.y;    // row within the key head
  const Walk w = walk_of<Cfg<D>::kStep>(a, cut.x, rr / R * R, rr / R * R + R, p.group, false);
  if (static_cast<int>(blockIdx.y) >= w.rows) return;
  const int parts = cut.w - static_cast<int>(blockIdx.x) + 1;
  const long long row = static_cast<long long>(w.q_row0 + rr / p.group) * a.hq + head * p.group + rr % p.group;
  const auto place_of = [&](int s) { return (s == 0 ? cut.z : (static_cast<int>(blockIdx.x) + s) * 2) * R + static_cast<int>(blockIdx.y); };
  __shared__ float sm_acc[kW][D];
  __shared__ float sm_l[kW];
  float m = -INFINITY;
  for (int s = lane; s < parts; s += 32) m = fmaxf(m, p.part_ml[place_of(s)].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  float l = 0.f;
  float acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = warp; s < parts; s += kW) {
    const int at = place_of(s);
    const float2 v = p.part_ml[at];
    const float f = ex2(v.x - m);
    l += v.y * f;
    const float* src = p.part_o + static_cast<long long>(at) * D + lane * 2;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float2 y = *reinterpret_cast<const float2*>(src + i * 64);
      acc[2 * i] += y.x * f;
      acc[2 * i + 1] += y.y * f;
    }
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *reinterpret_cast<float2*>(&sm_acc[warp][i * 64 + lane * 2]) = make_float2(acc[2 * i], acc[2 * i + 1]);
  if (lane == 0) sm_l[warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int v = 0; v < kW; ++v) l += sm_l[v];
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + row * D);
  if (threadIdx.x < D / 2) {
    float x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int v = 0; v < kW; ++v) {
      const float2 y = *reinterpret_cast<const float2*>(&sm_acc[v][threadIdx.x * 2]);
      x0 += y.x;
      x1 += y.y;
    }
    out[threadIdx.x] = pack2<BF>(x0 * inv, x1 * inv);
  }
}

int rows_per_tile(const Fp8AttendArgs& a) {
  const long long rows = static_cast<long long>(a.hq / a.c.heads) * a.max_q;
  // d 256: 16 rows convert a code for twice as many rows, which long prompts gain from (28 x 285 queries 350 -> 274 us, 1024
  // queries 235 -> 167), but a step's chain of instructions is longer (16 rows on 4 x 4000 tokens: 25 us, in two tiles 21).
  // 32 rows at d 64 were slower for few rows (32 rows behind a window: 69 against 58 us) and 6 % faster for prompts: left out.
  return rows <= 8 || (a.c.d == 256 && rows <= 32) ? 8 : 16;
}

int resident_ctas(int d, int rows) {
  const int per_sm = d != 64 ? 2 : (rows == 8 ? Tune<64, 1>::kCtas : Tune<64, 2>::kCtas);
  return per_sm * 148;
}

AttendParams plan(const Fp8AttendArgs& a) {
  AttendParams p = {};
  p.a = a;
  p.group = a.hq / a.c.heads;
  const int R = rows_per_tile(a);
  p.row_tiles = static_cast<int>((static_cast<long long>(p.group) * a.max_q + R - 1) / R);
  if (p.row_tiles < 1) p.row_tiles = 1;   // no queries: the rows behind the last sequence are still zeroed
  p.scale_log2 = a.scale * 1.4426950408889634f;
  const int step = a.c.d == 256 ? 16 : 32;
  long long tokens = a.max_kv;
  if (a.window_left >= 0) {
    const long long seen = static_cast<long long>(a.window_left) + R + 2 * step + (static_cast<long long>(a.sinks) + step - 1) / step * step;
    tokens = seen < tokens ? seen : tokens;
  }
  const long long steps = (tokens + step - 1) / step + 1;
  const long long items = static_cast<long long>(a.c.n) * a.c.heads * p.row_tiles;
  const long long resident = resident_ctas(a.c.d, R);
  // behind a window all long sequences are alike: whole ones, if they fill the SMs nearly evenly
  const long long waves = (items + resident - 1) / resident;
  const bool alike = tokens < a.max_kv && items * 4 >= waves * resident * 3;
  const bool countable = steps * a.c.n * p.row_tiles <= 0x7fffffff;   // the line's length per key head is an int
  const bool whole = steps <= (items >= 148 ? 2 : 1) * kDirectSteps + 1;
  if (!whole && !alike && countable && items > 0 && a.max_q > 0) {
    const long long most = steps * items / kMinShare + 1;
    p.ctas = static_cast<int>(most < resident ? most : resident);
  }
  return p;
}

// floats: the slots' outputs, their maxima and row sums, and what the CTAs began
long long workspace_of(const AttendParams& p) {
  if (p.ctas == 0) return 0;
  const long long slots = 2ll * p.ctas * rows_per_tile(p.a);
  return slots * (p.a.c.d + 2) + 4ll * p.ctas;
}

template <int D, int NT, bool BF>
cudaError_t launch(AttendParams p, cudaStream_t s) {
  constexpr int kSmem = Tune<D, NT>::kSmem;
  static std::atomic<uint64_t> ready{0};   // devices that allow the kernel its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!(ready.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(attend_kernel<D, NT, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(uint64_t{1} << (dev & 63), std::memory_order_relaxed);
  }
  if (p.ctas == 0) {
    const long long width = static_cast<long long>(p.a.c.heads) * p.row_tiles;
    if (width > 0x7fffffff) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(width), p.a.c.n > 0 ? p.a.c.n : 1);
    attend_kernel<D, NT, BF><<<grid, kWarps * 32, kSmem, s>>>(p);
    return cudaGetLastError();
  }
  const long long slots = 2ll * p.ctas * NT * 8;
  p.part_o = p.a.part;
  p.part_ml = reinterpret_cast<float2*>(p.a.part + slots * D);
  p.cuts = reinterpret_cast<int4*>(p.part_ml + slots);   // slots is even: 16-byte aligned
  attend_kernel<D, NT, BF><<<p.ctas, kWarps * 32, kSmem, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const long long tile_rows = static_cast<long long>(p.group) * p.a.max_q;
  cfg.gridDim = dim3(p.ctas, static_cast<unsigned>(tile_rows < NT * 8 ? tile_rows : NT * 8));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<D, NT * 8, BF>, p);
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
  if (!attend_ok(a) || a.tq == 0) return 0;
  return workspace_of(plan(a));
}

cudaError_t fp8_attend(const Fp8AttendArgs& a, cudaStream_t s) {
  if (!attend_ok(a)) return cudaErrorInvalidValue;
  if (a.tq == 0) return cudaSuccess;
  const AttendParams p = plan(a);
  if (p.ctas > 0 && a.part == nullptr) return cudaErrorInvalidValue;
  const int rows = rows_per_tile(a);
  if (a.c.d == 64) return rows == 8 ? launch_t<64, 1>(p, s) : launch_t<64, 2>(p, s);
  if (a.c.d == 128) return rows == 8 ? launch_t<128, 1>(p, s) : launch_t<128, 2>(p, s);
  return rows == 8 ? launch_t<256, 1>(p, s) : launch_t<256, 2>(p, s);
}

}  // namespace teb200
