// Attention over the paged 8-bit KV cache (records and pages: kvq_paged.cuh).
// Part of the kvq_lib.cu unity build.
//
// For query row i of a sequence (its new tokens are its last n tokens, row i at
// position len - n + i) and KV head h:
//   t_j = (q . kcode_j) ks_b scale log2(e)            (b the block of token j)
//   p_j = 2^(t_j - m), out = sum_j p_j vs_b vcode_j / sum_j p_j
// over the tokens j <= position, j > position - window. The value scale joins
// the exponent: w_j = 2^(t_j + log2 vs_b - m2 + lift) with m2 the running maximum
// of t_j + log2 vs_b, so that the fp16 weights of the second product are relative
// to the largest contribution p_j vs_b; the softmax sum is sum_j w_j / vs_b in the
// same reference, out = O / that. The lift puts the largest weight at 2^15, near
// fp16's end: weights are normal numbers down to 2^-29 of it and steps of 2^-39
// below (2^-25 and 2^-35 in the kernel of many rows, whose m2 may lag behind), so
// a block whose scale one large channel sets leaves the others' weights their
// bits; only where scales differ by more do the smaller blocks lose them. Codes are
// exact in fp16 (8 bits), fp16 queries too, and bf16 queries once a row is scaled
// by a power of two (elements below 2^-31 of their row's largest lose bits);
// products and sums are fp32. The only other roundings to fewer bits are w_j
// (fp16, relative 2^-12) and the output.
#pragma once
#include <atomic>

#include "kvq_paged.cuh"

namespace kvq {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLift = 15.f;  // log2 of the largest weight (fp16 ends at 65504)

struct AttnArgs {
  View v;
  const void* q;
  int64_t q_tok, q_head;  // strides in elements
  int group, max_new, window;
  float scale_log2;       // softmax scale * log2(e)
  void* out;              // [total, heads * group, D]
  float2* ml;             // [total, heads * group] or null: (max, 1 / sum) of each row
  float* part;            // workspace
  int n_workers;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D (16 x 8, fp32) += A (16 x 16, fp16) B (16 x 8, fp16).
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The four codes of a word as two fp16 pairs (exact).
template <int KIND>
__device__ __forceinline__ void code_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == kInt8) {
    // bytes u = code + 128 under the high byte 0x64 are the fp16 numbers 1024 + u
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t a = prmt(w, 0x64646464u, 0x4140), b = prmt(w, 0x64646464u, 0x4342);
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// First token that a row at `pos` sees. A row before the first token (pos < 0) sees none,
// whatever this says; windows reach INT32_MAX, so pos is clamped before it is subtracted.
__device__ __forceinline__ int first_seen(int pos, int window) {
  return window > 0 ? max(0, max(pos, 0) - window + 1) : 0;
}

// What one call sees of sequence b. A row group is R = 8 * NT query rows (token,
// query head of the KV head's group), row r being token r / group.
struct Seq {
  int slot, len, n, lo_blk, n_blk, groups;
  int64_t r0;
};
// The parts of a Seq that come from memory, kept in shared memory by kernels that
// need a sequence more than once (calls of up to kSeqCache sequences).
constexpr int kSeqCache = 1024;
__device__ __forceinline__ Seq make_seq(const AttnArgs& a, int slot, int len, int n, int64_t r0,
                                        int R) {
  Seq s;
  s.slot = slot;
  s.len = len;
  s.n = n;
  s.r0 = r0;
  s.lo_blk = first_seen(len - n, a.window) / kBlock;
  // an empty sequence still has a (wholly masked) block, which writes its rows
  s.n_blk = n == 0 ? 0 : max(1, (len + kBlock - 1) / kBlock - s.lo_blk);
  s.groups = (int)(((int64_t)n * a.group + R - 1) / R);
  return s;
}

__device__ __forceinline__ Seq load_seq(const AttnArgs& a, int64_t b, int R,
                                        const int4* cache = nullptr) {
  if (cache) {
    const int4 c = cache[b];
    return make_seq(a, c.x, c.y, c.z, c.w, R);
  }
  int64_t r0, r1;
  a.v.rows(b, r0, r1);
  int n = (int)(r1 - r0);
  if (n > a.max_new) {
    atomicOr(&g_status, kStatusBadIndex);
    n = 0;
  }
  const int slot = a.v.slot(b);
  return make_seq(a, slot, slot < 0 ? 0 : a.v.length(slot), n, r0, R);
}

// Work is a flat sequence of 16-token blocks over (sequence, head, row group),
// and worker w of W takes an equal share of it, whatever the lengths are. Each
// unit counts kUnitCost blocks more than it has, its first places: starting and
// ending one takes a warp about 2 us, a block 0.84 us. (Batches of 16 ragged
// sequences measure the same with and without; it is for many short ones.)
// pre[b] = places of the sequences before b, per head. Block-wide; pre has B + 1.
constexpr int kUnitCost = 2;
template <int THREADS>
__device__ __forceinline__ int64_t block_prefix(const AttnArgs& a, int R, int64_t* pre,
                                                int64_t* sums, int4* cache = nullptr) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int64_t base = 0;
  for (int64_t b0 = 0; b0 < a.v.B; b0 += THREADS) {
    const int64_t b = b0 + threadIdx.x;
    int64_t x = 0;
    if (b < a.v.B) {
      const Seq s = load_seq(a, b, R);
      x = (int64_t)(s.n_blk + kUnitCost) * s.groups;
      if (cache) cache[b] = make_int4(s.slot, s.len, s.n, (int)s.r0);
    }
    int64_t incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) sums[wid] = incl;
    __syncthreads();
    int64_t before = base;
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < wid) before += sums[i];
      base += sums[i];
    }
    if (b < a.v.B) pre[b] = before + incl - x;
    __syncthreads();
  }
  if (threadIdx.x == 0) pre[a.v.B] = base;
  __syncthreads();
  return base * a.v.heads;
}

// Workers that a call of `total` blocks keeps busy.
__device__ __forceinline__ int64_t workers_of(const AttnArgs& a, int64_t total) {
  return max((int64_t)1, min((int64_t)a.n_workers, total));
}

__host__ __device__ constexpr int part_floats(int D, int NT) { return 8 * NT * (D + 4); }

// One row group's running state in a warp. Scores are S^T (tokens x rows): lane
// (g, c) = (lane / 4, lane % 4) holds tokens g, g + 8 of rows 2c, 2c + 1 of each
// 8-row tile; outputs are O^T (channels x rows) in the same layout.
template <int D, int NT>
struct State {
  float o[D / 16][NT][4];
  float m[NT][2], m2[NT][2], l[NT][2];
  __device__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.f;
      m[t][0] = m[t][1] = m2[t][0] = m2[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }
  }
};

// Query fragments of a row group: rows in the B operand's columns.
template <int D, int NT, typename T>
__device__ __forceinline__ void load_q(const AttnArgs& a, const Seq& s, int h, int row0, int lane,
                                       uint32_t (&qf)[D / 16][NT][2], float (&qs)[NT][2]) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = row0 + 8 * t + g;
    const bool valid = r < s.n * a.group;
    const T* p = (const T*)a.q + (s.r0 + r / a.group) * a.q_tok +
                 (int64_t)(h * a.group + r % a.group) * a.q_head;
    float f = 1.f, inv = 1.f;
    uint2 w[D / 16];
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      w[j] = valid ? *reinterpret_cast<const uint2*>(p + 16 * j + 4 * c) : make_uint2(0, 0);
    if constexpr (!std::is_same<T, __half>::value) {
      float mx = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const float2 x = to_float2<T>(w[j].x), y = to_float2<T>(w[j].y);
        mx = fmaxf(fmaxf(mx, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // the row's largest value to [2^14, 2^15)
      const int e = max(-100, (int)((__float_as_uint(mx) >> 23) & 255) - 127);
      if (mx > 0.f && mx < INFINITY) {
        f = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        inv = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const float2 x = to_float2<T>(w[j].x), y = to_float2<T>(w[j].y);
        w[j] = make_uint2(half2_bits(x.x * f, x.y * f), half2_bits(y.x * f, y.y * f));
      }
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      qf[j][t][0] = w[j].x;
      qf[j][t][1] = w[j].y;
    }
    // the scores' factor, from the lanes of rows 2c and 2c + 1
    qs[t][0] = a.scale_log2 * __shfl_sync(0xffffffffu, inv, 8 * c);
    qs[t][1] = a.scale_log2 * __shfl_sync(0xffffffffu, inv, 8 * c + 4);
  }
}

// NB blocks of 16 tokens (records rec[], first tokens t0[]) into the state; two at a
// time halve the reductions and give the warp twice the independent work. MASK:
// some token is hidden from some row, or past the end; a null rec hides its block.
template <int D, int KIND, int NT, int NB, bool MASK>
__device__ __forceinline__ void block_step(State<D, NT>& st, const uint8_t* const (&rec)[NB],
                                           const int (&t0)[NB], const uint32_t (&qf)[D / 16][NT][2],
                                           const float (&qs)[NT][2], int len,
                                           const int (&lo)[NT][2], const int (&hi)[NT][2],
                                           int lane) {
  const int g = lane >> 2, c = lane & 3;
  float x[NB][NT][4], lv[NB], ivs[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float s[NT][2][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][0][e] = s[t][1][e] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 k4 = *reinterpret_cast<const uint4*>(rec[n] + 512 * i + 16 * lane);
      const uint32_t w[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        uint32_t a0, a1, a2, a3;
        code_halves<KIND>(w[2 * jj], a0, a2);
        code_halves<KIND>(w[2 * jj + 1], a1, a3);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mma16816(s[t][jj], a0, a1, a2, a3, qf[2 * i + jj][t][0], qf[2 * i + jj][t][1]);
      }
    }
    const float2 sc = *reinterpret_cast<const float2*>(rec[n] + 32 * D);
    lv[n] = __log2f(sc.y);
    ivs[n] = __fdividef(1.f, sc.y);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[n][t][e] = (s[t][0][e] + s[t][1][e]) * (sc.x * qs[t][e & 1]);
        if (MASK) {
          const int j = t0[n] + g + 8 * (e >> 1);
          if (j > hi[t][e & 1] || j < lo[t][e & 1]) x[n][t][e] = -INFINITY;
        }
      }
  }
  uint32_t pb[NB][NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    bool grew = false;
    float alpha[2], ref[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float bm = fmaxf(x[n][t][r], x[n][t][r + 2]);
        st.m[t][r] = fmaxf(st.m[t][r], bm);  // of the lane's tokens; joined at the end
        top = fmaxf(top, bm + lv[n]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float was = st.m2[t][r], now = fmaxf(was, top);
      grew |= now > was;
      const float base = now == -INFINITY ? 0.f : now;
      ref[r] = base - kLift;
      alpha[r] = exp2_approx(was - base);
      st.m2[t][r] = now;
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        st.o[i][t][0] *= alpha[0];
        st.o[i][t][1] *= alpha[1];
        st.o[i][t][2] *= alpha[0];
        st.o[i][t][3] *= alpha[1];
      }
      st.l[t][0] *= alpha[0];
      st.l[t][1] *= alpha[1];
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = exp2_approx(x[n][t][e] + (lv[n] - ref[e & 1]));
      st.l[t][0] = fmaf(w[0] + w[2], ivs[n], st.l[t][0]);
      st.l[t][1] = fmaf(w[1] + w[3], ivs[n], st.l[t][1]);
      pb[n][t][0] = transpose8x8(half2_bits(w[0], w[1]));
      pb[n][t][1] = transpose8x8(half2_bits(w[2], w[3]));
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    uint32_t vmask = 0xffffffffu;
    if (MASK && KIND == kE4m3) {
      // places past the end may hold anything, and 0 times a NaN code is a NaN
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t0[n] + 2 * c + (e & 1) + 8 * (e >> 1) >= len) vmask &= ~(0xffu << (8 * e));
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 v4 = *reinterpret_cast<const uint4*>(rec[n] + 16 * D + 512 * i + 16 * lane);
      const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
      for (int mm = 0; mm < 2; ++mm) {
        uint32_t a0, a1, a2, a3;
        code_halves<KIND>(MASK ? w[2 * mm] & vmask : w[2 * mm], a0, a2);
        code_halves<KIND>(MASK ? w[2 * mm + 1] & vmask : w[2 * mm + 1], a1, a3);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mma16816(st.o[2 * i + mm][t], a0, a1, a2, a3, pb[n][t][0], pb[n][t][1]);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// (max, 1 / sum) of a row in natural units, from the maximum of its scores and its sum
// relative to 2^ref (both in log2 units); a row that sees nothing has (-inf, inf).
__device__ __forceinline__ float2 row_stats(float m, float ref, float l) {
  if (l == 0.f) return make_float2(-INFINITY, INFINITY);
  return make_float2(m * kLn2, __fdiv_rn(1.f, l * exp2f(ref - m)));
}

// 8 consumer warps, and 4 that feed two each. A copy is issued for one lane at a time
// (~190 cycles each), so one warp that fed all eight was what bound the kernel: 1500
// cycles for 8 records, the rate of HBM itself (262144 tokens x 32 heads, passes of a
// graph: 370 us with one, 315 with four).
constexpr int kAttnWarps = 8, kFeeds = 2;
constexpr int kAttnThreads = 32 * (kAttnWarps + kAttnWarps / kFeeds);
constexpr int kSms = 148;

template <int D>
struct Ring {
  // 6 (D = 128) or 11 records per warp, up to 197 KB in flight per SM; the rest of
  // shared memory holds the prefix of up to kMaxSeqs sequences
  static constexpr int kStages = D == 128 ? 6 : 11;
  static constexpr int kBytes = kAttnWarps * kStages * rec_bytes(D);
};

template <int D>
struct AttnSmem {
  alignas(128) uint8_t ring[kAttnWarps][Ring<D>::kStages][rec_bytes(D)];
  uint64_t full[kAttnWarps][Ring<D>::kStages], empty[kAttnWarps][Ring<D>::kStages];
  int skip[kAttnWarps][Ring<D>::kStages];
  int abort;
  int64_t sums[32];
  alignas(16) int64_t pre[2];  // B + 1, then the sequences (16 bytes each)
};

// Where a worker stands in its share of the blocks.
struct Cursor {
  int64_t x, end;
  int64_t b;
  Seq s;
  int unit, blk0, n;
  // The next piece (blocks of one unit); false when the share is done.
  __device__ bool next(const AttnArgs& a, int R, const int64_t* pre, const int4* cache) {
    n = 0;
    while (x < end && n == 0) find(a, R, pre, cache);
    return n > 0;
  }
  __device__ void find(const AttnArgs& a, int R, const int64_t* pre, const int4* cache) {
    int64_t lo = 0, hi = a.v.B;  // largest b with pre[b] * heads <= x
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (pre[mid] * a.v.heads <= x) lo = mid;
      else hi = mid;
    }
    b = lo;
    s = load_seq(a, b, R, cache);
    const int len = s.n_blk + kUnitCost;
    const int64_t rem = x - pre[b] * a.v.heads;
    unit = (int)(rem / len);
    const int at = (int)(rem % len), to = (int)min((int64_t)len, at + (end - x));
    x += to - at;
    blk0 = max(at - kUnitCost, 0);
    n = max(to - kUnitCost, 0) - blk0;
  }
};

// One CTA per SM. Every consumer warp works through its own share of the blocks
// with its own ring of records, so no warp waits for another one; a lane of a
// feeding warp keeps each ring full: one bulk copy per record, on across the ends of
// units. Bound by HBM: 262144 tokens x 32 heads, 2.16 GB, take 316 us once 512 MB of
// something else have been read (6.8 TB/s; a copy, which writes as much as it reads,
// measures 6.55), 347 after 512 MB have been written, 322 to 357 a call in long runs of
// them; 16 sequences of up to 8192, 0.145 GB, 37 us, of which ~7 pass before the first
// record, ~5 in the join, and the last SM ends ~5 after the median one. 16 rows at D = 128
// spill about 200 bytes a thread (168 registers), 8 rows nothing.
template <int D, int KIND, int NT, typename T>
__global__ void __launch_bounds__(kAttnThreads, 1) attend_kernel(AttnArgs a) {
  constexpr int R = 8 * NT, S = Ring<D>::kStages;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  AttnSmem<D>& sm = *reinterpret_cast<AttnSmem<D>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < kAttnWarps * S) {
    sm100::mbar_init(&sm.full[0][0] + threadIdx.x, 1);
    sm100::mbar_init(&sm.empty[0][0] + threadIdx.x, 1);
  }
  if (threadIdx.x == 0) sm.abort = 0;
  sm100::fence_mbar_init();
  wait_previous();
  let_next_start();  // only now: the join reads lengths before its own wait
  int4* cache =
      a.v.B <= kSeqCache ? reinterpret_cast<int4*>(sm.pre + ((a.v.B + 2) & ~1ll)) : nullptr;
  const int64_t total =
      block_prefix<kAttnThreads>(a, R, sm.pre, sm.sums, cache);  // syncs the block
  if (total == 0) return;
  const int64_t W = workers_of(a, total);
  volatile int* abort = &sm.abort;

  if (warp >= kAttnWarps) {
    // a lane feeds warp `to`; lanes poll, none waits for another one's ring
    const int to = (warp - kAttnWarps) * kFeeds + lane % kFeeds;
    const int64_t w = (int64_t)to * gridDim.x + blockIdx.x;
    Cursor c;
    c.x = c.end = 0;
    if (lane < kFeeds && w < W) {
      c.x = total * w / W;
      c.end = total * (w + 1) / W;
    }
    bool more = c.next(a, R, sm.pre, cache);
    uint32_t k = 0;  // records issued
    int i = 0, col = 0, in_page = 0, ahead = -1;
    const uint8_t *page = nullptr, *rec = nullptr;
    // The next record's address is ready before its place is, and the table is read
    // a page ahead, so that a lane that polls waits for no memory.
    auto page_id = [&](int at) {
      return at * a.v.blocks * kBlock < c.s.len ? a.v.table[(int64_t)c.s.slot * a.v.n_cols + at]
                                                : -1;
    };
    auto take_page = [&]() {
      const int p = ahead;
      ahead = page_id(col + 1);
      if (p >= 0 && p < a.v.n_pages) {
        page = a.v.pool + p * a.v.page_bytes() + c.unit / c.s.groups * a.v.head_bytes();
      } else {
        page = nullptr;
        if (c.s.len > 0) atomicOr(&g_status, kStatusBadIndex);
      }
    };
    auto find_record = [&]() {  // of block i of the piece
      if (i == 0) {
        const int blk = c.s.lo_blk + c.blk0;
        col = blk / a.v.blocks;
        in_page = blk % a.v.blocks;
        ahead = page_id(col);
        take_page();
      } else if (++in_page == a.v.blocks) {
        in_page = 0;
        ++col;
        take_page();
      }
      rec = page ? page + (int64_t)in_page * rec_bytes(D) : nullptr;
    };
    if (more) find_record();
    uint32_t polls = 0;
    unsigned long long t0 = 0;
    while (__any_sync(0xffffffffu, more)) {
      if (more) {
        const int st = k % S;
        if (k < S || sm100::mbar_poll(&sm.empty[to][st], (k / S - 1) & 1)) {
          sm.skip[to][st] = rec == nullptr;
          if (rec) {
            sm100::mbar_arrive_expect_tx(&sm.full[to][st], rec_bytes(D));
            sm100::bulk_g2s(sm.ring[to][st], rec, rec_bytes(D), &sm.full[to][st]);
          } else {
            sm100::mbar_arrive(&sm.full[to][st]);
          }
          ++k;
          if (++i == c.n) {
            i = 0;
            more = c.next(a, R, sm.pre, cache);
          }
          if (more) find_record();
          polls = 0;
        } else if ((++polls & 255) == 0) {  // the clock is slow to read
          if (polls == 256) t0 = sm100::global_ns();
          if (*abort || sm100::global_ns() - t0 > sm100::kWaitLimitNs) {
            *abort = 1;
            atomicOr(&g_status, 2);
            more = false;
          }
        }
      }
      __syncwarp();
    }
    // the copies still in flight land before the block's memory is given up
    for (int j = 0; j < S; ++j) {
      const uint32_t q = k - 1 - j;
      if (k == 0 || (uint32_t)j >= k) break;
      t0 = sm100::global_ns();
      while (!sm100::mbar_test(&sm.full[to][q % S], (q / S) & 1) &&
             sm100::global_ns() - t0 < sm100::kWaitLimitNs) {
      }
    }
    return;
  }

  const int64_t w = (int64_t)warp * gridDim.x + blockIdx.x;
  if (w >= W) return;
  Cursor cur;
  cur.x = total * w / W;
  cur.end = total * (w + 1) / W;
  const int g = lane >> 2, c = lane & 3;
  uint32_t k = 0;
  while (cur.next(a, R, sm.pre, cache)) {
    const Seq& s = cur.s;
    const int n = cur.n, h = cur.unit / s.groups, row0 = cur.unit % s.groups * R;
    uint32_t qf[D / 16][NT][2];
    float qs[NT][2];
    load_q<D, NT, T>(a, s, h, row0, lane, qf, qs);
    int lo[NT][2], hi[NT][2];
    const int rows = s.n * a.group;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = row0 + 8 * t + 2 * c + r, pos = s.len - s.n + row / a.group;
        hi[t][r] = row < rows ? pos : -1;
        lo[t][r] = first_seen(pos, a.window);
      }
    // tokens [see_lo, see_hi] are visible to every row of the group
    const int see_hi = s.len - s.n + row0 / a.group;
    const int last = s.len - s.n + (min(row0 + R, rows) - 1) / a.group;
    const int see_lo = first_seen(last, a.window);
    State<D, NT> st;
    st.clear();
    auto visible = [&](int t0) { return t0 >= see_lo && t0 + kBlock - 1 <= see_hi; };
    for (int i = 0; i < n;) {
      const int t0 = (s.lo_blk + cur.blk0 + i) * kBlock;
      const int s0 = k % S, s1 = (k + 1) % S;
      if (!sm100::mbar_wait(&sm.full[warp][s0], (k / S) & 1, abort)) return;
      const uint8_t* r0 = sm.ring[warp][s0];
      bool pair = i + 1 < n;
      if (pair) {
        if (!sm100::mbar_wait(&sm.full[warp][s1], ((k + 1) / S) & 1, abort)) return;
        pair = !sm.skip[warp][s0] && !sm.skip[warp][s1];
      }
      if (pair) {
        const uint8_t* const rec[2] = {r0, sm.ring[warp][s1]};
        const int at[2] = {t0, t0 + kBlock};
        if (visible(t0) && visible(t0 + kBlock))
          block_step<D, KIND, NT, 2, false>(st, rec, at, qf, qs, s.len, lo, hi, lane);
        else
          block_step<D, KIND, NT, 2, true>(st, rec, at, qf, qs, s.len, lo, hi, lane);
      } else if (!sm.skip[warp][s0]) {
        const uint8_t* const rec[1] = {r0};
        const int at[1] = {t0};
        block_step<D, KIND, NT, 1, true>(st, rec, at, qf, qs, s.len, lo, hi, lane);
      }
      const int used = pair ? 2 : 1;
      __syncwarp();
      if (lane < used) sm100::mbar_arrive(&sm.empty[warp][lane ? s1 : s0]);
      i += used;
      k += used;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int o = 4; o <= 16; o *= 2) {
          st.l[t][r] += __shfl_xor_sync(0xffffffffu, st.l[t][r], o);
          st.m[t][r] = fmaxf(st.m[t][r], __shfl_xor_sync(0xffffffffu, st.m[t][r], o));
        }
    const bool whole = n == s.n_blk;  // the whole unit: its rows are done
    float* p = a.part + (2 * w + (cur.blk0 == 0)) * part_floats(D, NT);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int at_row = 8 * t + 2 * c + r, row = row0 + at_row;
        if (row >= rows) continue;
        if (whole) {
          const int64_t at = (s.r0 + row / a.group) * ((int64_t)a.v.heads * a.group) +
                             h * a.group + row % a.group;
          const float inv = st.l[t][r] == 0.f ? 0.f : __fdiv_rn(1.f, st.l[t][r]);
          T* out = (T*)a.out + at * D;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            out[16 * i + g] = from_float<T>(st.o[i][t][r] * inv);
            out[16 * i + 8 + g] = from_float<T>(st.o[i][t][r + 2] * inv);
          }
          if (a.ml && g == 0) a.ml[at] = row_stats(st.m[t][r], st.m2[t][r] - kLift, st.l[t][r]);
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            p[at_row * D + 16 * i + g] = st.o[i][t][r];
            p[at_row * D + 16 * i + 8 + g] = st.o[i][t][r + 2];
          }
          if (g == 0)
            *reinterpret_cast<float4*>(p + R * D + 4 * at_row) =
                make_float4(st.m2[t][r], st.l[t][r], st.m[t][r], 0.f);
        }
      }
  }
}

// A warp's part of joining the n pieces of a row: pieces part, part + split, ..,
// weighted by 2^(their reference - the largest of all). piece(i) gives the place of
// piece i, its rows first, then (reference, sum, maximum, -) of each. The lane's
// channels are C * lane .. + C - 1; l is the lane's share of the sum.
template <int D, typename Piece>
__device__ __forceinline__ void join_row(int n, int part, int split, int rows, int r, Piece piece,
                                         int lane, float (&o)[D / 32], float& m, float& m2,
                                         float& l) {
  constexpr int C = D / 32;
  m = m2 = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) o[i] = 0.f;
  auto load = [&](int i, float (&x)[C]) {
    const float* p = piece(i) + r * D + C * lane;
    if constexpr (C == 4) {
      const float4 y = *reinterpret_cast<const float4*>(p);
      x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(p);
      x[0] = y.x; x[1] = y.y;
    }
  };
  // the first pieces and all statistics are fetched together
  constexpr int kAhead = 4;
  float first[kAhead][C];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (part + split * i < n) load(part + split * i, first[i]);
  float4 own = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);  // of piece part + split * lane
  if (part + split * lane < n)
    own = *reinterpret_cast<const float4*>(piece(part + split * lane) + rows * D + 4 * r);
  m2 = own.x;
  m = own.z;
  if (split > 1 || n > 32) {
#pragma unroll 4
    for (int i = lane; i < n; i += 32) {
      const float4 q = *reinterpret_cast<const float4*>(piece(i) + rows * D + 4 * r);
      m2 = fmaxf(m2, q.x);
      m = fmaxf(m, q.z);
    }
  }
  m2 = warp_max(m2);
  m = warp_max(m);
  const float ref = m2 == -INFINITY ? 0.f : m2;
  for (int i0 = part; i0 < n; i0 += 32 * split) {  // pieces i0, i0 + split, ..
    float f = 0.f;
    const int mine = i0 + split * lane;
    if (mine < n) {
      const float4 q =
          i0 == part ? own : *reinterpret_cast<const float4*>(piece(mine) + rows * D + 4 * r);
      f = exp2_approx(q.x - ref);
      l = fmaf(q.y, f, l);
    }
    const int k = min(32, (n - i0 + split - 1) / split);
    int i = 0;
    if (i0 == part) {
#pragma unroll
      for (; i < kAhead; ++i) {
        const float w = __shfl_sync(0xffffffffu, f, i);
        if (i < k)
#pragma unroll
          for (int e = 0; e < C; ++e) o[e] = fmaf(first[i][e], w, o[e]);
      }
    }
#pragma unroll 8
    for (; i < k; ++i) {
      const float w = __shfl_sync(0xffffffffu, f, i);
      float x[C];
      load(i0 + split * i, x);
#pragma unroll
      for (int e = 0; e < C; ++e) o[e] = fmaf(x[e], w, o[e]);
    }
  }
}

// A joined row's output and statistics (l: the whole sum, relative to 2^ref).
template <int D, typename T>
__device__ __forceinline__ void store_row(const AttnArgs& a, int64_t at, int lane,
                                          const float (&o)[D / 32], float m, float ref, float l) {
  const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
  T* out = (T*)a.out + at * D + D / 32 * lane;
#pragma unroll
  for (int e = 0; e < D / 32; e += 2)
    *reinterpret_cast<uint32_t*>(out + e) =
        l == 0.f ? 0u : from_float2<T>(o[e] * inv, o[e + 1] * inv);
  if (a.ml && lane == 0) a.ml[at] = row_stats(m, ref, l);
}

// Joins the pieces of the units that several workers share, in a fixed order. A
// CTA takes `rows` of the unit_rows rows that a unit can have, 4 / rows warps each
// (few units have many pieces); a lane adds D / 32 channels of its warp's pieces,
// 32 weights at a time. Four warps fit beside an attention CTA (eight do not: the
// registers), so the CTAs are there, lengths read, when the last piece is written.
constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32;

template <int D, int NT, typename T>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(AttnArgs a, int unit_rows, int rows) {
  constexpr int R = 8 * NT, C = D / 32;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  int64_t* pre = reinterpret_cast<int64_t*>(smem_raw);
  __shared__ int64_t sums[32];
  __shared__ float acc[kJoinWarps][D], sum[kJoinWarps];
  let_next_start();
  // the attention kernel has waited for whatever writes lengths and rows, so they are
  // read ahead of the wait for it
  const int64_t total = block_prefix<kJoinThreads>(a, R, pre, sums);
  const int64_t W = workers_of(a, total);
  const int64_t b = blockIdx.y;
  const Seq s = load_seq(a, b, R);
  const int split = kJoinWarps / rows, wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_unit = unit_rows / rows;
  const int first = (int)(blockIdx.x % per_unit) * rows, unit = blockIdx.x / per_unit;
  const int r = first + wid / split, part = wid % split;
  const int h = unit / max(1, s.groups), row = unit % max(1, s.groups) * R + r;
  // worker w holds the places [total w / W, total (w + 1) / W)
  const int64_t x1 = pre[b] * a.v.heads + (int64_t)(unit + 1) * (s.n_blk + kUnitCost);
  const int64_t x0 = x1 - s.n_blk;
  const bool here = total > 0 && unit < s.groups * a.v.heads && row < s.n * a.group;
  const int64_t w0 = here ? ((x0 + 1) * W - 1) / total : 0;
  const int64_t w1 = here ? (x1 * W - 1) / total : 0;
  wait_previous();
  const int n = w1 > w0 ? (int)(w1 - w0) + 1 : 0;  // the row's pieces (0: nothing to join)
  float m, m2, l, o[C];
  // the first piece is its worker's last, the others their workers' first
  join_row<D>(
      n, part, split, R, r,
      [&](int i) { return a.part + (2 * (w0 + i) + (i == 0)) * part_floats(D, NT); }, lane, o, m,
      m2, l);
  l = warp_sum(l);
  if (split > 1) {
#pragma unroll
    for (int e = 0; e < C; ++e) acc[wid][C * lane + e] = o[e];
    if (lane == 0) sum[wid] = l;
    __syncthreads();
    if (part) return;
    for (int i = 1; i < split; ++i) {
#pragma unroll
      for (int e = 0; e < C; ++e) o[e] += acc[wid + i][C * lane + e];
      l += sum[wid + i];
    }
  }
  if (n == 0) return;
  const int64_t at = (s.r0 + row / a.group) * ((int64_t)a.v.heads * a.group) + h * a.group +
                     row % a.group;
  store_row<D, T>(a, at, lane, o, m, m2 - kLift, l);
}

// Rows of a call's largest sequence: 8-row tiles where one is enough, up to three
// groups of two, else (0) the 128-row tiles of kvq_paged_tile.cuh. 23 sequences of up
// to 6000 tokens, window 2500, D = 64 / 128: 48 rows 75 / 109 us in groups against
// 101 / 136 in tiles, 64 rows 108 / 137 against 102 / 141; one of 32768 tokens: 32
// rows 51 against 62, 64 rows 77 against 65.
constexpr int kGroupRows = 48;
inline int row_tiles(int64_t max_new, int64_t group) {
  return max_new * group <= 8 ? 1 : max_new * group <= kGroupRows ? 2 : 0;
}

// Allows `kernel` `bytes` of dynamic shared memory on the current device; `done` is
// the kernel's own set of the devices where that has been said already.
template <typename K>
static void allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) ==
      cudaSuccess)
    done.fetch_or(bit, std::memory_order_relaxed);
}

template <int D, int KIND, int NT, typename T>
static int launch_attend(AttnArgs a, cudaStream_t st) {
  const int64_t groups = ((int64_t)a.max_new * a.group + 8 * NT - 1) / (8 * NT);
  a.n_workers = kSms * kAttnWarps;
  const int64_t cached = a.v.B <= kSeqCache ? a.v.B : 0;
  const int smem = (int)(sizeof(AttnSmem<D>) + a.v.B * sizeof(int64_t) + cached * sizeof(int4));
  static_assert(sizeof(AttnSmem<D>) + kMaxSeqs * sizeof(int64_t) <= 227 * 1024 &&
                    kSeqCache * (sizeof(int64_t) + sizeof(int4)) <= kMaxSeqs * sizeof(int64_t),
                "shared memory");
  static std::atomic<uint64_t> done{0};
  allow_smem(attend_kernel<D, KIND, NT, T>, 227 * 1024, done);
  int rc = launch_next("paged_attention", attend_kernel<D, KIND, NT, T>, dim3(kSms), kAttnThreads,
                       smem, st, a);
  if (rc) return rc;
  // rows per CTA: as few CTAs as keep the SMs busy, for they start beside the last
  // attention CTAs
  int unit_rows = 1;
  while (unit_rows < 8 * NT && unit_rows < (int64_t)a.max_new * a.group) unit_rows *= 2;
  const int64_t units = groups * a.v.heads * a.v.B;
  int rows = unit_rows < kJoinWarps ? unit_rows : kJoinWarps;
  while (rows > 1 && units * (unit_rows / rows) * 2 <= kSms) rows /= 2;
  const dim3 grid((unsigned)(groups * a.v.heads * (unit_rows / rows)), (unsigned)a.v.B);
  return launch_next("paged_attention (join)", attend_join_kernel<D, NT, T>, grid, kJoinThreads,
                     (int)((a.v.B + 1) * sizeof(int64_t)), st, a, unit_rows, rows);
}

}  // namespace paged
}  // namespace kvq
