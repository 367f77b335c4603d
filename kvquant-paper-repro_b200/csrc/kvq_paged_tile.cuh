// Attention over the paged 8-bit KV cache for many query rows (prompt chunks,
// drafted tokens): tcgen05 matrix products with TMEM accumulators. Part of the
// kvq_lib.cu unity build; arithmetic as in kvq_paged_attn.cuh.
//
// A unit is 256 query rows (token, head of the group) of one KV head, in two
// tiles of 128 rows that take turns on the tensor core: while one tile's softmax
// runs, the other tile's products do. Keys and values come in tiles of 128
// tokens:
//   S_t = Q_t K^T          A = Q_t (shared), B = K (shared), both K-major
//   O_t += P_t V           A = P_t (TMEM, over S_t's columns), B = V^T (shared)
// Warps: 0-3 and 4-7 the softmax of tile 0 and 1 (a thread owns a row), 8-11 turn
// records into fp16 tiles, 12 issues the products, 13 fetches records. The
// record order makes each 4-byte value word a row segment of a core matrix, so
// a warp writes whole 128-byte core matrices without bank conflicts.
// One CTA per SM takes an equal share of all (unit, token tile) pairs; a unit
// cut by a share's end is joined by tile_join_kernel. Two chunks of 2048 tokens x 4
// heads over 8200 and 10007 tokens, 8 KV heads: 754 us = 0.78 PFLOP/s, 47 % of the
// measured bf16 rate. A token tile takes about 5500 cycles: a tile's softmax ~3300 and
// its rescalings of O (MUFU 1024, two warps to a partition) and then its 16 products ~1900
// follow each other, and the two tiles overlap only in part. Two issuing warps, one per
// tile, were slower (951 us against 725 then): their products interleave and both
// softmaxes fall together. About 110 bytes a thread spill.
#pragma once
#include "kvq_paged_attn.cuh"

namespace kvq {
namespace paged {

constexpr int kTileRows = 128, kUnitRows = 256, kTileTok = 128;
constexpr int kTileRecs = kTileTok / kBlock;  // records of a token tile
constexpr int kGroupRecs = 4, kGroups = 4;  // records come in groups of 64 tokens
constexpr int kRawStages = kGroups * kGroupRecs, kSlots = 3;
constexpr int kTileThreads = 16 * 32;  // warps 14 and 15 only complete their warpgroup
// Registers per thread of the warpgroups (softmax twice, dequantising, products and
// copies): together the 4 x 128 of the launch. The softmax keeps a row's 128 scores.
constexpr int kRegsSoftmax = 192, kRegsDequant = 80, kRegsIssue = 48;
static_assert(2 * kRegsSoftmax + kRegsDequant + kRegsIssue <= 4 * 128, "register shares");
constexpr int kDequantWarp = 8, kMmaWarp = 12, kLoadWarp = 13;
constexpr int64_t kTileParts = 2 * kSms;  // pieces in the workspace, then B + 1 int32
// The maximum may grow by 2^kLazy before O is rescaled, and weights are lifted by that
// much less: together 2^15.875, below fp16's end. (Two chunks of 2048 tokens: 728 us at 8
// without a lift, 767 at 4; what a rescaling costs is a pass over O in TMEM.)
constexpr float kTileLift = 11.f, kLazy = 4.875f;

template <int D>
struct TileSmem {
  alignas(128) uint8_t q[2][kTileRows * D * 2];
  alignas(128) uint8_t slot[kSlots][kTileTok * D * 2];  // K and V tiles in turn
  alignas(128) uint8_t raw[kRawStages][rec_bytes(D)];
  uint64_t raw_full[kGroups], raw_empty[kGroups];
  uint64_t slot_full[kSlots], slot_empty[kSlots];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], drain;
  float4 scale[2][kTileRecs];  // (key scale, log2 value scale, 1 / value scale, -) of a tile
  int64_t sums[32];
  int skip[kRawStages];
  uint32_t tmem;
  int abort;
};

// Token tiles [t0, t0 + n) that row group r of a sequence sees (at least one).
__device__ __forceinline__ void unit_tiles(const AttnArgs& a, const Seq& s, int r, int& t0,
                                           int& n) {
  const int p0 = s.len - s.n + (int)((int64_t)r * kUnitRows / a.group);
  const int p1 = s.len - s.n +
                 min(s.n - 1, (int)(((int64_t)r * kUnitRows + kUnitRows - 1) / a.group));
  t0 = first_seen(p0, a.window) / kTileTok;
  n = max(1, max(p1, 0) / kTileTok - t0 + 1);
}

// As block_prefix, over token tiles; pre may be in global memory, where every CTA
// writes the same values and reads its own.
template <int THREADS>
__device__ __forceinline__ int64_t tile_prefix(const AttnArgs& a, int32_t* pre, int64_t* sums) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int64_t base = 0;
  for (int64_t b0 = 0; b0 < a.v.B; b0 += THREADS) {
    const int64_t b = b0 + threadIdx.x;
    int64_t x = 0;
    if (b < a.v.B) {
      const Seq s = load_seq(a, b, kUnitRows);
      for (int r = 0; r < s.groups; ++r) {
        int t0, n;
        unit_tiles(a, s, r, t0, n);
        x += n;
      }
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
    if (b < a.v.B) pre[b] = (int32_t)(before + incl - x);
    __syncthreads();
  }
  if (threadIdx.x == 0) pre[a.v.B] = (int32_t)base;
  __syncthreads();
  if (base > INT32_MAX) {  // more work than any call has: refused
    if (threadIdx.x == 0) atomicOr(&g_status, kStatusBadIndex);
    return 0;
  }
  return base * a.v.heads;
}

__device__ __forceinline__ int64_t tile_workers(int64_t total) {
  return max((int64_t)1, min((int64_t)kSms, total));
}

struct TileCursor {
  int64_t x, end;
  Seq s;
  int h, row0, t0, n_unit, first, n;  // piece: tiles [first, first + n) of the unit's n_unit
  // Warp-collective.
  __device__ bool next(const AttnArgs& a, const int32_t* pre, int lane) {
    if (x >= end) return false;
    int64_t lo = 0, hi = a.v.B;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if ((int64_t)pre[mid] * a.v.heads <= x) lo = mid;
      else hi = mid;
    }
    s = load_seq(a, lo, kUnitRows);
    const int64_t per = pre[lo + 1] - pre[lo];
    const int64_t rem64 = x - (int64_t)pre[lo] * a.v.heads;
    h = (int)(rem64 / per);
    int rem = (int)(rem64 % per);
    for (int r0 = 0;; r0 += 32) {
      int mt0 = 0, mn = 0;
      if (r0 + lane < s.groups) unit_tiles(a, s, r0 + lane, mt0, mn);
      int incl = mn;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, incl > rem);
      if (past || r0 + 32 >= s.groups) {
        const int l = past ? __ffs(past) - 1 : 31;
        t0 = __shfl_sync(0xffffffffu, mt0, l);
        n_unit = __shfl_sync(0xffffffffu, mn, l);
        first = rem - (__shfl_sync(0xffffffffu, incl, l) - n_unit);
        row0 = (r0 + l) * kUnitRows;
        break;
      }
      rem -= __shfl_sync(0xffffffffu, incl, 31);
    }
    n = (int)min((int64_t)(n_unit - first), end - x);
    x += n;
    return true;
  }
  __device__ int tiles(const AttnArgs& a) const {  // halves of the unit that have rows
    return s.n * a.group - row0 > kTileRows ? 2 : 1;
  }
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
        "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
      : "memory");
}

// A query row to shared memory as fp16 (rows of the A operand, core matrices
// [D / 8][row / 8]); returns the factor of its scores. Negative softmax scales
// turn the row's sign, so the factor is >= 0 and maxima keep their meaning.
template <int D, typename T>
__device__ __forceinline__ float stage_q(const AttnArgs& a, const T* p, bool valid, uint8_t* q,
                                         int row) {
  uint4 w[D / 8];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
    w[i] = valid ? *reinterpret_cast<const uint4*>(p + 8 * i) : make_uint4(0, 0, 0, 0);
  float f = 1.f, inv = 1.f;
  if constexpr (!std::is_same<T, __half>::value) {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = to_float2<T>(x[e]);
        mx = fmaxf(mx, fmaxf(fabsf(y.x), fabsf(y.y)));
      }
    }
    const int e = max(-100, (int)((__float_as_uint(mx) >> 23) & 255) - 127);
    if (mx > 0.f && mx < INFINITY) {
      f = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
      inv = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
    }
  }
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (!std::is_same<T, __half>::value) {
        const float2 y = to_float2<T>(x[e]);
        x[e] = half2_bits(y.x * f, y.y * f);
      }
      x[e] ^= sign;
    }
    *reinterpret_cast<uint4*>(q + i * (kTileRows * 16) + (row >> 3) * 128 + (row & 7) * 16) =
        make_uint4(x[0], x[1], x[2], x[3]);
  }
  return fabsf(a.scale_log2) * inv;
}

// One lane of a converged warp, always the same one. Under this predicate (unlike
// lane == 0) the compiler keeps the operands of a product in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// Two fp32 operations in one instruction (each rounded as the scalar one).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Softmax state of a thread's row: the maximum of the scores, the reference of
// the weights and the sum relative to it (log2 units).
struct RowState {
  float m, ref, l;
};

// One tile of a row: scores from TMEM, weights back over the first half of their
// columns. masked: some row of the warp does not see all 128 tokens; the row sees
// the columns c with (unsigned)(c + first) <= span. The factors of the scores are
// kept above 0, so that a hidden score of -inf stays one.
constexpr float kLeastFactor = 0x1p-100f;
template <int D>
__device__ __forceinline__ void softmax_tile(RowState& st, uint32_t ts, uint32_t to, bool has_o,
                                             const float4* sc, float qs, bool masked, int first,
                                             uint32_t span) {
  using namespace sm100;
  float top = -INFINITY;
  uint32_t x[4][32];
#pragma unroll
  for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, x[q]);
  tmem_wait_ld();
  if (masked) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if ((uint32_t)(first + 32 * q + e) > span) x[q][e] = 0xff800000u;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint32_t* y = x[q] + 16 * b;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(y[e]);
#pragma unroll
      for (int e = 4; e < 16; e += 4)
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = fmaxf(v[z], __uint_as_float(y[e + z]));
      const float bm = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
      const float4 f = sc[2 * q + b];
      const float tm = bm * fmaxf(f.x * qs, kLeastFactor);
      st.m = fmaxf(st.m, tm);
      top = fmaxf(top, tm + f.y);
    }
  }
  if (__any_sync(0xffffffffu, top > st.ref + kLazy)) {
    const float now = fmaxf(st.ref, top);
    const float alpha = now == -INFINITY ? 1.f : exp2_approx(st.ref - now);
    st.ref = now;
    st.l *= alpha;
    if (has_o) {
#pragma unroll 1
      for (int q = 0; q < D / 16; ++q) {
        uint32_t o[16];
        tmem_ld_32x32b_x16(to + 16 * q, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
        tmem_st16(to + 16 * q, o);
      }
    }
  }
  const float base = (st.ref == -INFINITY ? 0.f : st.ref) - kTileLift;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t p[16];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float4 f = sc[2 * q + b];
      const float fk = fmaxf(f.x * qs, kLeastFactor), fv = f.y - base;
      const uint64_t fk2 = pack2(fk, fk), fv2 = pack2(fv, fv);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float y0, y1;
        unpack2(fma2(pack2(__uint_as_float(x[q][16 * b + e]), __uint_as_float(x[q][16 * b + e + 1])),
                     fk2, fv2),
                y0, y1);
        y0 = exp2_approx(y0);
        y1 = exp2_approx(y1);
        sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pack2(y0, y1));
        p[8 * b + e / 2] = half2_bits(y0, y1);
      }
      float s0, s1;
      unpack2(add2(sum[0], sum[1]), s0, s1);
      st.l = fmaf(s0 + s1, f.z, st.l);
    }
    tmem_st16(ts + 16 * q, p);
  }
  tmem_wait_st();
}

template <int D, int KIND, typename T>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tile_kernel(AttnArgs a) {
  using namespace sm100;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  TileSmem<D>& sm = *reinterpret_cast<TileSmem<D>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  volatile int* abort = &sm.abort;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kGroups; ++i) {
      mbar_init(&sm.raw_full[i], 1);
      mbar_init(&sm.raw_empty[i], kGroupRecs);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sm.slot_full[i], 4);
      mbar_init(&sm.slot_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm.q_full[t], kTileRows);
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.p_full[t], kTileRows);
      mbar_init(&sm.o_full[t], 1);
    }
    mbar_init(&sm.drain, 1);
    *abort = 0;
    fence_mbar_init();
  }
  wait_previous();
  let_next_start();  // only now: the join reads lengths before its own wait
  int32_t* pre = reinterpret_cast<int32_t*>(a.part + kTileParts * kUnitRows * (D + 4));
  const int64_t total = tile_prefix<kTileThreads>(a, pre, sm.sums);  // syncs the block
  const int64_t W = tile_workers(total);
  if (total == 0 || blockIdx.x >= W) return;
  if (warp == kMmaWarp) tmem_alloc(&sm.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // S_t at columns 128 t, O_t at 256 + D t: the whole TMEM is allocated, from 0
  TileCursor c;
  c.x = total * blockIdx.x / W;
  c.end = total * (blockIdx.x + 1) / W;
  uint32_t gi = 0;  // token tiles before the current one

  // A lane is issued one copy at a time (~190 cycles), so records that lie one after
  // another in a page come in one copy: a group is one to four copies.
  auto load_role = [&]() {
    uint32_t groups = 0;
    bool ok = true;
    while (ok && c.next(a, pre, lane)) {
      for (int i = 0; ok && i < 2 * c.n; ++i, ++groups) {
        const uint32_t st = groups % kGroups, use = groups / kGroups;
        if (use > 0 && !mbar_wait(&sm.raw_empty[st], (use - 1) & 1, abort)) {
          ok = false;
          break;
        }
        const int blk = (c.t0 + c.first) * kTileRecs + i * kGroupRecs + lane;
        const uint8_t* rec = lane < kGroupRecs && blk * kBlock < c.s.len
                                 ? a.v.record(c.s.slot, blk, c.h) : nullptr;
        const uint32_t have = __ballot_sync(0xffffffffu, rec != nullptr);
        if (lane < kGroupRecs) sm.skip[st * kGroupRecs + lane] = rec == nullptr;
        __syncwarp();
        if (lane == 0) {
          if (have) mbar_arrive_expect_tx(&sm.raw_full[st], __popc(have) * rec_bytes(D));
          else mbar_arrive(&sm.raw_full[st]);
        }
        __syncwarp();
        // the lane of a page's first record in the group copies all of them
        if (rec && (lane == 0 || blk % a.v.blocks == 0)) {
          int n = min(kGroupRecs - lane, a.v.blocks - blk % a.v.blocks);
          n = min(n, __ffs(~(have >> lane)) - 1);
          bulk_g2s(sm.raw[st * kGroupRecs + lane], rec, n * rec_bytes(D), &sm.raw_full[st]);
        }
        __syncwarp();
      }
    }
    // the copies still in flight land before the block ends
    for (uint32_t k = groups > kGroups ? groups - kGroups : 0; k < groups; ++k)
      mbar_wait(&sm.raw_full[k % kGroups], (k / kGroups) & 1, abort, false);
  };

  auto dequant_role = [&]() {
    const int dw = warp - kDequantWarp, g = lane >> 2, cc = lane & 3;
    while (c.next(a, pre, lane)) {
      for (int i = 0; i < c.n; ++i, ++gi) {
        const int tok0 = (c.t0 + c.first + i) * kTileTok;
        bool skip[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t k = 2 * gi + u, st = k % kGroups;
          if (!mbar_wait(&sm.raw_full[st], (k / kGroups) & 1, abort)) return;
          skip[u] = sm.skip[st * kGroupRecs + dw];
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t q = 2 * gi + kv, slot = q % kSlots, use = q / kSlots;
          if (use > 0 && !mbar_wait(&sm.slot_empty[slot], (use - 1) & 1, abort)) return;
          uint8_t* out = sm.slot[slot];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int j = dw + 4 * u;
            const uint8_t* rec = sm.raw[(2 * gi + u) % kGroups * kGroupRecs + dw];
            if (kv == 0 && lane == 0) {
              const float2 sc = *reinterpret_cast<const float2*>(rec + 32 * D);
              sm.scale[gi & 1][j] = skip[u] ? make_float4(0.f, -INFINITY, 0.f, 0.f)
                                            : make_float4(sc.x, __log2f(sc.y),
                                                          __fdividef(1.f, sc.y), 0.f);
            }
            uint32_t vmask = 0xffffffffu;
            if (KIND == kE4m3 && kv == 1 && tok0 + kBlock * j + kBlock > c.s.len) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (tok0 + kBlock * j + 2 * cc + (e & 1) + 8 * (e >> 1) >= c.s.len)
                  vmask &= ~(0xffu << (8 * e));
            }
#pragma unroll
            for (int m = 0; m < D / 32; ++m) {
              const uint4 x =
                  *reinterpret_cast<const uint4*>(rec + kv * 16 * D + 512 * m + 16 * lane);
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t lo, hi;
                code_halves<KIND>(kv ? w[e] & vmask : w[e], lo, hi);
                if (skip[u]) lo = hi = 0;
                if (kv == 0) {
                  // token 8 (2 j + (e & 1)) + g, channels 32 m + 16 (e >> 1) + 4 cc ..
                  const int tg = 2 * j + (e & 1), cg = 4 * m + 2 * (e >> 1) + (cc >> 1);
                  *reinterpret_cast<uint2*>(out + (tg * (D / 8) + cg) * 128 + g * 16 +
                                            (cc & 1) * 8) = make_uint2(lo, hi);
                } else {
                  // channel 32 m + 8 e + g, tokens 16 j + 2 cc, + 1 and those + 8
                  const int cg = 4 * m + e;
                  *reinterpret_cast<uint32_t*>(out + (2 * j * (D / 8) + cg) * 128 + g * 16 +
                                               cc * 4) = lo;
                  *reinterpret_cast<uint32_t*>(out + ((2 * j + 1) * (D / 8) + cg) * 128 + g * 16 +
                                               cc * 4) = hi;
                }
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sm.slot_full[slot]);
            if (kv == 1) {
              mbar_arrive(&sm.raw_empty[2 * gi % kGroups]);
              mbar_arrive(&sm.raw_empty[(2 * gi + 1) % kGroups]);
            }
          }
        }
      }
    }
  };

  auto mma_role = [&]() {
    constexpr uint32_t id_s = idesc_f16_f32(kTileRows, kTileTok);
    constexpr uint32_t id_o = idesc_f16_f32(kTileRows, D);
    uint32_t n_q0 = 0, n_q1 = 0, n_p0 = 0, n_p1 = 0;
    // One elected lane issues; a product takes 64 cycles, and its issue has to stay
    // below that (71 measured; 83 with lane == 0 for elect_one, ~160 when the
    // descriptors of every (tile, slot) are unrolled as constants and spill).
    auto issue_scores = [&](int t, uint32_t slot) {
      if (elect_one()) {
        const uint64_t qd = smem_desc(smem_addr(sm.q[t]), kTileRows * 16, 128);
        const uint64_t kd = smem_desc(smem_addr(sm.slot[slot]), 128, D * 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_f16_ss(t * kTileTok, qd + k * (2 * kTileRows * 16 / 16), kd + k * (256 / 16), id_s,
                     k > 0);
        mma_commit(&sm.s_full[t]);
      }
      __syncwarp();
    };
    while (c.next(a, pre, lane)) {
      const int nt = c.tiles(a);
      for (int i = 0; i < c.n; ++i, ++gi) {
        const uint32_t ks = (2 * gi) % kSlots, ku = (2 * gi) / kSlots;
        const uint32_t vs = (2 * gi + 1) % kSlots, vu = (2 * gi + 1) / kSlots;
        const uint32_t ns = (2 * gi + 2) % kSlots, nu = (2 * gi + 2) / kSlots;
        if (i == 0) {
          if (!mbar_wait(&sm.slot_full[ks], ku & 1, abort)) return;
#pragma unroll 1
          for (int t = 0; t < nt; ++t) {
            const uint32_t done = t ? n_q1++ : n_q0++;
            if (!mbar_wait(&sm.q_full[t], done & 1, abort)) return;
            tc_fence_after();
            issue_scores(t, ks);
          }
          if (elect_one()) mma_commit(&sm.slot_empty[ks]);
          __syncwarp();
        }
        if (!mbar_wait(&sm.slot_full[vs], vu & 1, abort)) return;
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
          const uint32_t done = t ? n_p1++ : n_p0++;
          if (!mbar_wait(&sm.p_full[t], done & 1, abort)) return;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t vd = smem_desc(smem_addr(sm.slot[vs]), D * 16, 128);
#pragma unroll
            for (int k = 0; k < kTileTok / 16; ++k)
              mma_f16_ts(2 * kTileTok + t * D, t * kTileTok + 8 * k, vd + k * (2 * D * 16 / 16),
                         id_o, i > 0 || k > 0);
            if (t == nt - 1) mma_commit(&sm.slot_empty[vs]);
            if (i + 1 == c.n) mma_commit(&sm.o_full[t]);
          }
          __syncwarp();
          if (i + 1 < c.n) {
            if (t == 0 && !mbar_wait(&sm.slot_full[ns], nu & 1, abort)) return;
            issue_scores(t, ns);
            if (t == nt - 1 && elect_one()) mma_commit(&sm.slot_empty[ns]);
            __syncwarp();
          }
        }
      }
    }
  };

  auto softmax_role = [&]() {
    const int t = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane 32 (warp % 4)
    const uint32_t ts = t * kTileTok + lanes, to = 2 * kTileTok + t * D + lanes;
    uint32_t n_s = 0, n_o = 0;
    while (c.next(a, pre, lane)) {
      if (t >= c.tiles(a)) {
        gi += c.n;
        continue;
      }
      const Seq& s = c.s;
      const int r = c.row0 + kTileRows * t + row, rows = s.n * a.group;
      const bool valid = r < rows;
      const int tok = valid ? r / a.group : 0;
      const int head = c.h * a.group + r % a.group;
      const float qs = stage_q<D, T>(
          a, (const T*)a.q + (s.r0 + tok) * a.q_tok + (int64_t)head * a.q_head, valid, sm.q[t],
          row);
      fence_proxy_async_smem();
      mbar_arrive(&sm.q_full[t]);
      // a row sees the tokens lo .. lo + span; rows past the end mask nothing and are
      // not stored; a row before the first token sees none
      const int pos = s.len - s.n + tok;
      int lo = 0;
      uint32_t span = INT_MAX;
      if (valid) {
        lo = pos < 0 ? INT_MAX : first_seen(pos, a.window);
        span = pos < 0 ? 0 : pos - lo;
      }
      const bool idle = !__any_sync(0xffffffffu, valid);
      RowState st = {-INFINITY, -INFINITY, 0.f};
      for (int i = 0; i < c.n; ++i, ++gi) {
        if (!mbar_wait(&sm.s_full[t], n_s++ & 1, abort)) return;
        tc_fence_after();
        if (!idle) {
          const int first = (c.t0 + c.first + i) * kTileTok - lo;
          const bool masked = __any_sync(
              0xffffffffu, first < 0 || (uint32_t)(first + kTileTok - 1) > span);
          softmax_tile<D>(st, ts, to, i > 0, sm.scale[gi & 1], qs, masked, first, span);
        }
        tc_fence_before();
        mbar_arrive(&sm.p_full[t]);
      }
      if (!mbar_wait(&sm.o_full[t], n_o++ & 1, abort)) return;
      tc_fence_after();
      if (idle) continue;
      const float l = st.l;
      const bool whole = c.n == c.n_unit;
      const float inv = !whole ? 1.f : l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      const int64_t at = (s.r0 + tok) * ((int64_t)a.v.heads * a.group) + head;
      float* part = a.part + (2 * (int64_t)blockIdx.x + (c.first == 0)) * (kUnitRows * (D + 4));
      const int ur = kTileRows * t + row;
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        uint32_t x[32];
        tmem_ld32(to + 32 * q, x);
        tmem_wait_ld();
        if (valid && whole) {
          T* out = (T*)a.out + at * D + 32 * q;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float y[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) y[z] = l == 0.f ? 0.f : __uint_as_float(x[e + z]) * inv;
            store8<T>(out + e, y);
          }
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(part + ur * D + 32 * q + e) =
                make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        }
      }
      if (valid && whole) {
        if (a.ml) a.ml[at] = row_stats(st.m, st.ref - kTileLift, l);
      } else if (valid) {
        *reinterpret_cast<float4*>(part + kUnitRows * D + 4 * ur) = make_float4(st.ref, l, st.m, 0.f);
      }
    }
  };

  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == kLoadWarp) load_role();
    else if (warp == kMmaWarp) mma_role();
  } else if (warp >= kDequantWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsDequant));
    dequant_role();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    softmax_role();
  }

  __syncwarp();
  if (warp == kMmaWarp) {  // products still in flight (after an abort) end first
    if (elect_one()) mma_commit(&sm.drain);
    __syncwarp();
    mbar_wait(&sm.drain, 0, abort, false);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(sm.tmem, 512);
}

// Joins a unit that the shares' ends cut: the CTA column of the unit's first
// inner cut adds its pieces in order, 16 rows per CTA, two per warp.
constexpr int kTileJoinRows = 16, kTileJoinThreads = 256;

template <int D, typename T>
__global__ void __launch_bounds__(kTileJoinThreads) tile_join_kernel(AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  int32_t* pre = reinterpret_cast<int32_t*>(smem_raw);
  __shared__ int64_t sums[32];
  let_next_start();
  const int64_t total = tile_prefix<kTileJoinThreads>(a, pre, sums);
  // every CTA waits, or a later launch could pass the attention kernel
  wait_previous();
  const int64_t W = tile_workers(total), cut = blockIdx.x + 1;
  if (total == 0 || cut >= W) return;
  TileCursor c;
  c.x = total * cut / W;
  c.end = total;
  const int64_t x = c.x;
  c.next(a, pre, threadIdx.x & 31);
  const int64_t start = x - c.first, end = start + c.n_unit;
  if (c.first == 0 || total * (cut - 1) / W > start) return;
  int n = 1;  // pieces: of the worker before the cut, and on to the unit's end
  while (cut - 1 + n < W && total * (cut - 1 + n) / W < end) ++n;
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < kTileJoinRows; i += kTileJoinThreads / 32) {
    const int ur = blockIdx.y * kTileJoinRows + i, r = c.row0 + ur;
    if (r >= c.s.n * a.group) return;
    float m, ref, l, o[D / 32];
    join_row<D>(
        n, 0, 1, kUnitRows, ur,
        [&](int j) {
          return a.part + (2 * (cut - 1 + j) + (j == 0)) * (kUnitRows * (D + 4));
        },
        lane, o, m, ref, l);
    l = warp_sum(l);
    const int64_t at = (c.s.r0 + r / a.group) * ((int64_t)a.v.heads * a.group) +
                       c.h * a.group + r % a.group;
    store_row<D, T>(a, at, lane, o, m, ref - kTileLift, l);
  }
}

template <int D, int KIND, typename T>
static int launch_attend_tile(AttnArgs a, cudaStream_t st) {
  const int smem = (int)sizeof(TileSmem<D>);
  static_assert(sizeof(TileSmem<D>) <= 227 * 1024, "shared memory");
  static std::atomic<uint64_t> done{0};
  allow_smem(attend_tile_kernel<D, KIND, T>, smem, done);
  int rc = launch_next("paged_attention (tiles)", attend_tile_kernel<D, KIND, T>, dim3(kSms),
                       kTileThreads, smem, st, a);
  if (rc) return rc;
  const int64_t rows = (int64_t)a.max_new * a.group;
  const int unit_rows = rows < kUnitRows ? (int)rows : kUnitRows;
  return launch_next("paged_attention (tile join)", tile_join_kernel<D, T>,
                     dim3(kSms - 1, (unit_rows + kTileJoinRows - 1) / kTileJoinRows),
                     kTileJoinThreads,
                     (int)((a.v.B + 1) * sizeof(int32_t)), st, a);
}

}  // namespace paged
}  // namespace kvq
