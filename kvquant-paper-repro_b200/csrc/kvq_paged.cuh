// Paged 8-bit KV cache: the record format, append, read, and the page operations
// (fork, extend with copy-on-write, free, compact, copy). The attention that
// reads the cache is in kvq_paged_attn.cuh. Part of the kvq_lib.cu unity build.
//
// A block is 16 tokens of one KV head and is one record of 32 * D + 16 bytes:
//   key codes [D/32][t%8][(d/4)%4][(d/16)%2][t/8][d%4]
//   value codes [D/32][d%8][(t/2)%4][(d/16)%2][(d/8)%2][t/8][t%2]
//   key scale, value scale (fp32), 8 zero bytes
// The byte order is that of the A fragments of mma.m16n8k16: lane 4g + c of a
// warp reads its share of both operands as D/32 16-byte words at 16 * lane,
// coalesced and free of bank conflicts, and no code moves between lanes. A
// record is one contiguous copy, scales included; a page (its blocks of every
// head) is one contiguous copy too.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "kvq_common.cuh"
#include "kvq_sm100.cuh"

namespace kvq {
namespace paged {

constexpr int kBlock = 16;                    // tokens per record
constexpr float kScaleFloor = 0x1p-32f;       // least scale of a block
constexpr int kMaxSeqs = 4096;                // sequences (or slots) per call
enum Kind : int { kInt8 = 0, kE4m3 = 1 };
enum StatusBit : int { kNoPages = 1, kBadSlot = 2 };  // bits of the page operations' status

// Programmatic dependent launch: a kernel launched with that attribute may start
// while the one before it in the stream still runs, and sees its writes only after
// wait_previous(); let_next_start() allows the next such launch to begin.
__device__ __forceinline__ void wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__host__ __device__ constexpr int rec_bytes(int D) { return 32 * D + 16; }

// The cache as one call sees it: a layer's pool, the page table and the call's
// sequences (rows of the table, with their shares of the call's token rows).
struct View {
  uint8_t* pool;
  int64_t n_pages;
  int heads, dim, blocks;      // blocks per page
  const int32_t* table;        // [n_slots, n_cols]
  int64_t n_slots, n_cols;
  const int32_t* lengths;      // [n_slots]
  const int32_t* slots;        // [B] or null: sequence b is slot b
  const int32_t* indptr;       // [B + 1] or null: total / B rows each
  int64_t B, total;

  __host__ __device__ int64_t head_bytes() const { return (int64_t)blocks * rec_bytes(dim); }
  __host__ __device__ int64_t page_bytes() const { return heads * head_bytes(); }

  // Sequence b's slot (-1: out of range, flagged).
  __device__ int slot(int64_t b) const {
    const int s = slots ? slots[b] : (int)b;
    if (s < 0 || s >= n_slots) {
      atomicOr(&g_status, kStatusBadIndex);
      return -1;
    }
    return s;
  }
  // Tokens of a slot (0 and flagged when its row cannot hold them).
  __device__ int length(int s) const {
    const int n = lengths[s];
    if (n < 0 || n > n_cols * blocks * kBlock) {
      atomicOr(&g_status, kStatusBadIndex);
      return 0;
    }
    return n;
  }
  // Rows [r0, r1) of the call that belong to sequence b (none and flagged when out of range).
  __device__ void rows(int64_t b, int64_t& r0, int64_t& r1) const {
    if (!indptr) {
      const int64_t n = total / B;
      r0 = b * n;
      r1 = r0 + n;
      return;
    }
    r0 = indptr[b];
    r1 = indptr[b + 1];
    if (r0 < 0 || r1 < r0 || r1 > total) {
      atomicOr(&g_status, kStatusBadIndex);
      r0 = r1 = 0;
    }
  }
  // Record of block `blk` of slot s, head h (null and flagged without a page).
  __device__ uint8_t* record(int s, int blk, int h) const {
    const int page = table[(int64_t)s * n_cols + blk / blocks];
    if (page < 0 || page >= n_pages) {
      atomicOr(&g_status, kStatusBadIndex);
      return nullptr;
    }
    return pool + page * page_bytes() + h * head_bytes() +
           (int64_t)(blk % blocks) * rec_bytes(dim);
  }
};

// Items of a call over the 16-token blocks that its rows touch: sequence b gets
// the items [indptr[b] / 16 + 2 b, indptr[b + 1] / 16 + 2 (b + 1)). m rows touch
// at most (m + 14) / 16 + 1 blocks wherever they start, which is never more than
// that range holds, so no prefix sum over the sequences is needed: an item finds
// its sequence by a search whose steps probe 32 places at once.
inline int64_t block_items(const View& v) {
  return v.indptr ? v.total / kBlock + 2 * v.B : v.B * (v.total / v.B / kBlock + 2);
}
__device__ __forceinline__ void find_item(const View& v, int64_t item, int lane, int64_t& b,
                                          int64_t& local) {
  if (!v.indptr) {
    const int64_t per = v.total / v.B / kBlock + 2;
    b = item / per;
    local = item % per;
    return;
  }
  int64_t lo = 0, hi = v.B;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t i = lo + (lane + 1) * step;
    const bool below = i < hi && v.indptr[i] / kBlock + 2 * i <= item;
    lo += step * __popc(__ballot_sync(0xffffffffu, below));
    hi = min(hi, lo + step);
  }
  b = lo;
  local = item - (v.indptr[lo] / kBlock + 2 * lo);
}

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t w);
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t from_float2(float a, float b);
template <>
__device__ __forceinline__ uint32_t from_float2<__half>(float a, float b) {
  return half2_bits(a, b);
}
template <>
__device__ __forceinline__ uint32_t from_float2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int KIND>
struct Code;
template <>
struct Code<kInt8> {
  static constexpr float kMax = 127.f;
  static constexpr uint32_t kZero = 0x80808080u;  // four codes of 0
  // Four codes from values already divided by the scale; NaN gives 0.
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
    auto q = [](float x) { return (uint32_t)(max(-127, min(127, __float2int_rn(x))) + 128); };
    return prmt(prmt(q(a), q(b), 0x0040), prmt(q(c), q(d), 0x0040), 0x5410);
  }
  // The same for values that are known to be finite and at most 127.4: adding
  // 1.5 * 2^23 + 128 rounds to nearest even and leaves the code in the low byte.
  static __device__ __forceinline__ uint32_t pack_fine(float a, float b, float c, float d) {
    auto q = [](float x) { return __float_as_uint(__fadd_rn(x, 12582912.f + 128.f)); };
    return prmt(prmt(q(a), q(b), 0x0040), prmt(q(c), q(d), 0x0040), 0x5410);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (float)(int)((w >> (8 * e)) & 0xffu) - 128.f;
  }
};
template <>
struct Code<kE4m3> {
  static constexpr float kMax = 448.f;
  static constexpr uint32_t kZero = 0u;
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
    auto two = [](float x, float y) {
      x = x == x ? x : 0.f;
      y = y == y ? y : 0.f;
      uint16_t r;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
      return (uint32_t)r;
    };
    return two(a, b) | (two(c, d) << 16);
  }
  // The same without the care for NaN.
  static __device__ __forceinline__ uint32_t pack_fine(float a, float b, float c, float d) {
    uint16_t l, h;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(l) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(d), "f"(c));
    return (uint32_t)l | ((uint32_t)h << 16);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      uint32_t h;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (8 * e))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x[e] = f.x;
      x[e + 1] = f.y;
    }
  }
};

// Bits of the 16-bit infinity; a magnitude's bits order like the magnitude, NaN last.
template <typename T>
__device__ constexpr uint32_t inf_bits() {
  return std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // NaN and the infinities do not set a scale
}

// Which channels and tokens a lane handles when rows of tokens are turned into a
// record or back, and where its words lie. Both maps read and write token rows
// in 16-byte words (8 channels).
//   keys: word `w` (channels 8x + 4w ..) of token t; the lane bits are chosen so
//   that the 32 words of one access fall into 32 banks.
//   values: the four tokens of one code word, 8 channels e.
struct KeyMap {
  int jj, xh, g01, r, swap;
  __device__ explicit KeyMap(int lane)
      : jj(lane & 1), xh((lane >> 1) & 1), g01(((lane >> 2) & 1) | ((lane >> 4) & 1) << 1),
        r((lane >> 3) & 1), swap((lane >> 4) & 1) {}
  // step: i * 2 + (g >> 2)
  __device__ int token(int step) const { return g01 + 4 * (step & 1) + 8 * r; }
  __device__ int channel(int step) const { return 32 * (step >> 1) + 16 * jj + 8 * xh; }
  __device__ int offset(int step, int w) const {
    return 512 * (step >> 1) + 64 * (g01 + 4 * (step & 1)) + 16 * (2 * xh + w) + 8 * jj + 4 * r;
  }
};
struct ValueMap {
  int c, y0;
  __device__ explicit ValueMap(int lane) : c(lane & 3), y0(lane >> 2) {}
  __device__ int token(int e) const { return 2 * c + (e & 1) + 8 * (e >> 1); }
  __device__ int channel(int step) const { return 8 * (y0 + 8 * step); }
  __device__ int offset(int step, int e) const {
    const int y = y0 + 8 * step;
    return 512 * (y >> 2) + 64 * e + 16 * c + 8 * ((y >> 1) & 1) + 4 * (y & 1);
  }
};

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// One warp per (touched block, head). A block started by the call gets
//   s = max(max|x| / Qmax, 2^-32), code = round(x / s) (as x times 1 / s),
// an open block keeps the larger of its scale and that, and its older codes are
// restated as round(code * s_old / s) when it grew: at most half a step of the
// new scale of error each time. Places past the last token hold the code 0.
// granted: the first token of each slot that its last extend granted (null: not kept);
// tokens before it are stored already, perhaps for several slots, and are not written over.
// Bound by HBM: 4 D bytes in and 2 D + 1 bytes out per token and head. 17 prompts, 8
// heads, D = 128, bf16 to e4m3: 41 us for 0.21 GB = 5.1 TB/s (128 registers, 16 warps an
// SM); one token of 64 sequences: 5 us, five dependent look-ups.
constexpr int kAppendWarps = 4;

// Largest finite magnitude of a lane's 16-byte words, over the warp; `fine`: all of
// them are finite (else the slow way leaves the others out).
template <int NC, typename T>
__device__ __forceinline__ float warp_amax(const uint4 (&x)[NC], bool& fine) {
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) mx = __vmaxu2(mx, w[e] & 0x7fff7fffu);
  }
  mx = __reduce_max_sync(0xffffffffu, max(lo16(mx), hi16(mx)));
  fine = mx < inf_bits<T>();
  if (fine) return to_float2<T>(mx).x;
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = to_float2<T>(w[e]);
      m = fmaxf(m, fmaxf(finite_abs(a.x), finite_abs(a.y)));
    }
  }
  return warp_max(m);
}

// A lane's words of the new tokens as codes into the record. FINE: all finite.
template <int D, int KIND, typename T, bool FINE>
__device__ __forceinline__ void put_keys(const uint4 (&x)[D / 16], float inv, const KeyMap& km,
                                         uint8_t* sm, int first, int last) {
  using C = Code<KIND>;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int t = km.token(i);
    const uint32_t xw[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int ww = w ^ km.swap;
      const float2 a = to_float2<T>(ww ? xw[2] : xw[0]), c = to_float2<T>(ww ? xw[3] : xw[1]);
      const float y[4] = {__fmul_rn(a.x, inv), __fmul_rn(a.y, inv), __fmul_rn(c.x, inv),
                          __fmul_rn(c.y, inv)};
      const uint32_t code = FINE ? C::pack_fine(y[0], y[1], y[2], y[3])
                                 : C::pack(y[0], y[1], y[2], y[3]);
      if (first == 0 || (t >= first && t < last))
        *reinterpret_cast<uint32_t*>(sm + km.offset(i, ww)) = code;
    }
  }
}
template <int D, int KIND, typename T, bool FINE>
__device__ __forceinline__ void put_values(const uint4 (&x)[D / 16], float inv,
                                           const ValueMap& vm, uint8_t* sm, int first, int last) {
  using C = Code<KIND>;
  uint32_t fresh = 0;  // bytes of a value word that are new tokens
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (vm.token(e) >= first && vm.token(e) < last) fresh |= 0xffu << (8 * e);
#pragma unroll
  for (int i = 0; i < D / 16; i += 4) {
    const uint32_t* xw[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) xw[z] = reinterpret_cast<const uint32_t*>(&x[i + z]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float2 a = to_float2<T>(xw[z][e >> 1]);
        y[z] = __fmul_rn((e & 1) ? a.y : a.x, inv);
      }
      const uint32_t code = FINE ? C::pack_fine(y[0], y[1], y[2], y[3])
                                 : C::pack(y[0], y[1], y[2], y[3]);
      uint32_t* at = reinterpret_cast<uint32_t*>(sm + 16 * D + vm.offset(i >> 2, e));
      *at = first == 0 ? code : (*at & ~fresh) | (code & fresh);
    }
  }
}

template <int D, int KIND, typename T>
__global__ void __launch_bounds__(32 * kAppendWarps, 4) append_kernel(
    View v, const T* __restrict__ k, int64_t k_tok, int64_t k_head, const T* __restrict__ val,
    int64_t v_tok, int64_t v_head, const int32_t* granted, int64_t n_warps) {
  constexpr int R = rec_bytes(D), NC = D / 16;  // NC: 16-byte words of a lane, K or V
  using C = Code<KIND>;
  __shared__ __align__(128) uint8_t smem[kAppendWarps][(R + 127) / 128 * 128];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t warp = (int64_t)blockIdx.x * kAppendWarps + wid;
  wait_previous();
  let_next_start();
  if (warp >= n_warps) return;
  const int h = (int)(warp % v.heads);
  int64_t b, local;
  find_item(v, warp / v.heads, lane, b, local);
  const int s = v.slot(b);
  if (s < 0) return;
  int64_t r0, r1;
  v.rows(b, r0, r1);
  const int len = v.length(s);
  const int start = len - (int)(r1 - r0);
  if (r1 == r0) return;
  // more new tokens than the slot holds, or than it was granted
  if (start < 0 || (granted && start < granted[s])) {
    atomicOr(&g_status, kStatusBadIndex);
    return;
  }
  const int64_t blk64 = start / kBlock + local;
  if (local < 0 || blk64 * kBlock >= len) return;
  const int t0 = (int)blk64 * kBlock;
  const int page = v.table[(int64_t)s * v.n_cols + blk64 / v.blocks];
  uint8_t* sm = smem[wid];

  // token t of the block is new when first <= t < last
  const int first = max(0, start - t0), last = min(kBlock, len - t0);
  const T* kp = k + (r0 + t0 - start) * k_tok + h * k_head;
  const T* vp = val + (r0 + t0 - start) * v_tok + h * v_head;
  const KeyMap km(lane);
  const ValueMap vm(lane);
  uint4 kx[NC], vx[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int t = km.token(i);
    kx[i] = make_uint4(0, 0, 0, 0);
    if (t >= first && t < last)
      kx[i] = *reinterpret_cast<const uint4*>(kp + t * k_tok + km.channel(i));
    const int tv = vm.token(i & 3);
    vx[i] = make_uint4(0, 0, 0, 0);
    if (tv >= first && tv < last)
      vx[i] = *reinterpret_cast<const uint4*>(vp + tv * v_tok + vm.channel(i >> 2));
  }
  if (page < 0 || page >= v.n_pages) {
    atomicOr(&g_status, kStatusBadIndex);
    return;
  }
  uint8_t* rec =
      v.pool + page * v.page_bytes() + h * v.head_bytes() + (blk64 % v.blocks) * (int64_t)R;
  bool k_fine, v_fine;
  float ks, vs, ki, vi;
  if (first == 0) {
    ks = fmaxf(__fmul_rn(warp_amax<NC, T>(kx, k_fine), 1.f / C::kMax), kScaleFloor);
    vs = fmaxf(__fmul_rn(warp_amax<NC, T>(vx, v_fine), 1.f / C::kMax), kScaleFloor);
    ki = __fdiv_rn(1.f, ks);
    vi = __fdiv_rn(1.f, vs);
  } else {
    // An open block: a lane's 16-byte words of the record hold, for keys, tokens
    // g and g + 8 in turn and, for values, the same four tokens in every word.
    uint4 old[2 * (D / 32)];
#pragma unroll
    for (int i = 0; i < 2 * (D / 32); ++i)
      old[i] = *reinterpret_cast<const uint4*>(rec + 512 * i + 16 * lane);
    const float2 sc = *reinterpret_cast<const float2*>(rec + 32 * D);
    ks = fmaxf(sc.x, fmaxf(__fmul_rn(warp_amax<NC, T>(kx, k_fine), 1.f / C::kMax), kScaleFloor));
    vs = fmaxf(sc.y, fmaxf(__fmul_rn(warp_amax<NC, T>(vx, v_fine), 1.f / C::kMax), kScaleFloor));
    ki = __fdiv_rn(1.f, ks);
    vi = __fdiv_rn(1.f, vs);
    const uint32_t keep_k[2] = {(lane >> 2) < first ? ~0u : 0u, (lane >> 2) + 8 < first ? ~0u : 0u};
    uint32_t keep_v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (2 * (lane & 3) + (e & 1) + 8 * (e >> 1) < first) keep_v |= 0xffu << (8 * e);
#pragma unroll
    for (int i = 0; i < 2 * (D / 32); ++i) {
      const bool key = i < D / 32;
      uint32_t w[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
      if (key ? ks > sc.x : vs > sc.y) {  // the scale grew: older codes anew
        const float f = key ? __fmul_rn(sc.x, ki) : __fmul_rn(sc.y, vi);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x[4];
          C::unpack(w[e], x);
          w[e] = C::pack(__fmul_rn(x[0], f), __fmul_rn(x[1], f), __fmul_rn(x[2], f),
                         __fmul_rn(x[3], f));
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // places after the older tokens: 0
        const uint32_t keep = key ? keep_k[e & 1] : keep_v;
        w[e] = (w[e] & keep) | (C::kZero & ~keep);
      }
      *reinterpret_cast<uint4*>(sm + 512 * i + 16 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
  }
  if (k_fine) put_keys<D, KIND, T, true>(kx, ki, km, sm, first, last);
  else put_keys<D, KIND, T, false>(kx, ki, km, sm, first, last);
  if (v_fine) put_values<D, KIND, T, true>(vx, vi, vm, sm, first, last);
  else put_values<D, KIND, T, false>(vx, vi, vm, sm, first, last);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2 * (D / 32); ++i)
    *reinterpret_cast<uint4*>(rec + 512 * i + 16 * lane) =
        *reinterpret_cast<const uint4*>(sm + 512 * i + 16 * lane);
  if (lane < 4) *reinterpret_cast<float*>(rec + 32 * D + 4 * lane) = lane == 0 ? ks : lane == 1 ? vs : 0.f;
}

// ---------------------------------------------------------------------------
// Read: the tokens [starts[b], starts[b] + rows of b) of each sequence as 16-bit
// or 32-bit values code * scale. One warp per touched block and `per_warp` heads:
// four in large calls, which then hide the look-ups (indptr, length, table) behind
// the records of the heads before.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(from_float2<__half>(x[0], x[1]), from_float2<__half>(x[2], x[3]),
                 from_float2<__half>(x[4], x[5]), from_float2<__half>(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
  using B = __nv_bfloat16;
  *reinterpret_cast<uint4*>(p) = make_uint4(from_float2<B>(x[0], x[1]), from_float2<B>(x[2], x[3]),
                                            from_float2<B>(x[4], x[5]), from_float2<B>(x[6], x[7]));
}

template <int D, int KIND, typename T>
__global__ void __launch_bounds__(32 * kAppendWarps) read_kernel(View v, const int32_t* starts,
                                                                 T* __restrict__ k,
                                                                 T* __restrict__ val,
                                                                 int64_t n_warps, int per_warp) {
  constexpr int R = rec_bytes(D), NC = D / 16;
  using C = Code<KIND>;
  __shared__ __align__(128) uint8_t smem[kAppendWarps][(R + 127) / 128 * 128];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t warp = (int64_t)blockIdx.x * kAppendWarps + wid;
  wait_previous();
  let_next_start();
  if (warp >= n_warps) return;
  const int splits = (v.heads + per_warp - 1) / per_warp;
  const int h0 = (int)(warp % splits) * per_warp, h1 = min(v.heads, h0 + per_warp);
  int64_t b, local;
  find_item(v, warp / splits, lane, b, local);
  const int s = v.slot(b);
  if (s < 0) return;
  int64_t r0, r1;
  v.rows(b, r0, r1);
  if (r1 == r0) return;
  const int start = starts ? starts[b] : 0;
  const int64_t end = start + (r1 - r0);
  if (start < 0 || end > v.length(s)) {
    atomicOr(&g_status, kStatusBadIndex);
    return;
  }
  const int64_t blk = start / kBlock + local;
  if (local < 0 || blk * kBlock >= end) return;
  const uint8_t* rec = v.record(s, (int)blk, h0);
  if (!rec) return;
  uint8_t* sm = smem[wid];
  uint4 next[2 * (D / 32)];
  float2 next_sc;
  auto fetch = [&](int h) {
    const uint8_t* p = rec + (h - h0) * v.head_bytes();
#pragma unroll
    for (int i = 0; i < 2 * (D / 32); ++i)
      next[i] = *reinterpret_cast<const uint4*>(p + 512 * i + 16 * lane);
    next_sc = *reinterpret_cast<const float2*>(p + 32 * D);
  };
  fetch(h0);
  const int64_t row0 = r0 + blk * kBlock - start;  // output row of the block's token 0
  const KeyMap km(lane);
  const ValueMap vm(lane);
  for (int h = h0; h < h1; ++h) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2 * (D / 32); ++i)
      *reinterpret_cast<uint4*>(sm + 512 * i + 16 * lane) = next[i];
    const float ks = next_sc.x, vs = next_sc.y;
    if (h + 1 < h1) fetch(h + 1);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t row = row0 + km.token(i);
      float x[8];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float y[4];
        C::unpack(*reinterpret_cast<const uint32_t*>(sm + km.offset(i, w)), y);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * w + e] = __fmul_rn(y[e], ks);
      }
      if (row >= r0 && row < r1) store8<T>(k + (row * v.heads + h) * D + km.channel(i), x);
    }
#pragma unroll
    for (int i = 0; i < NC / 4; ++i) {
      float x[4][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float y[4];
        C::unpack(*reinterpret_cast<const uint32_t*>(sm + 16 * D + vm.offset(i, e)), y);
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t][e] = __fmul_rn(y[t], vs);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t row = row0 + vm.token(t);
        if (row >= r0 && row < r1) store8<T>(val + (row * v.heads + h) * D + vm.channel(i), x[t]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Page operations. table [n_slots, n_cols] (-1: no page), lengths [n_slots],
// refs [n_pages] live on the device and only kernels change them, so a decode
// loop needs no host copy of them and no synchronisation.
// ---------------------------------------------------------------------------
struct Meta {
  int32_t* table;
  int64_t n_slots, n_cols;
  int32_t* lengths;
  int32_t* refs;
  int64_t n_pages, page_tokens;
};

constexpr int kPageThreads = 256;

// Whether list[i] is a slot that no earlier place of the list names (block-wide).
__device__ __forceinline__ bool own_slot(const int32_t* list, int64_t i, int64_t n_slots) {
  const int s = list[i];
  bool again = s < 0 || s >= n_slots;
  for (int64_t j = threadIdx.x; j < i; j += blockDim.x) again |= list[j] == s;
  return !__syncthreads_or(again);
}

// One CTA per slot: gives its pages up.
__global__ void __launch_bounds__(kPageThreads) free_kernel(Meta m, const int32_t* slots,
                                                            int32_t* status) {
  wait_previous();
  let_next_start();
  if (!own_slot(slots, blockIdx.x, m.n_slots)) {
    if (threadIdx.x == 0) atomicOr(status, kBadSlot);
    return;
  }
  int32_t* row = m.table + slots[blockIdx.x] * m.n_cols;
  for (int64_t c = threadIdx.x; c < m.n_cols; c += kPageThreads) {
    const int p = row[c];
    if (p >= 0 && p < m.n_pages) atomicSub(&m.refs[p], 1);
    row[c] = -1;
  }
  if (threadIdx.x == 0) m.lengths[slots[blockIdx.x]] = 0;
}

// One CTA per (src, dst): dst, which has to be empty, shares src's pages.
__global__ void __launch_bounds__(kPageThreads) fork_kernel(Meta m, const int32_t* src,
                                                            const int32_t* dst, int64_t n,
                                                            int32_t* status) {
  wait_previous();
  let_next_start();
  const int from = src[blockIdx.x], to = dst[blockIdx.x];
  bool bad = !own_slot(dst, blockIdx.x, m.n_slots);
  bool is_src = from < 0 || from >= m.n_slots;
  for (int64_t j = threadIdx.x; j < n; j += kPageThreads) is_src |= src[j] == to;
  bad |= __syncthreads_or(is_src);
  if (!bad) bad = m.lengths[to] != 0;
  __syncthreads();  // every thread has read the length before it is written
  if (bad) {
    if (threadIdx.x == 0) atomicOr(status, kBadSlot);
    return;
  }
  const int32_t* in = m.table + from * m.n_cols;
  int32_t* out = m.table + to * m.n_cols;
  for (int64_t c = threadIdx.x; c < m.n_cols; c += kPageThreads) {
    const int p = in[c];
    out[c] = p;
    if (p >= 0 && p < m.n_pages) atomicAdd(&m.refs[p], 1);
  }
  if (threadIdx.x == 0) m.lengths[to] = m.lengths[from];
}

// Block-wide exclusive scan of one int per thread (1024 threads); total to all.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) warp_sums[wid] = incl;
  __syncthreads();
  int before = 0, all = 0;
  {
    const int y = lane < nw ? warp_sums[lane] : 0;
    int z = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += u;
    }
    all = __shfl_sync(0xffffffffu, z, 31);
    before = __shfl_sync(0xffffffffu, z - y, wid);
  }
  __syncthreads();
  total = all;
  return before + incl - x;
}

constexpr int kPlanThreads = 1024, kPer = 4;  // pages per thread and scan

// Workspace of extend and compact: the number of page moves, then the moves.
struct Moves {
  int32_t count, pad[3];
};

// One CTA: pages for the new tokens of every slot, taken from the free ones in
// ascending order, slot after slot in the list's order. A slot whose last page
// is open and shared gets a page of its own for it (to be copied by
// move_kernel) unless every other holder stands before it in the list. When the
// call is refused nothing changes but `granted`: no token of its slots is.
__global__ void __launch_bounds__(kPlanThreads) extend_kernel(Meta m, const int32_t* slots,
                                                              int64_t n, const int32_t* n_new,
                                                              int n_new_all, int32_t* status,
                                                              Moves* moves, int2* list,
                                                              int32_t* pages, int32_t* granted) {
  static_assert(kPlanThreads == 32 * 32, "a warp holds one sum of every warp");
  wait_previous();
  let_next_start();
  __shared__ int warp_sums[32];
  __shared__ int last_page[kMaxSeqs];  // shared open page of slot i, or -1 - i
  __shared__ int need[kMaxSeqs];       // pages, then its offset; copy flag in `copies`
  __shared__ uint8_t copies[kMaxSeqs];
  __shared__ int64_t warp_asked[32];
  const int tid = threadIdx.x;
  auto refuse = [&](int why) {
    for (int64_t i = tid; granted && i < n; i += kPlanThreads)
      if (slots[i] >= 0 && slots[i] < m.n_slots) granted[slots[i]] = INT32_MAX;
    if (tid == 0) {
      atomicOr(status, why);
      moves->count = 0;
    }
  };
  int bad = 0;
  for (int i = tid; i < n; i += kPlanThreads) {
    const int s = slots[i], add = n_new ? n_new[i] : n_new_all;
    last_page[i] = -1 - i;
    need[i] = 0;
    if (s < 0 || s >= m.n_slots || add < 0) {
      bad |= kBadSlot;
      continue;
    }
    const int64_t len = m.lengths[s], P = m.page_tokens;
    if (len < 0 || (len + add + P - 1) / P > m.n_cols) {
      bad |= kBadSlot;
      continue;
    }
    need[i] = (int)((len + add + P - 1) / P - (len + P - 1) / P);
    if (add > 0 && len % P) {
      const int p = m.table[s * m.n_cols + len / P];
      if (p < 0 || p >= m.n_pages) bad |= kBadSlot;
      else if (m.refs[p] > 1) last_page[i] = p;
    }
  }
  bad = __syncthreads_or(bad);
  int64_t asked = 0;  // pages of all slots; the 32-bit sums below hold up to n_pages
  for (int i = tid; i < n; i += kPlanThreads) {
    const int s = slots[i], p = last_page[i];
    int before = 0;
    for (int j = 0; j < i; ++j) {
      bad |= slots[j] == s ? kBadSlot : 0;
      before += last_page[j] == p;
    }
    const bool copy = p >= 0 && m.refs[p] - before > 1;
    copies[i] = copy;
    need[i] += copy;
    asked += need[i];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) asked += __shfl_xor_sync(0xffffffffu, asked, o);
  warp_asked[tid >> 5] = asked;
  bad = __syncthreads_or(bad);
  asked = warp_asked[tid & 31];
#pragma unroll
  for (int o = 16; o; o >>= 1) asked += __shfl_xor_sync(0xffffffffu, asked, o);
  if (bad || asked > m.n_pages) {
    refuse(bad ? kBadSlot : kNoPages);
    return;
  }
  int total = 0;
  for (int64_t i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int64_t i = i0 + tid;
    int sum;
    const int at = block_scan(i < n ? need[i] : 0, warp_sums, sum);
    if (i < n) need[i] = total + at;
    total += sum;
  }
  // the `total` lowest free pages
  int found = 0;
  for (int64_t p0 = 0; p0 < m.n_pages && found < total; p0 += kPlanThreads * kPer) {
    const int64_t p = p0 + tid * kPer;
    int free = 0;  // bit j: page p + j is free
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (p + j < m.n_pages && m.refs[p + j] == 0) free |= 1 << j;
    int sum, at = found + block_scan(__popc(free), warp_sums, sum);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if ((free >> j & 1) && at < total) pages[at++] = (int)(p + j);
    found += sum;
  }
  if (found < total) {
    refuse(kNoPages);
    return;
  }
  __syncthreads();
  int n_copies = 0;
  for (int64_t i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int64_t i = i0 + tid;
    const bool copy = i < n && copies[i];
    int sum;
    const int at = n_copies + block_scan(copy, warp_sums, sum);
    if (copy) list[at] = make_int2(last_page[i], pages[need[i]]);
    n_copies += sum;
  }
  if (tid == 0) moves->count = n_copies;
  const int lane = tid & 31;
  for (int64_t i = tid >> 5; i < n; i += kPlanThreads / 32) {
    const int s = slots[i], add = n_new ? n_new[i] : n_new_all;
    const int64_t len = m.lengths[s], P = m.page_tokens;
    const int64_t col = copies[i] ? len / P : (len + P - 1) / P, end = (len + add + P - 1) / P;
    for (int64_t c = col + lane; c < end; c += 32) {
      const int p = pages[need[i] + (c - col)];
      m.table[s * m.n_cols + c] = p;
      m.refs[p] = 1;
    }
    __syncwarp();
    if (lane == 0) {
      if (copies[i]) atomicSub(&m.refs[last_page[i]], 1);
      m.lengths[s] = (int)(len + add);
      if (granted) granted[s] = (int)len;
    }
  }
}

// One CTA: the live pages at or past the number of live pages, in ascending
// order, move into the free ones below it.
__global__ void __launch_bounds__(kPlanThreads) compact_kernel(const int32_t* refs,
                                                               int64_t n_pages, Moves* moves,
                                                               int2* list, int32_t* new_id,
                                                               int32_t* n_live) {
  wait_previous();
  let_next_start();
  __shared__ int warp_sums[32];
  int mine = 0;
  for (int64_t p = threadIdx.x; p < n_pages; p += kPlanThreads) mine += refs[p] > 0;
  int live;
  block_scan(mine, warp_sums, live);
  int holes = 0, movers = 0;
  for (int64_t p0 = 0; p0 < n_pages; p0 += kPlanThreads * kPer) {
    const int64_t p = p0 + threadIdx.x * kPer;
    int hole = 0, mover = 0;  // bit j: of page p + j
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool is_live = p + j < n_pages && refs[p + j] > 0;
      if (p + j < live && !is_live) hole |= 1 << j;
      if (p + j >= live && is_live) mover |= 1 << j;
    }
    // both counts in one scan: at most 4096 of each
    int sums, at = block_scan(__popc(hole) | __popc(mover) << 16, warp_sums, sums);
    int at_hole = holes + (at & 0xffff), at_mover = movers + (at >> 16);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (hole >> j & 1) list[at_hole++].y = (int)(p + j);
      if (mover >> j & 1) list[at_mover++].x = (int)(p + j);
    }
    holes += sums & 0xffff;
    movers += sums >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) new_id[list[i].x] = list[i].y;
  if (threadIdx.x == 0) {
    moves->count = movers;
    *n_live = live;
  }
}

// What a compaction changes beside the pages: table entries and counts.
struct Renumber {
  int32_t* table;  // null: nothing
  int64_t n;
  int32_t* refs;
  int64_t n_pages;
  const int32_t *new_id, *n_live;
};

// Copies pages src -> dst of every layer as the list says, in equal pieces of up to
// 16 KB per CTA, and renumbers. Bound by HBM. (Pieces of 16 KB and a rest of 0.5 KB:
// 103 us for 983 pages of 2 x 131 KB; 32 KB pieces, eight words a thread: 114.)
__global__ void __launch_bounds__(kPageThreads) move_kernel(const uint8_t* __restrict__ src,
                                                            uint8_t* __restrict__ dst,
                                                            int64_t src_layer, int64_t dst_layer,
                                                            int64_t page_bytes, int n_layers,
                                                            const Moves* moves, const int2* list,
                                                            Renumber rn) {
  constexpr int kDeep = 4;
  constexpr int64_t kStep = kPageThreads * 16;
  wait_previous();
  let_next_start();
  const int count = moves->count;
  const int64_t chunks = (page_bytes + kStep * kDeep - 1) / (kStep * kDeep);
  const int64_t chunk_bytes = (page_bytes / 16 + chunks - 1) / chunks * 16;
  const int64_t items = (int64_t)count * n_layers * chunks;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t chunk = it % chunks, pair = it / chunks;
    const int2 mv = list[pair / n_layers];
    const int64_t layer = pair % n_layers;
    const uint8_t* from = src + layer * src_layer + mv.x * page_bytes;
    uint8_t* to = dst + layer * dst_layer + mv.y * page_bytes;
    const int64_t end = min(page_bytes, (chunk + 1) * chunk_bytes);
    const int64_t o = chunk * chunk_bytes + threadIdx.x * 16;
    uint4 x[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (o + i * kStep < end) x[i] = *reinterpret_cast<const uint4*>(from + o + i * kStep);
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (o + i * kStep < end) *reinterpret_cast<uint4*>(to + o + i * kStep) = x[i];
  }
  if (!rn.table) return;
  const int live = *rn.n_live;
  const int64_t stride = (int64_t)gridDim.x * kPageThreads;
  const int64_t i0 = (int64_t)blockIdx.x * kPageThreads + threadIdx.x;
  for (int64_t i = i0; i < rn.n; i += stride) {
    const int p = rn.table[i];
    if (p >= live && p < rn.n_pages) rn.table[i] = rn.new_id[p];
  }
  for (int64_t i = i0; i < count; i += stride) {
    rn.refs[list[i].y] = rn.refs[list[i].x];
    rn.refs[list[i].x] = 0;
  }
}

// The move list of a plain copy, with its pairs checked.
__global__ void __launch_bounds__(kPageThreads) pairs_kernel(const int32_t* src, int64_t n_src,
                                                             const int32_t* dst, int64_t n_dst,
                                                             int64_t n, Moves* moves, int2* list) {
  wait_previous();
  let_next_start();
  __shared__ int warp_sums[32];
  int kept = 0;  // the same in every thread
  for (int64_t i0 = 0; i0 < n; i0 += kPageThreads) {
    const int64_t i = i0 + threadIdx.x;
    bool ok = i < n;
    int a = 0, c = 0;
    if (ok) {
      a = src[i];
      c = dst[i];
      ok = a >= 0 && a < n_src && c >= 0 && c < n_dst;
      if (!ok) atomicOr(&g_status, kStatusBadIndex);
    }
    int sum;
    const int at = block_scan(ok, warp_sums, sum);
    if (ok) list[kept + at] = make_int2(a, c);
    kept += sum;
  }
  if (threadIdx.x == 0) moves->count = kept;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <typename... Params, typename... Args>
static int launch_next(const char* what, void (*kernel)(Params...), dim3 grid, int threads,
                       int smem, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch(what);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int check_view(const char* what, const View& v, int kind, int64_t page_tokens) {
  if (v.dim != 64 && v.dim != 128) {
    set_error("%s: head_dim must be 64 or 128 (got %d)", what, v.dim);
    return KVQ_ERR_UNSUPPORTED;
  }
  if (kind != kInt8 && kind != kE4m3) {
    set_error("%s: kind must be 0 (int8) or 1 (e4m3), got %d", what, kind);
    return KVQ_ERR_UNSUPPORTED;
  }
  if (page_tokens < kBlock || page_tokens > 1024 || page_tokens % kBlock) {
    set_error("%s: page_tokens must be a multiple of 16 in 16..1024 (got %lld)", what,
              (long long)page_tokens);
    return KVQ_ERR_INVALID;
  }
  if (v.n_pages < 1 || v.n_pages > INT32_MAX || v.heads < 1 || v.heads > 1024 || v.n_slots < 1 ||
      v.n_slots > INT32_MAX || v.n_cols < 1 || v.n_cols > INT32_MAX / page_tokens) {
    set_error("%s: pool or table of an impossible size (pages %lld, heads %d, table %lld x %lld)",
              what, (long long)v.n_pages, v.heads, (long long)v.n_slots, (long long)v.n_cols);
    return KVQ_ERR_INVALID;
  }
  if (v.B < 1 || v.B > kMaxSeqs || (!v.slots && v.B > v.n_slots)) {
    set_error("%s: %lld sequences (1..%d, and no more than the table's rows without slots)", what,
              (long long)v.B, kMaxSeqs);
    return KVQ_ERR_INVALID;
  }
  if (v.total < 0 || v.total > INT32_MAX || (!v.indptr && v.total % v.B)) {
    set_error("%s: %lld rows do not divide among %lld sequences", what, (long long)v.total,
              (long long)v.B);
    return KVQ_ERR_INVALID;
  }
  if (!v.pool || !aligned16(v.pool) || !v.table || !v.lengths) {
    set_error("%s: the pool must be 16-byte aligned and the table and lengths given", what);
    return KVQ_ERR_INVALID;
  }
  return KVQ_OK;
}

inline int check_meta(const char* what, const Meta& m) {
  if (!m.table || !m.refs || m.n_slots < 1 || m.n_slots > INT32_MAX || m.n_cols < 1 ||
      m.n_pages < 1 || m.n_pages > INT32_MAX || m.page_tokens < kBlock ||
      m.page_tokens % kBlock || m.n_cols > INT32_MAX / m.page_tokens) {
    set_error("%s: invalid table (%lld x %lld), counts (%lld pages) or page size %lld", what,
              (long long)m.n_slots, (long long)m.n_cols, (long long)m.n_pages,
              (long long)m.page_tokens);
    return KVQ_ERR_INVALID;
  }
  return KVQ_OK;
}

inline View make_view(uint8_t* pool, int64_t n_pages, int64_t heads, int64_t dim, int64_t page_tokens,
                      const int32_t* table, int64_t n_slots, int64_t n_cols,
                      const int32_t* lengths, const int32_t* slots, const int32_t* indptr,
                      int64_t B, int64_t total) {
  View v;
  v.pool = pool;
  v.n_pages = n_pages;
  v.heads = (int)(heads < 0 || heads > INT32_MAX ? 0 : heads);
  v.dim = (int)(dim < 0 || dim > INT32_MAX ? 0 : dim);
  v.blocks = (int)(page_tokens / kBlock);
  v.table = table;
  v.n_slots = n_slots;
  v.n_cols = n_cols;
  v.lengths = lengths;
  v.slots = slots;
  v.indptr = indptr;
  v.B = B;
  v.total = total;
  return v;
}

template <int D, int KIND, typename T>
static int launch_append(const View& v, const void* k, int64_t k_tok, int64_t k_head,
                         const void* val, int64_t v_tok, int64_t v_head, const int32_t* granted,
                         cudaStream_t st) {
  const int64_t warps = block_items(v) * v.heads;
  const int64_t grid = (warps + kAppendWarps - 1) / kAppendWarps;
  return launch_next("paged_append", append_kernel<D, KIND, T>, dim3((unsigned)grid),
                     32 * kAppendWarps, 0, st, v, (const T*)k, k_tok, k_head, (const T*)val, v_tok,
                     v_head, granted, warps);
}

template <int D, int KIND, typename T>
static int launch_read(const View& v, const int32_t* starts, void* k, void* val, cudaStream_t st) {
  const int per_warp = block_items(v) * v.heads > 148 * 64 ? 4 : 1;
  const int64_t warps = block_items(v) * ((v.heads + per_warp - 1) / per_warp);
  const int64_t grid = (warps + kAppendWarps - 1) / kAppendWarps;
  return launch_next("paged_read", read_kernel<D, KIND, T>, dim3((unsigned)grid),
                     32 * kAppendWarps, 0, st, v, starts, (T*)k, (T*)val, warps, per_warp);
}

inline int launch_move(const char* what, const uint8_t* src, uint8_t* dst, int64_t src_layer,
                       int64_t dst_layer, int64_t page_bytes, int64_t n_layers,
                       const Moves* moves, const int2* list, const Renumber& rn, cudaStream_t st) {
  return launch_next(what, move_kernel, dim3(148 * 8), kPageThreads, 0, st, src, dst, src_layer,
                     dst_layer, page_bytes, (int)n_layers, moves, list, rn);
}

inline size_t plan_bytes(int64_t n_pages) {
  return sizeof(Moves) + (size_t)n_pages * (sizeof(int2) + sizeof(int32_t));
}

inline int check_pool(const char* what, const uint8_t* pool, int64_t n_layers, int64_t page_bytes) {
  if (!pool || !aligned16(pool) || n_layers < 1 || n_layers > INT32_MAX || page_bytes < 16 ||
      page_bytes % 16 || page_bytes > INT64_MAX / INT32_MAX) {
    set_error("%s: the pool must be 16-byte aligned with whole records (%lld layers, %lld bytes "
              "a page)", what, (long long)n_layers, (long long)page_bytes);
    return KVQ_ERR_INVALID;
  }
  return KVQ_OK;
}

}  // namespace paged
}  // namespace kvq

extern "C" int kvq_paged_append(const void* k, int64_t k_tok_stride, int64_t k_head_stride,
                                const void* v, int64_t v_tok_stride, int64_t v_head_stride,
                                int dtype, uint8_t* pool, int kind, int64_t n_pages,
                                int64_t n_heads, int64_t head_dim, int64_t page_tokens,
                                const int32_t* table, int64_t n_slots, int64_t n_cols,
                                const int32_t* lengths, const int32_t* slots,
                                const int32_t* indptr, int64_t B, int64_t total, void* stream) {
  return kvq_paged_append_granted(k, k_tok_stride, k_head_stride, v, v_tok_stride, v_head_stride,
                                  dtype, pool, kind, n_pages, n_heads, head_dim, page_tokens,
                                  table, n_slots, n_cols, lengths, slots, indptr, B, total,
                                  nullptr, stream);
}

extern "C" int kvq_paged_append_granted(const void* k, int64_t k_tok_stride, int64_t k_head_stride,
                                        const void* v, int64_t v_tok_stride, int64_t v_head_stride,
                                        int dtype, uint8_t* pool, int kind, int64_t n_pages,
                                        int64_t n_heads, int64_t head_dim, int64_t page_tokens,
                                        const int32_t* table, int64_t n_slots, int64_t n_cols,
                                        const int32_t* lengths, const int32_t* slots,
                                        const int32_t* indptr, int64_t B, int64_t total,
                                        const int32_t* granted, void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  const View w = make_view(pool, n_pages, n_heads, head_dim, page_tokens, table, n_slots, n_cols,
                           lengths, slots, indptr, B, total);
  int rc = check_view("paged_append", w, kind, page_tokens);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) {
    set_error("paged_append: dtype must be 0 (fp16) or 1 (bf16), got %d", dtype);
    return KVQ_ERR_UNSUPPORTED;
  }
  if (total == 0) return KVQ_OK;
  if (!k || !v || !aligned16(k) || !aligned16(v) || k_tok_stride % 8 || k_head_stride % 8 ||
      v_tok_stride % 8 || v_head_stride % 8) {
    set_error("paged_append: k and v rows must be 16-byte aligned (strides multiples of 8)");
    return KVQ_ERR_INVALID;
  }
  if (block_items(w) * w.heads > (int64_t)INT32_MAX * kAppendWarps) {
    set_error("paged_append: too many rows in one call");
    return KVQ_ERR_INVALID;
  }
  const cudaStream_t st = as_stream(stream);
#define KVQ_PAGED_APPEND(D, KIND, T) \
  launch_append<D, KIND, T>(w, k, k_tok_stride, k_head_stride, v, v_tok_stride, v_head_stride, \
                            granted, st)
#define KVQ_PAGED_PICK(D, T) \
  (kind == kInt8 ? KVQ_PAGED_APPEND(D, kInt8, T) : KVQ_PAGED_APPEND(D, kE4m3, T))
  if (head_dim == 64)
    return dtype == 0 ? KVQ_PAGED_PICK(64, __half) : KVQ_PAGED_PICK(64, __nv_bfloat16);
  return dtype == 0 ? KVQ_PAGED_PICK(128, __half) : KVQ_PAGED_PICK(128, __nv_bfloat16);
#undef KVQ_PAGED_PICK
#undef KVQ_PAGED_APPEND
}

extern "C" int kvq_paged_read(const uint8_t* pool, int kind, int64_t n_pages, int64_t n_heads,
                              int64_t head_dim, int64_t page_tokens, const int32_t* table,
                              int64_t n_slots, int64_t n_cols, const int32_t* lengths,
                              const int32_t* slots, const int32_t* starts, const int32_t* indptr,
                              int64_t B, int64_t total, void* k_out, void* v_out, int dtype,
                              void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  const View w = make_view(const_cast<uint8_t*>(pool), n_pages, n_heads, head_dim, page_tokens,
                           table, n_slots, n_cols, lengths, slots, indptr, B, total);
  int rc = check_view("paged_read", w, kind, page_tokens);
  if (rc) return rc;
  if (dtype < 0 || dtype > 2) {
    set_error("paged_read: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32), got %d", dtype);
    return KVQ_ERR_UNSUPPORTED;
  }
  if (total == 0) return KVQ_OK;
  if (!k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) {
    set_error("paged_read: the outputs must be 16-byte aligned");
    return KVQ_ERR_INVALID;
  }
  if (block_items(w) * w.heads > (int64_t)INT32_MAX * kAppendWarps) {
    set_error("paged_read: too many rows in one call");
    return KVQ_ERR_INVALID;
  }
  const cudaStream_t st = as_stream(stream);
#define KVQ_PAGED_READ(D, T)                                           \
  (kind == kInt8 ? launch_read<D, kInt8, T>(w, starts, k_out, v_out, st) \
                 : launch_read<D, kE4m3, T>(w, starts, k_out, v_out, st))
  if (head_dim == 64)
    return dtype == 0   ? KVQ_PAGED_READ(64, __half)
           : dtype == 1 ? KVQ_PAGED_READ(64, __nv_bfloat16)
                        : KVQ_PAGED_READ(64, float);
  return dtype == 0   ? KVQ_PAGED_READ(128, __half)
         : dtype == 1 ? KVQ_PAGED_READ(128, __nv_bfloat16)
                      : KVQ_PAGED_READ(128, float);
#undef KVQ_PAGED_READ
}

extern "C" int kvq_paged_free(int32_t* table, int64_t n_slots, int64_t n_cols, int32_t* lengths,
                              int32_t* refs, int64_t n_pages, int64_t page_tokens,
                              const int32_t* slots, int64_t n, int32_t* status, void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  const Meta m{table, n_slots, n_cols, lengths, refs, n_pages, page_tokens};
  int rc = check_meta("paged_free", m);
  if (rc) return rc;
  if (n < 0 || n > kMaxSeqs || !lengths || !status || (n && !slots)) {
    set_error("paged_free: %lld slots (0..%d), with lengths and status", (long long)n, kMaxSeqs);
    return KVQ_ERR_INVALID;
  }
  if (n == 0) return KVQ_OK;
  return launch_next("paged_free", free_kernel, dim3((unsigned)n), kPageThreads, 0,
                     as_stream(stream), m, slots, status);
}

extern "C" int kvq_paged_fork(int32_t* table, int64_t n_slots, int64_t n_cols, int32_t* lengths,
                              int32_t* refs, int64_t n_pages, int64_t page_tokens,
                              const int32_t* src, const int32_t* dst, int64_t n, int32_t* status,
                              void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  const Meta m{table, n_slots, n_cols, lengths, refs, n_pages, page_tokens};
  int rc = check_meta("paged_fork", m);
  if (rc) return rc;
  if (n < 0 || n > kMaxSeqs || !lengths || !status || (n && (!src || !dst))) {
    set_error("paged_fork: %lld pairs (0..%d), with lengths and status", (long long)n, kMaxSeqs);
    return KVQ_ERR_INVALID;
  }
  if (n == 0) return KVQ_OK;
  return launch_next("paged_fork", fork_kernel, dim3((unsigned)n), kPageThreads, 0,
                     as_stream(stream), m, src, dst, n, status);
}

extern "C" size_t kvq_paged_extend_workspace(int64_t n_pages) {
  return kvq::paged::plan_bytes(n_pages < 0 ? 0 : n_pages);
}

extern "C" int kvq_paged_extend(uint8_t* pool, int64_t n_layers, int64_t layer_stride,
                                int64_t page_bytes, int32_t* table, int64_t n_slots,
                                int64_t n_cols, int32_t* lengths, int32_t* refs, int64_t n_pages,
                                int64_t page_tokens, const int32_t* slots, int64_t n,
                                const int32_t* n_new, int64_t n_new_all, int32_t* status,
                                void* workspace, size_t workspace_bytes, void* stream) {
  return kvq_paged_extend_granting(pool, n_layers, layer_stride, page_bytes, table, n_slots, n_cols,
                                   lengths, refs, n_pages, page_tokens, slots, n, n_new, n_new_all,
                                   status, workspace, workspace_bytes, nullptr, stream);
}

extern "C" int kvq_paged_extend_granting(uint8_t* pool, int64_t n_layers, int64_t layer_stride,
                                         int64_t page_bytes, int32_t* table, int64_t n_slots,
                                         int64_t n_cols, int32_t* lengths, int32_t* refs,
                                         int64_t n_pages, int64_t page_tokens,
                                         const int32_t* slots, int64_t n, const int32_t* n_new,
                                         int64_t n_new_all, int32_t* status, void* workspace,
                                         size_t workspace_bytes, int32_t* granted, void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  const Meta m{table, n_slots, n_cols, lengths, refs, n_pages, page_tokens};
  int rc = check_meta("paged_extend", m);
  if (!rc) rc = check_pool("paged_extend", pool, n_layers, page_bytes);
  if (rc) return rc;
  if (n < 0 || n > kMaxSeqs || !lengths || !status || (n && !slots)) {
    set_error("paged_extend: %lld slots (0..%d), with lengths and status", (long long)n, kMaxSeqs);
    return KVQ_ERR_INVALID;
  }
  if (!n_new && (n_new_all < 0 || n_new_all > INT32_MAX / 2)) {
    set_error("paged_extend: %lld new tokens", (long long)n_new_all);
    return KVQ_ERR_INVALID;
  }
  if (layer_stride % 16 || (n_layers > 1 && layer_stride < n_pages * page_bytes)) {
    set_error("paged_extend: layer stride %lld", (long long)layer_stride);
    return KVQ_ERR_INVALID;
  }
  if (!workspace || !aligned16(workspace) || workspace_bytes < plan_bytes(n_pages)) {
    set_error("paged_extend: workspace too small or unaligned (%zu < %zu)", workspace_bytes,
              plan_bytes(n_pages));
    return KVQ_ERR_INVALID;
  }
  if (n == 0) return KVQ_OK;
  Moves* moves = static_cast<Moves*>(workspace);
  int2* list = reinterpret_cast<int2*>(moves + 1);
  int32_t* pages = reinterpret_cast<int32_t*>(list + n_pages);
  const cudaStream_t st = as_stream(stream);
  rc = launch_next("paged_extend", extend_kernel, dim3(1), kPlanThreads, 0, st, m, slots, n, n_new,
                   (int)n_new_all, status, moves, list, pages, granted);
  if (rc) return rc;
  return launch_move("paged_extend (copy)", pool, pool, layer_stride, layer_stride, page_bytes,
                     n_layers, moves, list, Renumber{}, st);
}

extern "C" int kvq_paged_compact(uint8_t* pool, int64_t n_layers, int64_t layer_stride,
                                 int64_t page_bytes, int32_t* table, int64_t n_slots,
                                 int64_t n_cols, int32_t* refs, int64_t n_pages, int32_t* n_live,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  const Meta m{table, n_slots, n_cols, nullptr, refs, n_pages, kBlock};
  int rc = check_meta("paged_compact", m);
  if (!rc) rc = check_pool("paged_compact", pool, n_layers, page_bytes);
  if (rc) return rc;
  if (!n_live) {
    set_error("paged_compact: n_live is null");
    return KVQ_ERR_INVALID;
  }
  if (layer_stride % 16 || (n_layers > 1 && layer_stride < n_pages * page_bytes)) {
    set_error("paged_compact: layer stride %lld", (long long)layer_stride);
    return KVQ_ERR_INVALID;
  }
  if (!workspace || !aligned16(workspace) || workspace_bytes < plan_bytes(n_pages)) {
    set_error("paged_compact: workspace too small or unaligned (%zu < %zu)", workspace_bytes,
              plan_bytes(n_pages));
    return KVQ_ERR_INVALID;
  }
  Moves* moves = static_cast<Moves*>(workspace);
  int2* list = reinterpret_cast<int2*>(moves + 1);
  int32_t* new_id = reinterpret_cast<int32_t*>(list + n_pages);
  const cudaStream_t st = as_stream(stream);
  rc = launch_next("paged_compact", compact_kernel, dim3(1), kPlanThreads, 0, st, refs, n_pages,
                   moves, list, new_id, n_live);
  if (rc) return rc;
  return launch_move("paged_compact (copy)", pool, pool, layer_stride, layer_stride, page_bytes,
                     n_layers, moves, list,
                     Renumber{table, n_slots * n_cols, refs, n_pages, new_id, n_live}, st);
}

extern "C" size_t kvq_paged_copy_workspace(int64_t n) {
  return sizeof(kvq::paged::Moves) + (n < 0 ? 0 : (size_t)n) * sizeof(int2);
}

extern "C" int kvq_paged_copy(const uint8_t* src_pool, int64_t src_pages,
                              int64_t src_layer_stride, uint8_t* dst_pool, int64_t dst_pages,
                              int64_t dst_layer_stride, int64_t n_layers, int64_t page_bytes,
                              const int32_t* src, const int32_t* dst, int64_t n, void* workspace,
                              size_t workspace_bytes, void* stream) {
  using namespace kvq;
  using namespace kvq::paged;
  clear_error();
  int rc = check_pool("paged_copy", src_pool, n_layers, page_bytes);
  if (!rc) rc = check_pool("paged_copy", dst_pool, n_layers, page_bytes);
  if (rc) return rc;
  if (n < 0 || n > INT32_MAX || (n && (!src || !dst)) || src_pages < 1 || dst_pages < 1 ||
      src_pages > INT32_MAX || dst_pages > INT32_MAX || src_layer_stride % 16 ||
      dst_layer_stride % 16 ||
      (n_layers > 1 && (src_layer_stride < src_pages * page_bytes ||
                        dst_layer_stride < dst_pages * page_bytes))) {
    set_error("paged_copy: invalid pairs (%lld), pools (%lld, %lld pages) or layer strides",
              (long long)n, (long long)src_pages, (long long)dst_pages);
    return KVQ_ERR_INVALID;
  }
  if (n == 0) return KVQ_OK;
  if (!workspace || !aligned16(workspace) || workspace_bytes < kvq_paged_copy_workspace(n)) {
    set_error("paged_copy: workspace too small or unaligned (%zu < %zu)", workspace_bytes,
              kvq_paged_copy_workspace(n));
    return KVQ_ERR_INVALID;
  }
  Moves* moves = static_cast<Moves*>(workspace);
  int2* list = reinterpret_cast<int2*>(moves + 1);
  const cudaStream_t st = as_stream(stream);
  rc = launch_next("paged_copy", pairs_kernel, dim3(1), kPageThreads, 0, st, src, src_pages, dst,
                   dst_pages, n, moves, list);
  if (rc) return rc;
  return launch_move("paged_copy (pages)", src_pool, dst_pool, src_layer_stride, dst_layer_stride,
                     page_bytes, n_layers, moves, list, Renumber{}, st);
}
