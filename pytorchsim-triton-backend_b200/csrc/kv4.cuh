// The 4-bit paged cache of keys and values (format: include/ptsim_b200.h, ptsim_kv4_params): store, load and the attention
// of one new token per slot.  No counterpart in the reference, whose decode program reads a dense bf16 cache (decode.cuh).
//
// Attention.  With codes c, scale a and minimum b per (key, group of the head dimension), the cached key is a c + b =
// a (c - 8) + (b + 8 a) and the score z = sum_g a_g (q . (c - 8))_g + (b_g + 8 a_g) sum(q)_g: the tensor core multiplies q by
// small integers, exact in 16 bits, and the parameters enter in fp32, once per (key, group).  Likewise
// O = sum_k (p a_g) (c - 8) + p (b_g + 8 a_g), with p a_g rounded to fp16 as the product's operand (2^-12 of what multiplies
// |c - 8| <= 8; small ones: kKvTop) and the second sum kept per row in fp32.  Both products run in fp16 whatever the cache's type: a byte of two
// codes becomes two fp16 operands by half a byte permute (0x64 above the byte: 1024 + lo + 16 hi), one mask-and-or
// (1032 + 16 hi), one subtraction (lo - 8) and one fused multiply-add (hi - 8), two of them on the FMA pipe; bf16, with 7 bits
// of mantissa, takes a shift more per pair, all on the half-rate ALU pipe, which bounded that form (63 % busy, 467 warp
// instructions per 16 keys, 166 us of kernel at 4 slots of up to 131072 keys; this one 310 and 111 us).  Queries fit fp16 after division
// by their row's power of two; the weights' V scales by a power of two that follows the largest scale seen.  The operands are centred because a
// constant offset costs the sums their low bits: with 128 + c for V, 10^5 keys ended 2.4e-2 off (the tensor core truncates).
//
// The products have K and V as the 16-row operand: S^T = K q^T, O^T = V^T P^T (mma.sync m16n8k16, N = 8 query rows of one KV
// head), so up to 8 query heads per KV head waste nothing, half of what a 16-row query tile costs; tcgen05.mma, whose
// smallest M is 64 and whose operands come from shared memory as 16 bits, would need the unpacked tile written back.  Both operands
// take their k index in any order both sides agree on, which the page format uses: 16-byte (K) and 8-byte (V) shared loads
// without bank conflicts give words whose nibbles are the fragments.
//
// Bound: HBM, (D + 8 D / group) bytes per key and KV head (144 at D 128, group 64: 3.5 times fewer than bf16), and before
// it the issue slots (60 % busy with three warps per scheduler, ALU 47 %; a fourth warp, at 128 registers, changed nothing): of the
// 310 warp instructions per 16 keys 120 unpack (48 for K, 72 for V), the rest are parameters, weights, maxima, products and parts,
// and with four query rows a KV head half of the lanes' weights are padding.  Both kernels: 64 slots of up to 8191 keys 65 us, 3.7 TB/s
// of cache; 4 slots of up to 131072 keys 118 us, 4.1 TB/s, 0.64 of the measured copy bandwidth.  Work is one list of 64-key tiles over (slot, KV head), cut into equal contiguous
// ranges, one per warp: a warp streams its tiles by bulk copies through a ring of its own (no barrier between warps) and keeps
// the online softmax in registers.  Lengths are read on the device, so any raggedness is balanced to a tile.  A range that
// holds only part of an item leaves (m, l, O) in the workspace and a second kernel (a programmatic dependent) merges the parts
// in key order: results do not depend on timing.
#pragma once
#include "sm100.cuh"
#include "decode.cuh"
#include "packed.cuh"
#include "pages.cuh"

namespace ptsim {

constexpr int kKvTile = 64;          // keys of a tile: what a warp is given and copies at once
constexpr int kKvPass = 32;          // keys of one pass over the softmax
constexpr int kKvStages = 2;
constexpr int kKvWarps = 4;

struct Kv4Args {
  const uint8_t *pool;               // of the launch's layer
  const int32_t *lens, *table, *cu;
  const int32_t *halt;               // (store) nonzero: write nothing; or null
  uint16_t *a, *b;                   // K and V, or q and o
  int64_t a_row, a_head, b_row, b_head;
  int64_t record;                    // bytes of one (page, KV head)
  int32_t tokens, slots, hkv, per, rb;   // per: query heads of a KV head; rb: blocks of 16 of them
  int32_t pages, page_size, page_log, max_pages;
  float sl;                          // scale * log2 e
  float *part_o, *part_ml;           // [2 * workers][16][D] and [2 * workers][16][2]
  int32_t *before;                   // [slots + 1] units of an item before a slot (kv4_units), for the merge
  int32_t workers, stall;
};

// 16-bit value <-> fp32 of the cache's type.
template <bool F16>
__device__ __forceinline__ float to_f32(uint32_t bits16) {
  if (!F16) return __uint_as_float(bits16 << 16);
  float f;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.f32.f16 %0, h;\n\t}" : "=f"(f) : "r"(bits16));
  return f;
}
template <bool F16>
__device__ __forceinline__ float lo_f32(uint32_t w) { return F16 ? to_f32<true>(w & 0xffffu) : lo_bf16(w); }
template <bool F16>
__device__ __forceinline__ float hi_f32(uint32_t w) { return F16 ? to_f32<true>(w >> 16) : hi_bf16(w); }

// The slot whose rows cu[s] .. cu[s + 1] hold row t, and the row's position in the slot's sequence (the rows are its
// last); -1 when the row is in no slot.  Whole warp; 32 table entries a step.
__device__ __forceinline__ int kv4_find(const Kv4Args &g, int t, int lane, int64_t *pos) {
  int lo = 0, n = g.slots;
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int at = lo + min((lane + 1) * step, n);
    const bool below = (lane + 1) * step < n && g.cu[at] <= t;
    const int k = __popc(__ballot_sync(0xffffffffu, below));
    lo += k * step;
    n = min(step, n - k * step);
  }
  const int c0 = g.cu[lo], c1 = g.cu[lo + 1];
  if (t < c0 || t >= c1) return -1;
  *pos = int64_t(g.lens[lo]) - c1 + t;
  return lo;
}

// The pool page of position `pos` of slot s, or -1 (recorded) when the row or the pool does not hold it.
__device__ __forceinline__ int kv4_page(const Kv4Args &g, int s, int64_t pos, int lane) {
  int page = -1;
  if (pos >= 0 && (pos >> g.page_log) < g.max_pages) page = g.table[int64_t(s) * g.max_pages + (pos >> g.page_log)];
  if (page >= 0 && page < g.pages) return page;
  if (lane == 0) record_status(PTSIM_E_OOB);
  return -1;
}

// Where lane i of a (token, head) keeps its word: lanes 0 .. D/8 - 1 hold K words (d = 8 i ..), the next D/8 V words
// (d = w 64 + 4 c .. and w 64 + 32 + 4 c .., c = i % 8, w = i / 8), in the block that begins at `rec`.
template <int D, int NG>
struct Kv4Lane {
  static constexpr int kLanes = D / 4;             // lanes of one (token, head)
  int i, d0, d1, word;
  bool is_v;
  __device__ __forceinline__ Kv4Lane(int lane) {
    const int l = lane % kLanes;
    is_v = l >= D / 8;
    i = l % (D / 8);
    d0 = is_v ? (i >> 3) * 64 + (i & 7) * 4 : i * 8;
    d1 = is_v ? d0 + 32 : d0 + 4;
    word = is_v ? (i & 7) * (D / 64) + (i >> 3) : (i & 3) * (D / 32) + (i >> 2);
  }
  // Byte offsets within a record of this lane's word and of its token's parameters.
  __device__ __forceinline__ void place(int at, int page_log, int *code, int *par) const {
    const int bs_log = min(page_log, 5), bs = 1 << bs_log;
    const int base = (at >> bs_log) * (bs * (D + 8 * NG)), t = at & (bs - 1);
    const int r = is_v ? (t & ~7) | ((t & 1) << 2) | ((t >> 1) & 3) : t;
    const int w = is_v && D == 128 && (r & 2) ? word ^ 8 : word;
    *code = base + (is_v ? bs * (D / 2) : 0) + r * (D / 2) + w * 4;
    *par = base + bs * D + (is_v ? bs * 4 * NG : 0) + t * 4 * NG;
  }
};

// Minimum of the halves of a and b, a NaN where either is one.
template <bool F16>
__device__ __forceinline__ uint32_t min_16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (F16) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t max_16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (F16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// (minimum, -maximum), as a pair, of two minima and two maxima.
template <bool F16>
__device__ __forceinline__ uint32_t extremes(uint32_t lo, uint32_t hi) {
  return min_16x2<F16>(__byte_perm(lo, hi, 0x5410) ^ 0x80000000u, __byte_perm(lo, hi, 0x7632) ^ 0x80000000u);
}

// half / 7.5 correctly rounded: the quotient by the rounded reciprocal, corrected by its exact remainder (Markstein's
// method, for a divisor known in advance).
__device__ __forceinline__ float over_seven_and_a_half(float half) {
  constexpr float r = 1.f / 7.5f;
  const float q = half * r;
  return fmaf(fmaf(-7.5f, q, half), r, q);
}

// Eight values (two runs of four, a scale and a minimum for each) to codes, nibble e the e-th value: rint of the fp32 quotient
// y / step, y = x - mn.  The quotient by the approximate reciprocal, corrected by its exact remainder, is within 2^-43 of y / step
// before its rounding, and no y / step (24 bits by at most 11) lies on or within 2^-35 of the middle of two floats: it
// is the rounded quotient, ties of codes (every 400th value of a bf16 grid) included.  A float plus 1.5 * 2^23 is rounded to an
// integer in its low byte; of the eight bytes `even` takes the low nibbles of the result, `odd` the high ones.
template <bool F16>
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&w)[4], const float (&step)[2], const float (&mn)[2], uint32_t even, uint32_t odd) {
  // Steps from kTiny on are rounded by at most 2^-9 of themselves: no quotient passes 15.5, remainders are exact and the
  // reciprocal is a normal number; up to kHuge y does not overflow.
  constexpr float kMagic = 12582912.f, kTiny = F16 ? 6.103515625e-5f : 1e-30f, kHuge = 2e37f;
  uint32_t run[2];                     // the codes of four values, one a byte
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float2 m2 = make_float2(-mn[k], -mn[k]), s2 = make_float2(-step[k], -step[k]);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(step[k]));
    const float2 r2 = make_float2(r, r);
    uint32_t pair[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t x = w[2 * k + e];
      const float2 y = __fadd2_rn(make_float2(lo_f32<F16>(x), hi_f32<F16>(x)), m2), q0 = __fmul2_rn(y, r2);
      const float2 q = __ffma2_rn(__ffma2_rn(s2, q0, y), r2, q0), t = __fadd2_rn(q, make_float2(kMagic, kMagic));
      pair[e] = __byte_perm(__float_as_uint(t.x), __float_as_uint(t.y), 0x0040);
    }
    run[k] = __byte_perm(pair[0], pair[1], 0x5410);
  }
  // A step too small for its reciprocal or a range too large for y: halves, which fp32 holds exactly, and the division.  No step (a
  // constant, or no number): code 0.
  const auto rare = [](float s) { return s < kTiny || (!F16 && s > kHuge); };
  if (rare(step[0]) || rare(step[1])) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!rare(step[k])) continue;
      run[k] = 0;
      if (step[k] == 0.f) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = w[2 * k + e / 2];
        const float y = (e & 1 ? hi_f32<F16>(x) : lo_f32<F16>(x)) * 0.5f - mn[k] * 0.5f;
        run[k] |= uint32_t(fminf(rintf(__fdiv_rn(y, step[k] * 0.5f)), 15.f)) << (8 * e);
      }
    }
  }
  return __byte_perm(run[0], run[1], even) + 16 * __byte_perm(run[0], run[1], odd);
}

// One (token, head) per D / 4 lanes, eight values a lane, `HS` steps of 128 / D heads a warp: their loads are issued before the
// token's place is looked up, so a warp waits for the two once.  Extremes are packed 16-bit minima of x and -x, one shuffle a step.
// HBM is the floor (K and V read, D + 8 D / group bytes written per head: 16 us at 24062 tokens of 8 heads of 128), the issue slots
// bound it: 143 warp instructions per (token, head), 71 % busy, 39 us; 135 us with divisions and one head a warp, 43 with four.
// The lookup is 150 of a warp's instructions, so a grid of tokens by heads, without a division, and many steps.
template <int D, int NG, bool F16, int HS>
__global__ void __launch_bounds__(256) kv4_store_kernel(const __grid_constant__ Kv4Args g, uint8_t *pool) {
  constexpr int kLanes = D / 4, kHeads = 32 / kLanes, kGroup = D / NG;
  const int lane = threadIdx.x & 31;
  const uint32_t t = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int h0 = int(blockIdx.y) * (kHeads * HS) + lane / kLanes;
  pdl_enter();
  if (halted(g.halt) || t >= uint32_t(g.tokens)) return;
  const Kv4Lane<D, NG> me(lane);
  const uint16_t *src = me.is_v ? g.b + t * g.b_row : g.a + t * g.a_row;
  const int64_t step_h = me.is_v ? g.b_head : g.a_head;
  uint32_t w[HS][4];
#pragma unroll
  for (int i = 0; i < HS; ++i) {
    const int h = h0 + i * kHeads;
    uint2 x0 = make_uint2(0, 0), x1 = x0;
    if (h < g.hkv) {
      x0 = *reinterpret_cast<const uint2 *>(src + h * step_h + me.d0);
      x1 = *reinterpret_cast<const uint2 *>(src + h * step_h + me.d1);
    }
    w[i][0] = x0.x, w[i][1] = x0.y, w[i][2] = x1.x, w[i][3] = x1.y;
  }
  int64_t pos = 0;
  const int slot = kv4_find(g, int(t), lane, &pos);
  if (slot < 0) return;
  const int page = kv4_page(g, slot, pos, lane);
  if (page < 0) return;
  int code_at, par_at;
  me.place(int(pos) & ((1 << g.page_log) - 1), g.page_log, &code_at, &par_at);
  uint8_t *rec = pool + int64_t(page) * g.hkv * g.record;
  const uint32_t even = me.is_v ? 0x6420 : 0x5140, odd = me.is_v ? 0x7531 : 0x7362;   // K: value d in nibble d / 2 + 4 (d % 2)
#pragma unroll
  for (int i = 0; i < HS; ++i) {
    const int h = h0 + i * kHeads;
    if (h - lane / kLanes >= g.hkv) break;                                // the whole warp
    // (minimum, -maximum) of the lane's two runs of four; one group but for V in groups of 32.
    const uint32_t lo0 = min_16x2<F16>(w[i][0], w[i][1]), lo1 = min_16x2<F16>(w[i][2], w[i][3]);
    const uint32_t hi0 = max_16x2<F16>(w[i][0], w[i][1]), hi1 = max_16x2<F16>(w[i][2], w[i][3]);
    uint32_t m0 = extremes<F16>(min_16x2<F16>(lo0, lo1), max_16x2<F16>(hi0, hi1)), m1 = m0;
    if (kGroup == 32 && me.is_v) m0 = extremes<F16>(lo0, hi0), m1 = extremes<F16>(lo1, hi1);
    // Lanes of a group: group / 8 consecutive ones (V in groups of 32: the eight lanes of its 64 values, by run).
#pragma unroll
    for (int s = 1; s < (kGroup > 64 ? 16 : 8); s *= 2) {
      const uint32_t a = min_16x2<F16>(m0, __shfl_xor_sync(0xffffffffu, m0, s));
      const uint32_t b = kGroup > 32 ? a : min_16x2<F16>(m1, __shfl_xor_sync(0xffffffffu, m1, s));
      if (kGroup > 32 || s < 4 || me.is_v) m0 = a, m1 = b;
    }
    float step[2], mn[2];
    uint32_t par[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t m = r ? m1 : m0;
      mn[r] = lo_f32<F16>(m);
      const float half = hi_f32<F16>(m) * -0.5f - mn[r] * 0.5f;           // half the range: the range itself could overflow
      const bool fine = half < INFINITY;                                  // false for NaN too
      par[r] = fine ? pack_16x2<F16>(over_seven_and_a_half(half), mn[r]) : (F16 ? 0x7e007e00u : 0x7fc07fc0u);   // the minimum is exact
      step[r] = fine ? lo_f32<F16>(par[r]) : 0.f;                         // a group that is no number: codes 0
    }
    const uint32_t word = quantise8<F16>(w[i], step, mn, even, odd);
    if (h >= g.hkv) continue;
    uint8_t *to = rec + h * g.record;
    *reinterpret_cast<uint32_t *>(to + code_at) = word;
    // The first lane of each group writes its parameters.
    if (me.d0 % kGroup == 0) *reinterpret_cast<uint32_t *>(to + par_at + 4 * (me.d0 / kGroup)) = par[0];
    if (kGroup == 32 && me.is_v && (me.i & 7) == 0) *reinterpret_cast<uint32_t *>(to + par_at + 4 * (me.d1 / kGroup)) = par[1];
  }
}

// The reverse, the same lanes and steps: 86 warp instructions per (token, head), 25 us where the bytes take 16; 78 us with one
// head a warp, 28 with four.
template <int D, int NG, bool F16, int HS>
__global__ void __launch_bounds__(256) kv4_load_kernel(const __grid_constant__ Kv4Args g) {
  constexpr int kLanes = D / 4, kHeads = 32 / kLanes, kGroup = D / NG;
  const int lane = threadIdx.x & 31;
  const uint32_t t = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int h0 = int(blockIdx.y) * (kHeads * HS) + lane / kLanes;
  pdl_enter();
  if (t >= uint32_t(g.tokens)) return;
  int64_t pos = 0;
  const int slot = kv4_find(g, int(t), lane, &pos);
  if (slot < 0) return;
  const int page = kv4_page(g, slot, pos, lane);
  const Kv4Lane<D, NG> me(lane);
  int code_at, par_at;
  me.place(int(pos) & ((1 << g.page_log) - 1), g.page_log, &code_at, &par_at);
  const uint8_t *rec = g.pool + int64_t(max(page, 0)) * g.hkv * g.record;
  uint32_t word[HS], p0[HS], p1[HS];
#pragma unroll
  for (int i = 0; i < HS; ++i) {
    const int h = h0 + i * kHeads;
    word[i] = p0[i] = p1[i] = 0;                              // a page outside the pool reads as zeros
    if (page < 0 || h >= g.hkv) continue;
    const uint8_t *at = rec + h * g.record;
    word[i] = *reinterpret_cast<const uint32_t *>(at + code_at);
    p0[i] = *reinterpret_cast<const uint32_t *>(at + par_at + 4 * (me.d0 / kGroup));
    p1[i] = kGroup > 32 ? p0[i] : *reinterpret_cast<const uint32_t *>(at + par_at + 4 * (me.d1 / kGroup));
  }
  // Bytes of values 0 - 3 and 4 - 7: K keeps value d in nibble d / 2 + 4 (d % 2), so low nibbles are one pair, V value e in nibble e.
  const uint32_t bytes0 = me.is_v ? 0x4140 : 0x4240, bytes1 = me.is_v ? 0x4342 : 0x4341;
  const uint32_t pair0 = me.is_v ? 0x5410 : 0x3210, pair1 = me.is_v ? 0x7632 : 0x7654;
  uint16_t *dst = me.is_v ? g.b + t * g.b_row : g.a + t * g.a_row;
  const int64_t step_h = me.is_v ? g.b_head : g.a_head;
#pragma unroll
  for (int i = 0; i < HS; ++i) {
    const int h = h0 + i * kHeads;
    if (h - lane / kLanes >= g.hkv) break;                    // the whole warp
    // Two bytes at a time: 1024 + lo + 16 hi, less 1024 + 16 hi is lo, and a sixteenth of that less 64 is hi, in fp16 and exact.
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t par = e ? p1[i] : p0[i], x2 = __byte_perm(word[i], 0x64646464u, e ? bytes1 : bytes0), y = x2 & 0xfff0fff0u;
      uint32_t lo, hi;
      asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(x2), "r"(y));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(hi) : "r"(y), "r"(0x2c002c00u), "r"(0xd400d400u));
      const float s = lo_f32<F16>(par), mn = hi_f32<F16>(par);
      const float2 s2 = make_float2(s, s), mn2 = make_float2(mn, mn);
      const float2 a = __ffma2_rn(s2, make_float2(lo_f32<true>(lo), hi_f32<true>(lo)), mn2);
      const float2 b = __ffma2_rn(s2, make_float2(lo_f32<true>(hi), hi_f32<true>(hi)), mn2);
      const uint32_t o0 = pack_16x2<F16>(a.x, a.y), o1 = pack_16x2<F16>(b.x, b.y);
      out[2 * e] = __byte_perm(o0, o1, pair0), out[2 * e + 1] = __byte_perm(o0, o1, pair1);
    }
    if (h >= g.hkv) continue;
    *reinterpret_cast<uint2 *>(dst + h * step_h + me.d0) = make_uint2(out[0], out[1]);
    *reinterpret_cast<uint2 *>(dst + h * step_h + me.d1) = make_uint2(out[2], out[3]);
  }
}

// -------------------------------------------------------------------------------------------------------------------
// Attention
// -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_16n8_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same product onto c0 in the even columns and c1 in the odd ones.
__device__ __forceinline__ void mma_16n8_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// x = a pair of fp16 1024 + lo + 16 hi (codes lo, hi of a byte): the pairs lo - 8 and hi - 8, exact.
__device__ __forceinline__ void split_codes(uint32_t x, uint32_t &lo, uint32_t &hi) {
  const uint32_t y = and_or(x, 0xfff0fff0u, 0x00080008u);                                // 1032 + 16 hi
  asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(y));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(hi) : "r"(y), "r"(0x2c002c00u), "r"(0xd488d488u));   // y / 16 - 72.5
}

// The pairs lo - 8 and 1032 + 16 hi.
__device__ __forceinline__ void split_offset(uint32_t x, uint32_t &lo, uint32_t &hi) {
  hi = and_or(x, 0xfff0fff0u, 0x00080008u);
  asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(x), "r"(hi));
}

// How far (log2) a score may pass its row's reference before the reference moves, and where (log2) the largest V scale seen is
// brought by a power of two.  A weight times a scale is an fp16 operand, at most 2^(4 + 11); with the largest scale it is rounded by
// 2^-12 of itself down to weights of 2^-24 (16 below the row's top score) and by 2^-35 of that scale behind.  A reference that moves
// at 2^8 leaves a range of 2^-20 for the same times (64 slots of up to 8191 keys 65.2 us, 65.3 with 2^4), one at 2^2 costs the
// rows that share a warp more moves (33 slots of up to 5000 keys, 16 rows a KV head of 64: 20.0 us, 18.6 with 2^4).
constexpr int kKvGrow = 4, kKvTop = 15 - kKvGrow;

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// Tiles of a slot of length `len`, 0 (recorded) for a length the table's row cannot hold.
__device__ __forceinline__ int kv4_tiles(const Kv4Args &g, int len) {
  if (len < 0 || len > int64_t(g.max_pages) * g.page_size) {
    record_status(PTSIM_E_OOB);
    return 0;
  }
  return (len + kKvTile - 1) / kKvTile;
}

// Work list: every item (KV head, row block) of every slot that holds keys, kKvItemCost units and then a unit per tile; worker w
// takes units [w c, (w + 1) c), c = kv4_share.  The cost stands for what a part costs beside its tiles (q fetched and
// converted, sums over lanes, the part written: about one tile); without it the workers that got many short items ended a
// fifth after the others (64 slots of up to 8191 keys).
constexpr int kKvItemCost = 1;
__device__ __forceinline__ int kv4_units(int tiles) { return tiles > 0 ? tiles + kKvItemCost : 0; }
// Units of a worker: the list's length over the workers, rounded up (the last workers may get none, the longest range is
// no longer than in an even cut).
__device__ __forceinline__ uint32_t kv4_share(uint32_t total, int workers) { return (total + uint32_t(workers) - 1) / uint32_t(workers); }

template <int D, int NG, int NT, bool F16>
__global__ void __launch_bounds__(kKvWarps * 32, NT == 1 && NG < 4 ? 3 : 2) kv4_attn_kernel(const __grid_constant__ Kv4Args g) {
  constexpr int kStage = kKvTile * (D + 8 * NG);            // bytes of a tile: two blocks of 32 keys or four of 16
  constexpr int kWordsK = D / 32, kWordsV = D / 64;         // words a lane takes of a K and of a V row
  constexpr int kGroup = D / NG;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *ring = smem + (threadIdx.x >> 5) * kKvStages * kStage;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kKvWarps * kKvStages * kStage) + (threadIdx.x >> 5) * kKvStages;
  int32_t *good = reinterpret_cast<int32_t *>(smem + kKvWarps * kKvStages * (kStage + 8)) + (threadIdx.x >> 5) * kKvStages;
  int32_t *sums = reinterpret_cast<int32_t *>(smem + kKvWarps * kKvStages * (kStage + 12));   // [2 * kKvWarps]
  int32_t *before = sums + 2 * kKvWarps;                    // [slots + 1] units of an item before a slot
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, qd = lane & 3;
  const uint32_t wl = g.stall ? kTestWaitUs : kWaitUs;
  if (lane == 0) {
    for (int i = 0; i < kKvStages; ++i) sm100::mbar_init(&full[i], 1);
    sm100::fence_barrier_init();
  }
  pdl_enter();

  // before[s], and how many slots before s hold keys: a thread sums a run of slots, the runs are scanned over the CTA.
  uint16_t *held = reinterpret_cast<uint16_t *>(before + g.slots + 1);
  const int run = (g.slots + kKvWarps * 32 - 1) / (kKvWarps * 32), s_lo = threadIdx.x * run;
  int mine = 0, some = 0;
  for (int s = s_lo; s < min(s_lo + run, g.slots); ++s) {
    const int u = kv4_units(kv4_tiles(g, g.lens[s]));
    mine += u;
    some += u > 0;
  }
  int scan = mine, scan2 = some;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o), up2 = __shfl_up_sync(0xffffffffu, scan2, o);
    if (lane >= o) scan += up, scan2 += up2;
  }
  if (lane == 31) sums[warp] = scan, sums[kKvWarps + warp] = scan2;
  __syncthreads();
  for (int w = 0; w < warp; ++w) scan += sums[w], scan2 += sums[kKvWarps + w];
  int at = scan - mine, at2 = scan2 - some;
  for (int s = s_lo; s < min(s_lo + run, g.slots); ++s) {
    before[s] = at;
    held[s] = uint16_t(at2);
    const int u = kv4_units(kv4_tiles(g, g.lens[s]));
    at += u;
    at2 += u > 0;
  }
  if (threadIdx.x == kKvWarps * 32 - 1) before[g.slots] = scan, held[g.slots] = uint16_t(scan2);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = threadIdx.x; s <= g.slots; s += kKvWarps * 32) g.before[s] = before[s];

  const int items = g.hkv * g.rb;                           // items of a slot
  const uint32_t total = uint32_t(before[g.slots]) * uint32_t(items), share = kv4_share(total, g.workers);
  const uint32_t worker = uint32_t(warp) * gridDim.x + blockIdx.x;
  const uint64_t from = uint64_t(worker) * share;
  if (from >= total) return;
  const uint32_t w_lo = uint32_t(from), w_hi = uint32_t(min(from + share, uint64_t(total)));

  // Position in the list: slot, its length and tiles, KV head and row block, tile of the item.
  struct Cursor {
    int slot, len, tiles, head, block, tile;
  };
  // The tile that unit x belongs to (an item's first one for the units of its cost); *index: tiles before it in the list.
  auto seek = [&](uint32_t x, uint32_t *index) {
    int lo = 0, hi = g.slots;                               // the last slot with before * items <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (uint32_t(before[mid]) * uint32_t(items) <= x) lo = mid;
      else hi = mid;
    }
    Cursor c;
    c.slot = lo;
    const uint32_t units = uint32_t(before[lo + 1] - before[lo]), in = x - uint32_t(before[lo]) * uint32_t(items), item = in / units;
    c.tiles = int(units) - kKvItemCost;
    c.head = int(item);
    c.block = 0;
    if (g.rb > 1) c.head = int(item) / g.rb, c.block = int(item) % g.rb;
    c.tile = max(0, int(in - item * units) - kKvItemCost);
    *index = uint32_t(before[lo] - kKvItemCost * held[lo]) * uint32_t(items) + item * uint32_t(c.tiles) + uint32_t(c.tile);
    return c;
  };
  auto next_item = [&](Cursor &c) {
    c.tile = 0;
    if (++c.block < g.rb) return;
    c.block = 0;
    if (++c.head < g.hkv) return;
    c.head = 0;
    do {
      ++c.slot;
      c.tiles = c.slot < g.slots ? before[c.slot + 1] - before[c.slot] - kKvItemCost : 1;
    } while (c.tiles <= 0);
    c.len = c.slot < g.slots ? g.lens[c.slot] : 0;
  };

  // Producer side: lane k < parts holds the pool page of the k-th part of the tile that is copied next.
  const int bs = 1 << min(g.page_log, 5), part_log = min(g.page_log, 6), parts = kKvTile >> part_log;   // a block's keys; a copy's
  const uint32_t part_bytes = uint32_t((D + 8 * NG) << part_log);
  auto next_page = [&](const Cursor &c) {
    int page = -2;                                          // -2: no key of the slot lies there
    const int first = c.tile * kKvTile + (lane << part_log);
    if (lane < parts && first < c.len) {
      page = g.table[int64_t(c.slot) * g.max_pages + (first >> g.page_log)];
      if (page < 0 || page >= g.pages) page = -1;
    }
    return page;
  };
  int fill_st = 0;
  auto copy = [&](const Cursor &c, int page, bool withheld) {
    const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0);
    if (lane < parts && page == -1) record_status(PTSIM_E_OOB);
    if (lane == 0) {
      good[fill_st] = int(ok);
      sm100::mbar_arrive_expect_tx(&full[fill_st], part_bytes * __popc(ok));
    }
    __syncwarp();
    if (page >= 0 && !withheld) {
      const int part = ((c.tile * kKvTile + (lane << part_log)) & ((1 << g.page_log) - 1)) >> part_log;
      const uint8_t *src = g.pool + (int64_t(page) * g.hkv + c.head) * g.record + uint32_t(part) * part_bytes;
      sm100::bulk_load_g2s(ring + fill_st * kStage + lane * part_bytes, src, part_bytes, &full[fill_st]);
    }
    fill_st = fill_st + 1 == kKvStages ? 0 : fill_st + 1;
  };

  uint32_t index, end = uint32_t(before[g.slots] - kKvItemCost * held[g.slots]) * uint32_t(items);
  Cursor use = seek(w_lo, &index);
  use.len = g.lens[use.slot];
  Cursor fill = use;
  int filled = 0, page = next_page(fill);
  if (w_hi < total) seek(w_hi, &end);
  const int count = int(end - index);                       // 0: units of an item's cost only
  if (count == 0) return;
  auto feed = [&]() {                                       // copy the next tile, then fetch the pages of the one after it
    if (filled >= count) return;
    copy(fill, page, g.stall && index == 0 && filled == 0);   // test hook: armed, no copy in flight
    if (++filled < count) {
      if (++fill.tile == fill.tiles) next_item(fill);
      page = next_page(fill);
    }
  };
  for (int i = 0; i < kKvStages; ++i) feed();

  // Offsets of a 16-key step within a tile.
  const bool small = bs == 16;
  const int step_k = small ? 16 * (D + 8 * NG) : 8 * D, step_p = small ? 16 * (D + 8 * NG) : 64 * NG;
  const int v_at = bs * (D / 2) + qd * (D / 2) + (D == 128 ? (gq ^ ((qd & 2) << 1)) * 8 : gq * 4);
  const int kp_at = bs * D + gq * NG * 4, vp_at = kp_at + bs * 4 * NG;

  bool ok = true;
  int done = 0, st = 0, phase = 0;
  while (done < count) {
    // One item's part: tiles [use.tile, last) of (slot, KV head, row block).
    const int slot = use.slot, head = use.head, row0 = use.block * 16, len = use.len;
    const int first = use.tile, last = min(use.tiles, use.tile + count - done);
    const int rows = min(16, g.per - row0);
    const bool whole = first == 0 && last == use.tiles, opening = done == 0;

    uint32_t qb[NT][kWordsK][4];                            // fp16 pairs of d = 32 b + 8 qd + 0 .. 7 of row gq
    // Of rows 2 qd and 2 qd + 1: sums per group, what the operands' offsets add to a score (the odd pairs of K are
    // 1032 + 16 c, and their q is divided by 16: 72.5 more than c - 8), scale.
    float qsum[NT][2][NG], qoff[NT][2][NG], sl[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = t * 8 + gq;
      const uint16_t *q = g.a + slot * g.a_row + int64_t(head * g.per + row0 + r) * g.a_head + qd * 8;
      float s[NG], back = g.sl;
#pragma unroll
      for (int i = 0; i < NG; ++i) s[i] = 0.f;
#pragma unroll
      for (int b = 0; b < kWordsK; ++b) {
        const uint4 w = r < rows ? *reinterpret_cast<const uint4 *>(q + b * 32) : make_uint4(0, 0, 0, 0);
        qb[t][b][0] = w.x, qb[t][b][1] = w.y, qb[t][b][2] = w.z, qb[t][b][3] = w.w;
      }
      // To fp16, the row's largest value brought to its power of two, fp16 rows to 2^4 (bf16 keys may be 2^112 times larger, and their
      // products are fp32): bf16's 8 bits fit fp16's 11, and fp16 keeps its own (small rows too, of which a sixteenth would be
      // subnormal); values 2^-14 of that and less keep 2^-25 of it, a sixteenth of them 2^-21.  A row of zeros, or with an infinity
      // or a NaN, is converted as it is.
      constexpr int kTop = F16 ? 4 : 0;
      uint32_t most = 0;
#pragma unroll
      for (int b = 0; b < kWordsK; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = __vmaxu2(most, qb[t][b][i] & 0x7fff7fffu);
      most = max(most & 0xffffu, most >> 16);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int top = int(__float_as_uint(to_f32<F16>(most)) >> 23), e = top == 0 || top == 255 ? kTop : min(top - 127, 126);
      const float down = __uint_as_float(uint32_t(127 + kTop - e) << 23);
      back = g.sl / down;
#pragma unroll
      for (int b = 0; b < kWordsK; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) qb[t][b][i] = pack_16x2<true>(lo_f32<F16>(qb[t][b][i]) * down, hi_f32<F16>(qb[t][b][i]) * down);
      float odd[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) odd[i] = 0.f;
#pragma unroll
      for (int b = 0; b < kWordsK; ++b) {
        s[b * 32 / kGroup] += lo_f32<true>(qb[t][b][0]) + hi_f32<true>(qb[t][b][0]) + lo_f32<true>(qb[t][b][2]) + hi_f32<true>(qb[t][b][2]);
#pragma unroll
        for (int i = 1; i < 4; i += 2) {                    // the sixteenth is what the products see, its rounding included
          const float x0 = lo_f32<true>(qb[t][b][i]) * 0.0625f, x1 = hi_f32<true>(qb[t][b][i]) * 0.0625f;
          qb[t][b][i] = pack_16x2<true>(x0, x1);
          odd[b * 32 / kGroup] += lo_f32<true>(qb[t][b][i]) + hi_f32<true>(qb[t][b][i]);
        }
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        odd[i] += __shfl_xor_sync(0xffffffffu, odd[i], 1);
        odd[i] += __shfl_xor_sync(0xffffffffu, odd[i], 2);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
        s[i] = fmaf(16.f, odd[i], s[i]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          qsum[t][k][i] = __shfl_sync(0xffffffffu, s[i], 8 * qd + 4 * k);
          qoff[t][k][i] = -1160.f * __shfl_sync(0xffffffffu, odd[i], 8 * qd + 4 * k);
        }
      }
      sl[t][0] = __shfl_sync(0xffffffffu, back, 8 * qd);
      sl[t][1] = __shfl_sync(0xffffffffu, back, 8 * qd + 4);
    }
    // nm: the rows' references (log2), negated, 0 before the first score; room: the unscaled score that moves it, -inf before the first.
    float nm[NT][2], room[NT][2], l[NT][2], corr[NT][2][NG], o[NT][D / 16][4];
    float vdown = 1.f;                                      // power of two on the V scales
    uint32_t vroom = 0;                                     // largest V scale (bits) it allows, 0 before the first
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        nm[t][i] = l[t][i] = 0.f;
        room[t][i] = -INFINITY;
#pragma unroll
        for (int k = 0; k < NG; ++k) corr[t][i][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    }

    for (int tile = first; tile < last; ++tile) {
      // The outcome is made the warp's: one lane must not leave a loop that others vote in.
      if (!(ok = __all_sync(0xffffffffu, sm100::mbar_wait(&full[st], phase, wl)))) break;
      const int there = good[st];
#pragma unroll 1
      for (int pass = 0; pass < kKvTile / kKvPass; ++pass) {
      const uint8_t *buf = ring + st * kStage + pass * (kKvPass * (D + 8 * NG));
      // Keys past the length, or whose page is not there, take no part: score -inf and parameters 0.
      const int left = len - tile * kKvTile - pass * kKvPass;
      if (left <= 0) break;
      const bool partial = left < kKvPass || there != (1 << parts) - 1;
      float z[2][NT][4];                                    // [step][row block][key gq: rows 2 qd, + 1; key gq + 8: the same]
      uint32_t vp[2][2][NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t *kc = buf + h * step_k + gq * (D / 2) + qd * (D / 8);
        __align__(16) uint32_t wa[kWordsK], wb[kWordsK];
        uint32_t kp[2][NG];
        if (D == 128) {
          *reinterpret_cast<uint4 *>(wa) = *reinterpret_cast<const uint4 *>(kc);
          *reinterpret_cast<uint4 *>(wb) = *reinterpret_cast<const uint4 *>(kc + 8 * (D / 2));
        } else {
          *reinterpret_cast<uint2 *>(wa) = *reinterpret_cast<const uint2 *>(kc);
          *reinterpret_cast<uint2 *>(wb) = *reinterpret_cast<const uint2 *>(kc + 8 * (D / 2));
        }
        const uint32_t *kpar = reinterpret_cast<const uint32_t *>(buf + kp_at + h * step_p);
        const uint32_t *vpar = reinterpret_cast<const uint32_t *>(buf + vp_at + h * step_p);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          kp[0][i] = kpar[i], kp[1][i] = kpar[8 * NG + i];
          vp[h][0][i] = vpar[i], vp[h][1][i] = vpar[8 * NG + i];
        }
        float acc[NT][NG][4];
#pragma unroll
        for (int b = 0; b < kWordsK; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {                     // bytes 0 and 2: d = 0, 1 | 2, 3; bytes 1 and 3: 4, 5 | 6, 7
            uint32_t a[4];
            split_offset(__byte_perm(wa[b], 0x64646464u, e ? 0x4341 : 0x4240), a[0], a[2]);
            split_offset(__byte_perm(wb[b], 0x64646464u, e ? 0x4341 : 0x4240), a[1], a[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if (e == 0 && b * 32 % kGroup == 0) mma_16n8_first(acc[t][b * 32 / kGroup], a, qb[t][b][0], qb[t][b][1], qoff[t][0][b * 32 / kGroup],
                                                                          qoff[t][1][b * 32 / kGroup]);
              else mma_16n8_f16(acc[t][b * 32 / kGroup], a, qb[t][b][2 * e], qb[t][b][2 * e + 1]);
            }
          }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float a[NG], mid[NG];
#pragma unroll
          for (int i = 0; i < NG; ++i) a[i] = lo_f32<F16>(kp[k][i]), mid[i] = fmaf(8.f, a[i], hi_f32<F16>(kp[k][i]));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float2 s2 = __fmul2_rn(make_float2(mid[0], mid[0]), make_float2(qsum[t][0][0], qsum[t][1][0]));
#pragma unroll
            for (int n = 1; n < NG; ++n) s2 = __ffma2_rn(make_float2(mid[n], mid[n]), make_float2(qsum[t][0][n], qsum[t][1][n]), s2);
#pragma unroll
            for (int n = 0; n < NG; ++n) s2 = __ffma2_rn(make_float2(a[n], a[n]), make_float2(acc[t][n][2 * k], acc[t][n][2 * k + 1]), s2);
            z[h][t][2 * k] = s2.x, z[h][t][2 * k + 1] = s2.y;
          }
        }
        if (partial) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int key = h * 16 + k * 8 + gq;
            if (key < left && ((there >> ((pass * kKvPass + h * 16) >> part_log)) & 1)) continue;
#pragma unroll
            for (int t = 0; t < NT; ++t) z[h][t][2 * k] = z[h][t][2 * k + 1] = -INFINITY;
#pragma unroll
            for (int i = 0; i < NG; ++i) vp[h][k][i] = 0;
          }
        }
      }
      // A row's reference moves only when a score passes it by kKvGrow (the first key's always does).
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          grow |= fmaxf(fmaxf(z[0][t][i], z[0][t][i + 2]), fmaxf(z[1][t][i], z[1][t][i + 2])) > room[t][i];
      uint32_t vtop = vp[0][0][0];
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) vtop = __vmaxu2(vtop, vp[k >> 1][k & 1][i]);
      grow |= (vtop & 0xffffu) > vroom;
      if (__any_sync(0xffffffffu, grow)) {
        float f = 1.f;                                      // the V scales' power of two moves down
        uint32_t top = 0;                                   // the largest finite scale
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a = vp[k >> 1][k & 1][i] & 0xffffu;
            if (a < (F16 ? 0x7c00u : 0x7f80u)) top = max(top, a);
          }
        top = __reduce_max_sync(0xffffffffu, top);
        if (top > vroom) {
          const int e = max(int(__float_as_uint(to_f32<F16>(top)) >> 23) - 126, kKvTop - 126);   // 2^e > the scale, at most 2^128
          const float now = __uint_as_float(uint32_t(127 + kKvTop - e) << 23);
          f = vroom == 0 ? 1.f : now / vdown;
          vdown = now;
          vroom = !F16 ? uint32_t(e + 127) << 7 : e < -14 ? 1u << (e + 24) : uint32_t(e + 15) << 10;   // 2^e in the cache's type
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(fmaxf(z[0][t][i], z[0][t][i + 2]), fmaxf(z[1][t][i], z[1][t][i + 2]));
#pragma unroll
            for (int s = 4; s < 32; s *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
            const float to = top * sl[t][i];
            float alpha = 1.f;
            if (top > room[t][i] || (room[t][i] != -INFINITY && to > -nm[t][i])) {
              if (room[t][i] != -INFINITY) alpha = ex2_fast(-nm[t][i] - to);    // the first score: nothing to rescale
              nm[t][i] = -to;
              room[t][i] = top + float(kKvGrow) / sl[t][i];
            }
            l[t][i] *= alpha;
#pragma unroll
            for (int k = 0; k < NG; ++k) corr[t][i][k] *= alpha;
            alpha *= f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) o[t][k][i] *= alpha, o[t][k][i + 2] *= alpha;
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // Weights times the V scales, rounded: per group the operand [16 keys x 8 rows], transposed from the scores' layout.
        uint32_t pb[NT][NG][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float a[NG], mid[NG];
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            a[i] = lo_f32<F16>(vp[h][k][i]), mid[i] = fmaf(8.f, a[i], hi_f32<F16>(vp[h][k][i]));
            a[i] *= vdown;
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float2 p = __ffma2_rn(make_float2(z[h][t][2 * k], z[h][t][2 * k + 1]), make_float2(sl[t][0], sl[t][1]),
                                  make_float2(nm[t][0], nm[t][1]));
            p.x = ex2_fast(p.x), p.y = ex2_fast(p.y);
            const float2 sum = __fadd2_rn(make_float2(l[t][0], l[t][1]), p);
            l[t][0] = sum.x, l[t][1] = sum.y;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
              const float2 c = __ffma2_rn(p, make_float2(mid[i], mid[i]), make_float2(corr[t][0][i], corr[t][1][i]));
              corr[t][0][i] = c.x, corr[t][1][i] = c.y;
              const float2 w = __fmul2_rn(p, make_float2(a[i], a[i]));
              pb[t][i][k] = transpose_8x8(pack_16x2<true>(w.x, w.y));
            }
          }
        }
        const uint8_t *vc = buf + v_at + h * step_k;            // keys 2 qd, 2 qd + 1, 2 qd + 8, 2 qd + 9: rows qd, + 4, + 8, + 12
        __align__(8) uint32_t w[4][kWordsV];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (D == 128) *reinterpret_cast<uint2 *>(w[r]) = *reinterpret_cast<const uint2 *>(vc + r * 4 * (D / 2));
          else w[r][0] = *reinterpret_cast<const uint32_t *>(vc + r * 4 * (D / 2));
        }
#pragma unroll
        for (int v = 0; v < kWordsV; ++v)
#pragma unroll
          for (int half = 0; half < 2; ++half) {                // bytes 0, 1: d = 64 v + 4 gq ..; bytes 2, 3: 32 further
            const uint32_t lo = __byte_perm(w[0][v], w[1][v], half ? 0x7362 : 0x5140);   // the two keys' bytes, alternating
            const uint32_t hi = __byte_perm(w[2][v], w[3][v], half ? 0x7362 : 0x5140);
            const int gr = (v * 64 + half * 32) / kGroup;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t a[4];
              split_codes(__byte_perm(lo, 0x64646464u, e ? 0x4342 : 0x4140), a[0], a[1]);
              split_codes(__byte_perm(hi, 0x64646464u, e ? 0x4342 : 0x4140), a[2], a[3]);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_16n8_f16(o[t][v * 4 + half * 2 + e], a, pb[t][gr][0], pb[t][gr][1]);
            }
          }
      }
      }
      __syncwarp();                                           // every lane has read the stage: it may be filled again
      feed();
      ++done;
      st = st + 1 == kKvStages ? 0 : st + 1;
      phase ^= st == 0 ? 1 : 0;
    }
    if (!ok) break;

    // The part's rows: sums over the lanes of a row, then o or the workspace.  Rows 2 qd (+ 1), d = 64 v + 32 half + 4 gq + 0 .. 3.
    const int64_t slot_at = 2 * int64_t(worker) + (opening ? 0 : 1);
    const float up = 1.f / vdown;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = t * 8 + 2 * qd + i;
#pragma unroll
        for (int s = 4; s < 32; s *= 2) {
          l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], s);
#pragma unroll
          for (int k = 0; k < NG; ++k) corr[t][i][k] += __shfl_xor_sync(0xffffffffu, corr[t][i][k], s);
        }
        if (r >= rows) continue;
        const bool none = room[t][i] == -INFINITY && l[t][i] == 0.f;   // no key was there (its pages were not): zeros
        const float inv = !whole ? 1.f : none ? 0.f : 1.f / l[t][i];
        float *part = g.part_o + (slot_at * 16 + r) * D;
        uint16_t *out = g.b + slot * g.b_row + int64_t(head * g.per + row0 + r) * g.b_head;
#pragma unroll
        for (int v = 0; v < kWordsV; ++v)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int d = v * 64 + half * 32 + gq * 4, k = v * 4 + half * 2;
            const float c = corr[t][i][(v * 64 + half * 32) / kGroup];
            const float y0 = fmaf(o[t][k][i], up, c) * inv, y1 = fmaf(o[t][k][i + 2], up, c) * inv;
            const float y2 = fmaf(o[t][k + 1][i], up, c) * inv, y3 = fmaf(o[t][k + 1][i + 2], up, c) * inv;
            if (whole) *reinterpret_cast<uint2 *>(out + d) = make_uint2(pack_16x2<F16>(y0, y1), pack_16x2<F16>(y2, y3));
            else *reinterpret_cast<float4 *>(part + d) = make_float4(y0, y1, y2, y3);
          }
        if (!whole && gq == 0)
          *reinterpret_cast<float2 *>(g.part_ml + (slot_at * 16 + r) * 2) = make_float2(room[t][i] == -INFINITY ? -INFINITY : -nm[t][i], l[t][i]);
      }
    use.tile = last;
    if (last == use.tiles && done < count) next_item(use);
  }
  // After a wait that gave up, the copies in flight land (bounded) before the warp leaves its ring.
  if (!ok)
    for (int i = done; i < filled; ++i) {
      sm100::mbar_wait(&full[st], phase, wl);
      st = st + 1 == kKvStages ? 0 : st + 1;
      phase ^= st == 0 ? 1 : 0;
    }
}

// Merges the parts of an item that several workers hold, in key order; zeros for an empty slot.  grid (slots x items, row
// blocks of 128 / D rows), D / 4 lanes of four columns a row.  Each of the four warps goes over a quarter of the parts, D / 4 at a
// time: lane j fetches part j's (m, l) of the row, the maximum and the weights are shuffles, and the columns' loads of eight
// parts are in flight together; the quarters meet in shared memory.  (A thread per column that walked the parts one by one, two
// dependent loads a part, made 116 us of a call that now takes 19: 33 slots, 16 rows a KV head, about 40 parts an item.)
template <int D, bool F16>
__global__ void __launch_bounds__(128) kv4_merge_kernel(const __grid_constant__ Kv4Args g) {
  constexpr int kLanes = D / 4, kRows = 32 / kLanes;
  const int items = g.hkv * g.rb, slot = int(blockIdx.x) / items, item = int(blockIdx.x) % items;
  const int lane = threadIdx.x & 31, sub = lane / kLanes, col = lane % kLanes;
  const int head = item / g.rb, row0 = (item % g.rb) * 16;
  const int warp = threadIdx.x >> 5, r = int(blockIdx.y) * kRows + sub;
  __shared__ float4 quarter[3][32];
  __shared__ float2 quarter_ml[3][32];
  const bool live = r < min(16, g.per - row0);
  pdl_enter();
  const int before = g.before[slot], units = g.before[slot + 1] - before;
  const uint32_t share = kv4_share(uint32_t(g.before[g.slots]) * uint32_t(items), g.workers);
  const uint32_t u0 = uint32_t(before) * uint32_t(items) + uint32_t(item) * uint32_t(units);
  int64_t w0 = 0;
  int parts = 0, first = 0;                                    // first: the part of worker w0 is its last, not its opening one
  if (units > 0) {
    w0 = (u0 + kKvItemCost) / share;
    parts = int((u0 + units - 1) / share - w0) + 1;
    if (parts == 1) return;                                    // one worker held the whole item and wrote it
    first = uint32_t(w0) * share < u0 ? 1 : 0;
  }
  float top = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  const int rr = live ? r : 0;
  const int j_lo = parts * warp / 4, j_hi = parts * (warp + 1) / 4;
  for (int j0 = j_lo; j0 < j_hi; j0 += kLanes) {
    const int j = j0 + col;
    float m = -INFINITY, l = 0.f;
    if (j < j_hi) {
      const float2 ml = *reinterpret_cast<const float2 *>(g.part_ml + ((2 * (w0 + j) + (j == 0 ? first : 0)) * 16 + rr) * 2);
      m = ml.x, l = ml.y;
    }
    float now = m;
#pragma unroll
    for (int s = 1; s < kLanes; s *= 2) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, s));
    now = fmaxf(now, top);
    const float back = now == top ? 1.f : ex2_fast(top - now);
    float e = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2_fast(m - now);   // l of a part without a maximum: 0, or NaN to pass on
    float part = l * e;
#pragma unroll
    for (int s = 1; s < kLanes; s *= 2) part += __shfl_xor_sync(0xffffffffu, part, s);
    L = L * back + part;
    O.x *= back, O.y *= back, O.z *= back, O.w *= back;
    top = now;
    const int here = min(kLanes, j_hi - j0);
#pragma unroll 8
    for (int k = 0; k < here; ++k) {
      const float w = __shfl_sync(0xffffffffu, e, k, kLanes);
      const int64_t at = ((2 * (w0 + j0 + k) + (j0 + k == 0 ? first : 0)) * 16 + rr) * D + 4 * col;
      const float4 o = *reinterpret_cast<const float4 *>(g.part_o + at);
      O.x = fmaf(o.x, w, O.x), O.y = fmaf(o.y, w, O.y), O.z = fmaf(o.z, w, O.z), O.w = fmaf(o.w, w, O.w);
    }
  }
  if (warp > 0) quarter[warp - 1][lane] = O, quarter_ml[warp - 1][lane] = make_float2(top, L);
  __syncthreads();
  if (warp > 0 || !live) return;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float4 o = quarter[k][lane];
    const float2 ml = quarter_ml[k][lane];
    const float now = fmaxf(top, ml.x);
    const float a = now == top ? 1.f : ex2_fast(top - now), b = now == ml.x ? 1.f : ex2_fast(ml.x - now);   // equal: both may be -inf
    L = L * a + ml.y * b;
    O.x = O.x * a + o.x * b, O.y = O.y * a + o.y * b, O.z = O.z * a + o.z * b, O.w = O.w * a + o.w * b;
    top = now;
  }
  const float inv = top == -INFINITY && L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2 *>(g.b + slot * g.b_row + int64_t(head * g.per + row0 + r) * g.b_head + 4 * col) =
      make_uint2(pack_16x2<F16>(O.x * inv, O.y * inv), pack_16x2<F16>(O.z * inv, O.w * inv));
}

// Shared memory of a CTA of the attention: the warps' rings with their barriers and flags, the scan's sums, 6 bytes a slot.
constexpr int kv4_smem(int dim, int group, int slots) {
  return kKvWarps * kKvStages * (kKvTile * (dim + 8 * (dim / group)) + 12) + 8 * kKvWarps + 16 + 6 * (slots + 1);
}

// Workers of the attention: one warp each, as many as are resident at once.  By registers three CTAs an SM (168 a thread), two where
// 16 query heads or four groups of a head dimension take more (64 slots of up to 8191 keys, groups of 32 at D 128: 83 us with two CTAs
// and 213 registers, 116 with three and spills); by the SM's 228 KB, of which a CTA takes 1 KB and up to 128 bytes beside its own, two
// from 466 slots on at D 128 in groups of 64 (1024 slots of up to 1000 keys: 184 us, 235 when cut for three).
static int kv4_workers(const ptsim_kv4_params &p, int sm_count) {
  const int by_registers = p.hq / p.hkv <= 8 && p.dim / p.group < 4 ? 3 : 2;
  const int by_memory = (228 << 10) / (kv4_smem(int(p.dim), int(p.group), int(p.slots)) + 1152);
  return sm_count * (by_memory < by_registers ? by_memory : by_registers) * kKvWarps;
}

int64_t kv4_workspace(const ptsim_desc &d, int sm_count) {
  const ptsim_kv4_params &p = d.p.kv4;
  return (2 * int64_t(kv4_workers(p, sm_count)) * 16 * (p.dim + 2) + p.slots + 1) * int64_t(sizeof(float));
}

template <int D, int NG, int NT, bool F16>
static int run_kv4_attn(const Kv4Args &g, const LaunchCtx &c) {
  constexpr auto kern = kv4_attn_kernel<D, NG, NT, F16>;
  PTSIM_CUDA((smem_limit_once<kern>(kv4_smem(D, D / NG, PTSIM_KV4_SLOTS), c.device)));
  PTSIM_CUDA(launch_pdl(kern, dim3(unsigned(g.workers / kKvWarps)), dim3(kKvWarps * 32), kv4_smem(D, D / NG, g.slots), c.stream, g));
  const int rows = g.per < 16 ? g.per : 16;
  PTSIM_CUDA(launch_pdl(kv4_merge_kernel<D, F16>, dim3(unsigned(g.slots * g.hkv * g.rb), unsigned(ceil_div(rows * D, 128))), dim3(128), 0,
                        c.stream, g));
  return PTSIM_OK;
}

template <int D, int NG, bool F16>
static int run_kv4(const ptsim_desc &d, Kv4Args &g, uint8_t *pool, const LaunchCtx &c) {
  if (d.kind == PTSIM_KIND_ATTN_KV4)
    return d.p.kv4.hq / d.p.kv4.hkv <= 8 ? run_kv4_attn<D, NG, 1, F16>(g, c) : run_kv4_attn<D, NG, 2, F16>(g, c);
  // A warp takes eight steps of heads where that leaves every SM 12 warps or more, else one, so that few tokens spread: 600 tokens of
  // 8 heads of 128 are stored and loaded in 11 us with one step and 13 with eight, 1200 in 15 with either, 4500 in 28 and 22.
  constexpr int kHeads = 128 / D;
  const int64_t eight = g.tokens * ceil_div(g.hkv, 8 * kHeads), one = g.tokens * ceil_div(g.hkv, kHeads);
  const bool many = eight >= int64_t(c.sm_count) * 12 && one > eight;
  const dim3 grid(unsigned(ceil_div(g.tokens, 8)), unsigned(ceil_div(g.hkv, many ? 8 * kHeads : kHeads)));
  if (d.kind == PTSIM_KIND_KV4_STORE)
    PTSIM_CUDA(launch_pdl(many ? kv4_store_kernel<D, NG, F16, 8> : kv4_store_kernel<D, NG, F16, 1>, grid, dim3(256), 0, c.stream, g, pool));
  else
    PTSIM_CUDA(launch_pdl(many ? kv4_load_kernel<D, NG, F16, 8> : kv4_load_kernel<D, NG, F16, 1>, grid, dim3(256), 0, c.stream, g));
  return PTSIM_OK;
}

int launch_kv4(const ptsim_desc &d, void *const *ptrs, void *ws, size_t ws_bytes, const LaunchCtx &c) {
  const ptsim_kv4_params &p = d.p.kv4;
  const bool attn = d.kind == PTSIM_KIND_ATTN_KV4;
  if (p.slots == 0 || (!attn && p.tokens == 0)) return PTSIM_OK;
  Kv4Args g;
  memset(&g, 0, sizeof(g));
  g.record = p.page_size * (p.dim + 8 * (p.dim / p.group));
  uint8_t *pool = static_cast<uint8_t *>(ptrs[p.pool_arg]) + p.layer * p.pages * p.hkv * g.record;
  g.pool = pool;
  g.lens = static_cast<const int32_t *>(ptrs[p.lens_arg]);
  g.table = static_cast<const int32_t *>(ptrs[p.table_arg]);
  g.cu = attn ? nullptr : static_cast<const int32_t *>(ptrs[p.cu_arg]);
  g.halt = p.halt_arg_p1 == 0 ? nullptr : static_cast<const int32_t *>(ptrs[p.halt_arg_p1 - 1]);
  g.a = static_cast<uint16_t *>(ptrs[p.a_arg]) + p.a_off;
  g.b = static_cast<uint16_t *>(ptrs[p.b_arg]) + p.b_off;
  for (const void *q : {static_cast<const void *>(pool), static_cast<const void *>(g.a), static_cast<const void *>(g.b)})
    if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return fail(PTSIM_E_ARGS, "a tensor of the 4-bit cache is not 16-byte aligned");
  g.a_row = p.a_row, g.a_head = p.a_head, g.b_row = p.b_row, g.b_head = p.b_head;
  g.tokens = int(p.tokens);
  g.slots = int(p.slots);
  g.hkv = int(p.hkv);
  g.pages = int(p.pages);
  g.page_size = int(p.page_size);
  g.page_log = p.page_size == 16 ? 4 : p.page_size == 32 ? 5 : p.page_size == 64 ? 6 : 7;
  g.max_pages = int(p.max_pages);
  g.stall = (d.flags & PTSIM_FLAG_TEST_STALL) ? 1 : 0;
  if (attn) {
    g.per = int(p.hq / p.hkv);
    g.rb = int(ceil_div(g.per, 16));
    g.sl = p.scale * 1.4426950408889634f;
    g.workers = kv4_workers(p, c.sm_count);
    const int64_t need = kv4_workspace(d, c.sm_count);
    if (ws == nullptr || int64_t(ws_bytes) < need)
      return fail(PTSIM_E_RESOURCE, "4-bit cache attention needs %lld bytes of workspace, got %zu", (long long)need, ws_bytes);
    if (reinterpret_cast<uintptr_t>(ws) % 16 != 0) return fail(PTSIM_E_ARGS, "workspace is not 16-byte aligned");
    g.part_o = static_cast<float *>(ws);
    g.part_ml = g.part_o + 2 * int64_t(g.workers) * 16 * p.dim;
    g.before = reinterpret_cast<int32_t *>(g.part_ml + 2 * int64_t(g.workers) * 16 * 2);
  }
  const bool f16 = d.arg_dtype[p.a_arg] == PTSIM_DT_F16;
  switch (p.dim / p.group + (p.dim == 128 ? 10 : 0) + (f16 ? 100 : 0)) {
    case 1: return run_kv4<64, 1, false>(d, g, pool, c);
    case 2: return run_kv4<64, 2, false>(d, g, pool, c);
    case 11: return run_kv4<128, 1, false>(d, g, pool, c);
    case 12: return run_kv4<128, 2, false>(d, g, pool, c);
    case 14: return run_kv4<128, 4, false>(d, g, pool, c);
    case 101: return run_kv4<64, 1, true>(d, g, pool, c);
    case 102: return run_kv4<64, 2, true>(d, g, pool, c);
    case 111: return run_kv4<128, 1, true>(d, g, pool, c);
    case 112: return run_kv4<128, 2, true>(d, g, pool, c);
    case 114: return run_kv4<128, 4, true>(d, g, pool, c);
  }
  return fail(PTSIM_E_UNSUPPORTED, "a 4-bit cache of head dim %lld in groups of %lld", (long long)p.dim, (long long)p.group);
}

}  // namespace ptsim
