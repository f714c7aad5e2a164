// The 4-bit paged cache of keys and values (format: include/ptsim_b200.h, ptsim_kv4_params): store, load and the attention
// of one new token per slot.  No counterpart in the reference, whose decode program reads a dense bf16 cache (decode.cuh).
//
// Attention.  With codes c, scale a and minimum b per (key, group of the head dimension), the cached key is k = a c + b and
// the score z = sum_g a_g (q . c)_g + b_g sum(q)_g: the tensor core multiplies q by the small integers c, exact in 16 bits, and
// the parameters enter in fp32, once per (key, group).  Likewise O = sum_k (p a_g) (c - 8) + p (b_g + 8 a_g), with p a_g
// rounded to 16 bits as the product's operand (the rounding of P that decode.cuh makes, here of what multiplies |c - 8| <= 8)
// and the second sum kept per row in fp32.  A nibble becomes a 16-bit float by one mask-and-or, bf16 0x4300 | c = 128 + c and
// fp16 0x5400 | c << 4 = 64 + c.  For K the offset's share of a score, 128 sum(q), is taken off in the accumulator's start.
// For V it is subtracted from the operand: accumulated over 10^5 keys, an offset of 128 costs the sums their low bits
// (the tensor core truncates; measured 2.4e-2 of the result at 131072 keys against 1.7e-3 with c - 8).
//
// The products have K and V as the 16-row operand: S^T = K q^T, O^T = V^T P^T (mma.sync m16n8k16, N = 8 query rows of one KV
// head), so up to 8 query heads per KV head waste nothing, half of what a 16-row query tile costs; tcgen05.mma, whose
// smallest M is 64 and whose operands come from shared memory as 16 bits, would need the unpacked tile written back.  Both operands
// take their k index in any order both sides agree on, which the page format uses: 16-byte (K) and 8-byte (V) shared loads
// without bank conflicts give words whose nibbles are the fragments.
//
// Bound: HBM, (D + 8 D / group) bytes per key and KV head (144 at D 128, group 64: 3.5 times fewer than bf16), and close
// behind it the issue slots of the unpacking (about 250 warp instructions per 16 keys).  Work is one list of 32-key tiles over
// (slot, KV head), cut into equal contiguous ranges, one per warp: a warp streams its tiles by bulk copies through a ring of its
// own (no barrier between warps) and keeps the online softmax in registers.  Lengths are read on the device, so any
// raggedness is balanced to a tile.  A range that holds only part of an item leaves (m, l, O) in the workspace and a second
// kernel (a programmatic dependent) merges the parts in key order: results do not depend on timing.
#pragma once
#include "sm100.cuh"
#include "decode.cuh"
#include "packed.cuh"

namespace ptsim {

constexpr int kKvTile = 32;          // keys of a tile
constexpr int kKvStages = 3;
constexpr int kKvWarps = 4;

struct Kv4Args {
  const uint8_t *pool;               // of the launch's layer
  const int32_t *lens, *table, *cu;
  uint16_t *a, *b;                   // K and V, or q and o
  int64_t a_row, a_head, b_row, b_head;
  int64_t record;                    // bytes of one (page, KV head)
  int32_t tokens, slots, hkv, per, rb;   // per: query heads of a KV head; rb: blocks of 16 of them
  int32_t pages, page_size, max_pages;
  float sl;                          // scale * log2 e
  float *part_o, *part_ml;           // [2 * workers][16][D] and [2 * workers][16][2]
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
  if (pos >= 0 && pos / g.page_size < g.max_pages) page = g.table[int64_t(s) * g.max_pages + pos / g.page_size];
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
  __device__ __forceinline__ void place(int at, int page_size, int *code, int *par) const {
    const int bs = page_size < 32 ? page_size : 32;
    const int base = (at / bs) * (bs * (D + 8 * NG)), t = at % bs;
    const int r = is_v ? (t & ~7) | ((t & 1) << 2) | ((t >> 1) & 3) : t;
    const int w = is_v && D == 128 && (r & 2) ? word ^ 8 : word;
    *code = base + (is_v ? bs * (D / 2) : 0) + r * (D / 2) + w * 4;
    *par = base + bs * D + (is_v ? bs * 4 * NG : 0) + t * 4 * NG;
  }
};

// One (token, head) per D/4 lanes: eight values a lane, their group's minimum and maximum by shuffles.
template <int D, int NG, bool F16>
__global__ void __launch_bounds__(256) kv4_store_kernel(const __grid_constant__ Kv4Args g, uint8_t *pool) {
  constexpr int kLanes = D / 4, kHeads = 32 / kLanes;   // heads a warp takes at once
  const int lane = threadIdx.x & 31;
  const int hsteps = (g.hkv + kHeads - 1) / kHeads;
  const int64_t unit = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int t = int(unit / hsteps), h = int(unit % hsteps) * kHeads + lane / kLanes;
  pdl_enter();
  if (t >= g.tokens) return;
  const Kv4Lane<D, NG> me(lane);
  const bool live = h < g.hkv;
  uint2 x0 = make_uint2(0, 0), x1 = x0;
  if (live) {
    const uint16_t *src = me.is_v ? g.b + t * g.b_row + h * g.b_head : g.a + t * g.a_row + h * g.a_head;
    x0 = *reinterpret_cast<const uint2 *>(src + me.d0);
    x1 = *reinterpret_cast<const uint2 *>(src + me.d1);
  }
  int64_t pos = 0;
  const int slot = kv4_find(g, t, lane, &pos);
  if (slot < 0) return;
  const int page = kv4_page(g, slot, pos, lane);
  if (page < 0) return;
  const float x[8] = {lo_f32<F16>(x0.x), hi_f32<F16>(x0.x), lo_f32<F16>(x0.y), hi_f32<F16>(x0.y),
                      lo_f32<F16>(x1.x), hi_f32<F16>(x1.x), lo_f32<F16>(x1.y), hi_f32<F16>(x1.y)};
  // Extremes of the lane's two runs of four; one group but for V in groups of 32.
  float mn[2], mx[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mn[r] = nan_min(nan_min(x[4 * r], x[4 * r + 1]), nan_min(x[4 * r + 2], x[4 * r + 3]));
    mx[r] = nan_max(nan_max(x[4 * r], x[4 * r + 1]), nan_max(x[4 * r + 2], x[4 * r + 3]));
  }
  constexpr int kGroup = D / NG;
  if (kGroup > 32 || !me.is_v) {
    mn[0] = mn[1] = nan_min(mn[0], mn[1]);
    mx[0] = mx[1] = nan_max(mx[0], mx[1]);
  }
  // Lanes of a group: group / 8 consecutive ones (V in groups of 32: all eight of its 64 values' lanes, by run).
#pragma unroll
  for (int s = 1; s < (kGroup > 64 ? 16 : 8); s *= 2)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float a = nan_min(mn[r], __shfl_xor_sync(0xffffffffu, mn[r], s));
      const float b = nan_max(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], s));
      if (kGroup > 32 || s < 4 || me.is_v) mn[r] = a, mx[r] = b;
    }
  uint32_t word = 0, par[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float half = mx[r] * 0.5f - mn[r] * 0.5f;           // halves: the range itself could overflow
    const bool fine = half < INFINITY;                        // false for NaN too
    const uint32_t s16 = pack_16x2<F16>(__fdiv_rn(half, 7.5f), mn[r]);   // (scale, minimum); the minimum is exact
    const float step = lo_f32<F16>(s16);
    par[r] = fine ? s16 : (F16 ? 0x7e007e00u : 0x7fc07fc0u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = rintf(__fdiv_rn(x[4 * r + e] - mn[r], step));
      const uint32_t code = fine && step > 0.f ? uint32_t(fminf(fmaxf(q, 0.f), 15.f)) : 0u;
      const int d = 4 * r + e;                                // K: nibble (d / 2) + 4 (d % 2); V: run r, place e
      word |= code << (4 * (me.is_v ? d : (d >> 1) + 4 * (d & 1)));
    }
  }
  if (!live) return;
  int code_at, par_at;
  me.place(int(pos % g.page_size), g.page_size, &code_at, &par_at);
  uint8_t *rec = pool + (int64_t(page) * g.hkv + h) * g.record;
  *reinterpret_cast<uint32_t *>(rec + code_at) = word;
  // The first lane of each group writes its parameters.
  if (me.d0 % kGroup == 0) *reinterpret_cast<uint32_t *>(rec + par_at + 4 * (me.d0 / kGroup)) = par[0];
  if (kGroup == 32 && me.is_v && (me.i & 7) == 0) *reinterpret_cast<uint32_t *>(rec + par_at + 4 * (me.d1 / kGroup)) = par[1];
}

template <int D, int NG, bool F16>
__global__ void __launch_bounds__(256) kv4_load_kernel(const __grid_constant__ Kv4Args g) {
  constexpr int kLanes = D / 4, kHeads = 32 / kLanes, kGroup = D / NG;
  const int lane = threadIdx.x & 31;
  const int hsteps = (g.hkv + kHeads - 1) / kHeads;
  const int64_t unit = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int t = int(unit / hsteps), h = int(unit % hsteps) * kHeads + lane / kLanes;
  pdl_enter();
  if (t >= g.tokens) return;
  int64_t pos = 0;
  const int slot = kv4_find(g, t, lane, &pos);
  if (slot < 0 || h >= g.hkv) return;
  const int page = kv4_page(g, slot, pos, lane);
  const Kv4Lane<D, NG> me(lane);
  uint32_t word = 0, p0 = 0, p1 = 0;                          // a page outside the pool reads as zeros
  if (page >= 0) {
    int code_at, par_at;
    me.place(int(pos % g.page_size), g.page_size, &code_at, &par_at);
    const uint8_t *rec = g.pool + (int64_t(page) * g.hkv + h) * g.record;
    word = *reinterpret_cast<const uint32_t *>(rec + code_at);
    p0 = *reinterpret_cast<const uint32_t *>(rec + par_at + 4 * (me.d0 / kGroup));
    p1 = *reinterpret_cast<const uint32_t *>(rec + par_at + 4 * (me.d1 / kGroup));
  }
  uint32_t out[4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float s = lo_f32<F16>(r ? p1 : p0), mn = hi_f32<F16>(r ? p1 : p0);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 4 * r + e;
      y[e] = __fmaf_rn(s, float((word >> (4 * (me.is_v ? d : (d >> 1) + 4 * (d & 1)))) & 15u), mn);
    }
    out[2 * r] = pack_16x2<F16>(y[0], y[1]);
    out[2 * r + 1] = pack_16x2<F16>(y[2], y[3]);
  }
  uint16_t *dst = me.is_v ? g.b + t * g.b_row + h * g.b_head : g.a + t * g.a_row + h * g.a_head;
  *reinterpret_cast<uint2 *>(dst + me.d0) = make_uint2(out[0], out[1]);
  *reinterpret_cast<uint2 *>(dst + me.d1) = make_uint2(out[2], out[3]);
}

// -------------------------------------------------------------------------------------------------------------------
// Attention
// -------------------------------------------------------------------------------------------------------------------
template <bool F16>
__device__ __forceinline__ void mma_16n8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_16816(d, a, b0, b1);
}

// Nibbles j and 4 + j of w as a pair of 16-bit floats kOff + code.
template <bool F16, int J>
__device__ __forceinline__ uint32_t nibbles(uint32_t w) {
  if (F16) {
    const uint32_t s = J == 0 ? w << 4 : w >> (4 * (J > 0 ? J - 1 : 0));
    return (s & 0x00f000f0u) | 0x54005400u;
  }
  return ((w >> (4 * J)) & 0x000f000fu) | 0x43004300u;
}
// The same less kOff + 8: code - 8, exact.
template <bool F16, int J>
__device__ __forceinline__ uint32_t centred(uint32_t w) {
  uint32_t r;
  const uint32_t x = nibbles<F16, J>(w);
  if (F16) asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x54805480u));
  else asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x43084308u));
  return r;
}
template <bool F16>
constexpr float kKvOff = F16 ? 64.0f : 128.0f;

// How far (log2) a score may pass its row's reference before the reference moves.  The weight times the V scale is an operand
// in the cache's type: fp16 holds 2^2 times the largest scale of fp16 values, (2 * 65504) / 15, and no 2^3.
template <bool F16>
constexpr float kKvGrow = F16 ? 2.0f : 8.0f;

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

// Work list: tiles before slot s times the items (KV head, row block) of a slot; worker w takes tiles [w total / n,
// (w + 1) total / n).
__device__ __forceinline__ int64_t kv4_start(int64_t w, int64_t total, int64_t n) { return w * total / n; }
__device__ __forceinline__ int64_t kv4_worker(int64_t tile, int64_t total, int64_t n) { return ((tile + 1) * n - 1) / total; }

template <int D, int NG, int NT, bool F16>
__global__ void __launch_bounds__(kKvWarps * 32, NT == 1 ? 3 : 2) kv4_attn_kernel(const __grid_constant__ Kv4Args g) {
  constexpr int kStage = kKvTile * (D + 8 * NG);            // bytes of a tile: one block of 32 keys or two of 16
  constexpr int kWordsK = D / 32, kWordsV = D / 64;         // words a lane takes of a K and of a V row
  constexpr int kGroup = D / NG;
  constexpr float kOff = kKvOff<F16>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *ring = smem + (threadIdx.x >> 5) * kKvStages * kStage;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kKvWarps * kKvStages * kStage) + (threadIdx.x >> 5) * kKvStages;
  int32_t *good = reinterpret_cast<int32_t *>(smem + kKvWarps * kKvStages * (kStage + 8)) + (threadIdx.x >> 5) * kKvStages;
  int32_t *before = reinterpret_cast<int32_t *>(smem + kKvWarps * kKvStages * (kStage + 12));   // [slots + 1] tiles before a slot
  __shared__ int32_t sums[kKvWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, qd = lane & 3;
  const uint32_t wl = g.stall ? kTestWaitUs : kWaitUs;
  if (lane == 0) {
    for (int i = 0; i < kKvStages; ++i) sm100::mbar_init(&full[i], 1);
    sm100::fence_barrier_init();
  }
  pdl_enter();

  // before[s]: a thread sums a run of slots, the runs are scanned over the CTA.
  const int run = (g.slots + kKvWarps * 32 - 1) / (kKvWarps * 32), s_lo = threadIdx.x * run;
  int mine = 0;
  for (int s = s_lo; s < min(s_lo + run, g.slots); ++s) mine += kv4_tiles(g, g.lens[s]);
  int scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) sums[warp] = scan;
  __syncthreads();
  for (int w = 0; w < warp; ++w) scan += sums[w];
  int at = scan - mine;
  for (int s = s_lo; s < min(s_lo + run, g.slots); ++s) {
    before[s] = at;
    at += kv4_tiles(g, g.lens[s]);
  }
  if (threadIdx.x == kKvWarps * 32 - 1) before[g.slots] = scan;
  __syncthreads();

  const int items = g.hkv * g.rb;                           // items of a slot
  const int64_t total = int64_t(before[g.slots]) * items;
  const int64_t worker = int64_t(warp) * gridDim.x + blockIdx.x;
  const int64_t n = min(int64_t(g.workers), total);
  if (worker >= n) return;
  const int64_t w_lo = kv4_start(worker, total, n), w_hi = kv4_start(worker + 1, total, n);

  // Position in the list: slot, item of the slot, tile of the item.
  struct Cursor {
    int slot, item, tile, tiles;
  };
  auto seek = [&](int64_t x) {
    int lo = 0, hi = g.slots;                               // the last slot with before * items <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (int64_t(before[mid]) * items <= x) lo = mid;
      else hi = mid;
    }
    Cursor c;
    c.slot = lo;
    c.tiles = before[lo + 1] - before[lo];
    const int64_t in = x - int64_t(before[lo]) * items;
    c.item = int(in / c.tiles);
    c.tile = int(in % c.tiles);
    return c;
  };
  auto step = [&](Cursor &c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.item < items) return;
    c.item = 0;
    do {
      ++c.slot;
      c.tiles = c.slot < g.slots ? before[c.slot + 1] - before[c.slot] : 1;
    } while (c.tiles == 0);
  };

  // Producer side: lane k < parts holds the pool page of the k-th part of the tile that is copied next.
  const int bs = g.page_size < kKvTile ? g.page_size : kKvTile, parts = kKvTile / bs;
  const uint32_t part_bytes = uint32_t(bs * (D + 8 * NG));
  auto next_page = [&](const Cursor &c, bool any) {
    int page = -2;                                          // -2: no key of the slot lies there
    if (any && lane < parts) {
      const int first = c.tile * kKvTile + lane * bs;
      if (first < g.lens[c.slot]) {
        page = g.table[int64_t(c.slot) * g.max_pages + first / g.page_size];
        if (page < 0 || page >= g.pages) page = -1;
      }
    }
    return page;
  };
  auto copy = [&](const Cursor &c, int page, int64_t x) {
    const int st = int(x - w_lo) % kKvStages;
    const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0);
    if (lane < parts && page == -1) record_status(PTSIM_E_OOB);
    if (lane == 0) {
      good[st] = int(ok);
      sm100::mbar_arrive_expect_tx(&full[st], part_bytes * __popc(ok));
    }
    __syncwarp();
    if (page >= 0 && !(g.stall && blockIdx.x == 0 && warp == 0 && x == w_lo)) {   // test hook: armed, no copy in flight
      const int block = ((c.tile * kKvTile + lane * bs) & (g.page_size - 1)) / bs;
      const uint8_t *src = g.pool + (int64_t(page) * g.hkv + c.item / g.rb) * g.record + uint32_t(block) * part_bytes;
      sm100::bulk_load_g2s(ring + st * kStage + lane * part_bytes, src, part_bytes, &full[st]);
    }
  };

  Cursor use = seek(w_lo), fill = use;
  int64_t fx = w_lo;                                        // next tile to copy
  int page = next_page(fill, true);
  auto feed = [&]() {                                       // copy tile fx, then fetch the next one's pages
    if (fx >= w_hi) return;
    copy(fill, page, fx);
    ++fx;
    if (fx < w_hi) {
      step(fill);
      page = next_page(fill, true);
    }
  };
  for (int i = 0; i < kKvStages; ++i) feed();

  // Offsets of a 16-key step within a tile.
  const bool small = bs == 16;
  const int step_k = small ? 16 * (D + 8 * NG) : 8 * D, step_p = small ? 16 * (D + 8 * NG) : 64 * NG;
  const int v_at = bs * (D / 2), kp_at = bs * D, vp_at = kp_at + bs * 4 * NG;
  const int v_lane = qd * (D / 2) + (D == 128 ? (gq ^ ((qd & 2) << 1)) * 8 : gq * 4);

  bool ok = true;
  int64_t x = w_lo;
  while (ok && x < w_hi) {
    // One item's part: tiles [use.tile, last) of (slot, KV head, row block).
    const int slot = use.slot, head = use.item / g.rb, row0 = (use.item % g.rb) * 16;
    const int first = use.tile, last = int(min(int64_t(use.tiles), use.tile + (w_hi - x)));
    const int rows = min(16, g.per - row0), len = g.lens[slot];
    const bool whole = first == 0 && last == use.tiles, opening = x == w_lo;

    uint32_t qb[NT][kWordsK][4];                            // d = 32 b + 8 qd + 0 .. 7 of row gq
    float qsum[NT][2][NG];                                  // of rows 2 qd and 2 qd + 1, per group
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = t * 8 + gq;
      const uint16_t *q = g.a + slot * g.a_row + int64_t(head * g.per + row0 + r) * g.a_head + qd * 8;
      float s[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) s[i] = 0.f;
#pragma unroll
      for (int b = 0; b < kWordsK; ++b) {
        const uint4 w = r < rows ? *reinterpret_cast<const uint4 *>(q + b * 32) : make_uint4(0, 0, 0, 0);
        qb[t][b][0] = w.x, qb[t][b][1] = w.y, qb[t][b][2] = w.z, qb[t][b][3] = w.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[b * 32 / kGroup] += lo_f32<F16>(qb[t][b][i]) + hi_f32<F16>(qb[t][b][i]);
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
        qsum[t][0][i] = __shfl_sync(0xffffffffu, s[i], 8 * qd);
        qsum[t][1][i] = __shfl_sync(0xffffffffu, s[i], 8 * qd + 4);
      }
    }
    float m[NT][2], l[NT][2], corr[NT][2][NG], o[NT][D / 16][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[t][i] = -INFINITY;
        l[t][i] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) corr[t][i][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    }

    for (int tile = first; tile < last; ++tile, ++x) {
      const int st = int(x - w_lo) % kKvStages;
      if (!sm100::mbar_wait(&full[st], uint32_t(int(x - w_lo) / kKvStages) & 1, wl)) {
        ok = false;
        break;
      }
      const uint8_t *buf = ring + st * kStage;
      // Keys past the length, or whose page is not there, take no part: score -inf and parameters 0.
      const int left = len - tile * kKvTile, there = good[st];
      const bool partial = left < kKvTile || there != (1 << parts) - 1;
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
        const uint32_t *kpar = reinterpret_cast<const uint32_t *>(buf + kp_at + h * step_p) + gq * NG;
        const uint32_t *vpar = reinterpret_cast<const uint32_t *>(buf + vp_at + h * step_p) + gq * NG;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          kp[0][i] = kpar[i], kp[1][i] = kpar[8 * NG + i];
          vp[h][0][i] = vpar[i], vp[h][1][i] = vpar[8 * NG + i];
        }
        float acc[NT][NG][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            acc[t][i][0] = acc[t][i][2] = -kOff * qsum[t][0][i];
            acc[t][i][1] = acc[t][i][3] = -kOff * qsum[t][1][i];
          }
#pragma unroll
        for (int b = 0; b < kWordsK; ++b) {
          const uint32_t a0[4] = {nibbles<F16, 0>(wa[b]), nibbles<F16, 0>(wb[b]), nibbles<F16, 1>(wa[b]), nibbles<F16, 1>(wb[b])};
          const uint32_t a1[4] = {nibbles<F16, 2>(wa[b]), nibbles<F16, 2>(wb[b]), nibbles<F16, 3>(wa[b]), nibbles<F16, 3>(wb[b])};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_16n8<F16>(acc[t][b * 32 / kGroup], a0, qb[t][b][0], qb[t][b][1]);
            mma_16n8<F16>(acc[t][b * 32 / kGroup], a1, qb[t][b][2], qb[t][b][3]);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NG; ++i)
              s = fmaf(lo_f32<F16>(kp[k >> 1][i]), acc[t][i][k], fmaf(hi_f32<F16>(kp[k >> 1][i]), qsum[t][k & 1][i], s));
            z[h][t][k] = s * g.sl;
          }
        if (partial) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int key = h * 16 + k * 8 + gq;
            if (key < left && ((there >> (small ? h : 0)) & 1)) continue;
#pragma unroll
            for (int t = 0; t < NT; ++t) z[h][t][2 * k] = z[h][t][2 * k + 1] = -INFINITY;
#pragma unroll
            for (int i = 0; i < NG; ++i) vp[h][k][i] = 0;
          }
        }
      }
      // A row's reference moves only when a score passes it by kKvGrow (the first key always does).
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 8; ++k) grow |= z[k >> 2][t][k & 3] > m[t][k & 1] + kKvGrow<F16>;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(fmaxf(z[0][t][i], z[0][t][i + 2]), fmaxf(z[1][t][i], z[1][t][i + 2]));
#pragma unroll
            for (int s = 4; s < 32; s *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
            const float to = fmaxf(m[t][i], top);
            const float alpha = to == m[t][i] ? 1.f : ex2_fast(m[t][i] - to);   // equal: both may be -inf
            m[t][i] = to;
            l[t][i] *= alpha;
#pragma unroll
            for (int k = 0; k < NG; ++k) corr[t][i][k] *= alpha;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) o[t][k][i] *= alpha, o[t][k][i + 2] *= alpha;
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // Weights times the V scales, rounded: per group the operand [16 keys x 8 rows], transposed from the scores' layout.
        uint32_t pb[NT][NG][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float p[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            p[k] = ex2_fast(z[h][t][k] - (m[t][k & 1] == -INFINITY ? 0.f : m[t][k & 1]));
            l[t][k & 1] += p[k];
          }
#pragma unroll
          for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float a = lo_f32<F16>(vp[h][k][i]), mid = fmaf(8.f, a, hi_f32<F16>(vp[h][k][i]));
              const uint32_t w = pack_16x2<F16>(p[2 * k] * a, p[2 * k + 1] * a);
              corr[t][0][i] = fmaf(p[2 * k], mid, corr[t][0][i]);
              corr[t][1][i] = fmaf(p[2 * k + 1], mid, corr[t][1][i]);
              pb[t][i][k] = transpose_8x8(w);
            }
        }
        const uint8_t *vc = buf + v_at + h * step_k + v_lane;   // keys 2 qd, 2 qd + 1, 2 qd + 8, 2 qd + 9: rows qd, + 4, + 8, + 12
        __align__(8) uint32_t w[4][kWordsV];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (D == 128) *reinterpret_cast<uint2 *>(w[r]) = *reinterpret_cast<const uint2 *>(vc + r * 4 * (D / 2));
          else w[r][0] = *reinterpret_cast<const uint32_t *>(vc + r * 4 * (D / 2));
        }
#pragma unroll
        for (int v = 0; v < kWordsV; ++v)
#pragma unroll
          for (int half = 0; half < 2; ++half) {                // nibbles 0-3: d = 64 v + 4 gq ..; 4-7: 32 further
            const uint32_t lo = __byte_perm(w[0][v], w[1][v], half ? 0x7632 : 0x5410);
            const uint32_t hi = __byte_perm(w[2][v], w[3][v], half ? 0x7632 : 0x5410);
            const uint32_t a0[4] = {centred<F16, 0>(lo), centred<F16, 1>(lo), centred<F16, 0>(hi), centred<F16, 1>(hi)};
            const uint32_t a1[4] = {centred<F16, 2>(lo), centred<F16, 3>(lo), centred<F16, 2>(hi), centred<F16, 3>(hi)};
            const int gr = (v * 64 + half * 32) / kGroup;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma_16n8<F16>(o[t][v * 4 + half * 2], a0, pb[t][gr][0], pb[t][gr][1]);
              mma_16n8<F16>(o[t][v * 4 + half * 2 + 1], a1, pb[t][gr][0], pb[t][gr][1]);
            }
          }
      }
      __syncwarp();                                           // every lane has read the stage: it may be filled again
      feed();
    }
    if (!ok) break;

    // The part's rows: sums over the lanes of a row, then o or the workspace.  Rows 2 qd (+ 1), d = 64 v + 32 half + 4 gq + 0 .. 3.
    const int64_t slot_at = 2 * worker + (opening ? 0 : 1);
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
        const float inv = whole ? (m[t][i] == -INFINITY && l[t][i] == 0.f ? 0.f : 1.f / l[t][i]) : 1.f;
        float *part = g.part_o + (slot_at * 16 + r) * D;
        uint16_t *out = g.b + slot * g.b_row + int64_t(head * g.per + row0 + r) * g.b_head;
#pragma unroll
        for (int v = 0; v < kWordsV; ++v)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int d = v * 64 + half * 32 + gq * 4;
            const float c = corr[t][i][(v * 64 + half * 32) / kGroup];
            const float y0 = (o[t][v * 4 + half * 2][i] + c) * inv, y1 = (o[t][v * 4 + half * 2][i + 2] + c) * inv;
            const float y2 = (o[t][v * 4 + half * 2 + 1][i] + c) * inv, y3 = (o[t][v * 4 + half * 2 + 1][i + 2] + c) * inv;
            if (whole) *reinterpret_cast<uint2 *>(out + d) = make_uint2(pack_16x2<F16>(y0, y1), pack_16x2<F16>(y2, y3));
            else *reinterpret_cast<float4 *>(part + d) = make_float4(y0, y1, y2, y3);
          }
        if (!whole && gq == 0) {
          g.part_ml[(slot_at * 16 + r) * 2] = m[t][i];
          g.part_ml[(slot_at * 16 + r) * 2 + 1] = l[t][i];
        }
      }
    if (x < w_hi) use = seek(x);
  }
  // After a wait that gave up, the copies in flight land (bounded) before the warp leaves its ring.
  if (!ok)
    for (int64_t i = max(x, fx - kKvStages); i < fx; ++i)
      sm100::mbar_wait(&full[int(i - w_lo) % kKvStages], uint32_t(int(i - w_lo) / kKvStages) & 1, wl);
}

// One CTA per (slot, item): merges the parts of an item that several workers hold, in key order; zeros for an empty slot.
// Threads: D columns x 256 / D rows at a time.
template <int D, bool F16>
__global__ void __launch_bounds__(256) kv4_merge_kernel(const __grid_constant__ Kv4Args g) {
  __shared__ int32_t sums[2][8];
  const int items = g.hkv * g.rb, slot = int(blockIdx.x) / items, item = int(blockIdx.x) % items;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_enter();
  int total = 0, prior = 0;
  for (int s = threadIdx.x; s < g.slots; s += 256) {
    const int n = kv4_tiles(g, g.lens[s]);
    total += n;
    prior += s < slot ? n : 0;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  prior = __reduce_add_sync(0xffffffffu, prior);
  if (lane == 0) sums[0][warp] = total, sums[1][warp] = prior;
  __syncthreads();
  total = prior = 0;
  for (int w = 0; w < 8; ++w) total += sums[0][w], prior += sums[1][w];
  const int tiles = kv4_tiles(g, g.lens[slot]);
  const int head = item / g.rb, row0 = (item % g.rb) * 16, rows = min(16, g.per - row0);
  const int d = threadIdx.x % D;
  const int64_t all = int64_t(total) * items, n = min(int64_t(g.workers), all);
  const int64_t t0 = int64_t(prior) * items + int64_t(item) * tiles;
  int64_t w0 = 0, w1 = -1;
  if (tiles > 0) {
    w0 = kv4_worker(t0, all, n), w1 = kv4_worker(t0 + tiles - 1, all, n);
    if (w0 == w1) return;                                      // one worker held the whole item and wrote it
  }
  for (int r = threadIdx.x / D; r < rows; r += 256 / D) {
    float top = -INFINITY, L = 0.f, O = 0.f;
    auto at = [&](int64_t w) { return (2 * w + (kv4_start(w, all, n) >= t0 ? 0 : 1)) * 16 + r; };
    for (int64_t w = w0; w <= w1; ++w) top = fmaxf(top, g.part_ml[at(w) * 2]);
    for (int64_t w = w0; w <= w1; ++w) {
      const float mw = g.part_ml[at(w) * 2];
      const float e = mw == -INFINITY ? (g.part_ml[at(w) * 2 + 1] == 0.f ? 0.f : 1.f) : ex2_fast(mw - top);
      L += g.part_ml[at(w) * 2 + 1] * e;
      O += g.part_o[at(w) * D + d] * e;
    }
    const float y = top == -INFINITY && L == 0.f ? 0.f : O / L;
    g.b[slot * g.b_row + int64_t(head * g.per + row0 + r) * g.b_head + d] = uint16_t(pack_16x2<F16>(y, y) & 0xffffu);
  }
}

// Workers of a launch: one warp each, as many as are resident at once.
static int kv4_workers(const ptsim_kv4_params &p, int sm_count) {
  return sm_count * (p.hq / p.hkv <= 8 ? 3 : 2) * kKvWarps;
}

int64_t kv4_workspace(const ptsim_desc &d, int sm_count) {
  const ptsim_kv4_params &p = d.p.kv4;
  return 2 * int64_t(kv4_workers(p, sm_count)) * 16 * (p.dim + 2) * int64_t(sizeof(float));
}

template <int D, int NG, int NT, bool F16>
static int run_kv4_attn(const Kv4Args &g, const LaunchCtx &c) {
  constexpr auto kern = kv4_attn_kernel<D, NG, NT, F16>;
  constexpr int fixed = kKvWarps * kKvStages * (kKvTile * (D + 8 * NG) + 12) + 16;
  PTSIM_CUDA((smem_limit_once<kern>(fixed + 4 * (PTSIM_KV4_SLOTS + 1), c.device)));
  PTSIM_CUDA(launch_pdl(kern, dim3(unsigned(g.workers / kKvWarps)), dim3(kKvWarps * 32), fixed + 4 * (g.slots + 1), c.stream, g));
  PTSIM_CUDA(launch_pdl(kv4_merge_kernel<D, F16>, dim3(unsigned(g.slots * g.hkv * g.rb)), dim3(256), 0, c.stream, g));
  return PTSIM_OK;
}

template <int D, int NG, bool F16>
static int run_kv4(const ptsim_desc &d, Kv4Args &g, uint8_t *pool, const LaunchCtx &c) {
  if (d.kind == PTSIM_KIND_ATTN_KV4)
    return d.p.kv4.hq / d.p.kv4.hkv <= 8 ? run_kv4_attn<D, NG, 1, F16>(g, c) : run_kv4_attn<D, NG, 2, F16>(g, c);
  constexpr int kHeads = 128 / D;
  const int64_t units = g.tokens * ceil_div(g.hkv, kHeads);
  const dim3 grid(unsigned(ceil_div(units, 8)));
  if (d.kind == PTSIM_KIND_KV4_STORE)
    PTSIM_CUDA(launch_pdl(kv4_store_kernel<D, NG, F16>, grid, dim3(256), 0, c.stream, g, pool));
  else
    PTSIM_CUDA(launch_pdl(kv4_load_kernel<D, NG, F16>, grid, dim3(256), 0, c.stream, g));
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
