// Causal GQA attention of prompts of different lengths packed back to back (PTSIM_KIND_ATTN_PACKED); no counterpart in
// the reference, whose prefill program has one length (attention.cuh).
//
// Query i of a sequence with ql queries and kl keys sits at position p = i + kl - ql and sees keys j <= p.  With z_j =
// scale q.k_j the row's result is sum_j e^(z_j - m) v_j / sum_j e^(z_j - m) for any reference m: key tiles are visited once, the
// row keeps m, l = sum e^(z_j - m) and O = sum e^(z_j - m) v_j, and O and l are rescaled when m moves.
//
// One CTA per (128 T query rows of a sequence, head), T = 1 or 2 tiles of 128 rows that share each 128-key tile, with the
// hand-offs of attn2_fwd_kernel: warp 0 TMA, warp 1 tcgen05.mma, warps 2 and 3 below, then four softmax warps per tile; S, P
// and O in TMEM.  What is different:
//   - the lengths are known on the device only, so the grid is the bound floor(tokens / 128 T) + seqs items a head, and a CTA
//     finds its item in the tables: items go by descending number of key tiles over all sequences (the longest first, so the
//     CTAs that start last are short; by row index, 12 chunks behind prefixes of up to 1500 keys took 52 us, by tiles 37), by
//     a binary search on how many have at least x;
//   - T = 2 has K and V in two stages and an SM to itself; T = 1 has one stage and half an SM, so that the set-up, first
//     loads and epilogue of one item overlap another item's products (set-up to teardown, an item of one tile takes 17400 clocks,
//     of which 2100 are its softmax).  Which is faster is a matter of length: packed_tiles();
//   - masks: a tile past a row's position is masked by comparison, so tiles need no alignment with the lengths; only in the
//     32-column chunks that the diagonal crosses for a warp's rows, and chunks beyond it are not exponentiated;
//   - a V row that some row of the item does not see would still meet that row's P = 0, and 0 * NaN is NaN.  Warps 2 and 3
//     go over the V tiles that hold such rows (the last one to three of an item) before the MMA reads them: rows of the
//     next sequence are cleared, and a non-finite value within the sequence is cleared and noted per column with its first
//     key; the epilogue adds it to the rows that do see it.  The scan overlaps S = Q K^T and the first softmax;
//   - O leaves through Q's shared memory, whole rows by a few lanes each (a row a lane is 32 lines per store: 4000 clocks).
// Bound: the tensor core, 4 D flop per (query, key, head), and the exponential unit beside it (16384 exponentials of a score
// tile take as many clocks as its two products at D 128).  One prompt of 8192, 32 / 8 heads of 128: 532 us between idle gaps
// (1.03 PFLOP/s, 0.60 of the measured burst), 577 back to back under the power cap.  16 prompts of up to 1021: 115 us; each
// tile costs a chain of softmax, P V and next scores, and each item a set-up, first loads and an epilogue.  The register split leaves
// spills (at D 128 200 bytes of loads for T = 1, 372 for T = 2; 144 and 336 at D 64; the one-length kernel has none).
// P is rounded to the inputs' 16-bit type for the tensor core (half a step, 2^-9 of each weight for bf16, 2^-12 for fp16),
// as the prefill program does; z, m, l and O are fp32.
#pragma once
#include "attention.cuh"

namespace ptsim {

constexpr int kPackNever = 0x7fffffff;

struct PackedArgs {
  CUtensorMap tq, tk, tv;            // [heads][tokens][dim], box {64, 128, 1}
  const int32_t *cuq, *cuk;
  uint16_t *o;
  int64_t o_row, o_head;
  int32_t q_tokens, k_tokens, seqs, hq, per;   // per: query heads of one KV head
  float scale;
  int32_t stall;                     // PTSIM_FLAG_TEST_STALL
};

// Registers a thread after the split: first warpgroup, softmax warpgroups.  They draw on what the block is launched with, 168 a
// thread for T = 2 (384 threads), 128 for T = 1 (256 threads, two blocks an SM).
template <int T>
struct PackedShape {
  static constexpr int kThreads = 128 + 128 * T;
  static constexpr int kLaunchRegs = T == 2 ? 168 : 128;
  static constexpr int kRegs0 = T == 2 ? 56 : 48, kRegs1 = T == 2 ? 224 : 208;
  static_assert(128 * kRegs0 + 128 * T * kRegs1 <= kThreads * kLaunchRegs, "register split above the launch's registers");
};

template <int D, int T>
constexpr int packed_smem(int seqs) {
  return 3 * T * 128 * D * 2 + 1024 + 256 + 3 * D * 4 + seqs * 8;
}

// Two floats rounded to a packed pair of the 16-bit type (lo in bits 0-15).
template <bool F16>
__device__ __forceinline__ uint32_t pack_16x2(float lo, float hi) {
  if (!F16) return pack_bf16x2(lo, hi);
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 16-byte unit of eight 16-bit values: does any have all exponent bits set (an infinity or a NaN)?
template <bool F16>
__device__ __forceinline__ uint32_t nonfinite8(const uint4 &w) {
  constexpr uint32_t mask = F16 ? 0x7c007c00u : 0x7f807f80u, one = F16 ? 0x04000400u : 0x00800080u;
  return (((w.x & mask) + one) | ((w.y & mask) + one) | ((w.z & mask) + one) | ((w.w & mask) + one)) & 0x80008000u;
}

// An item: its first query row (-1: none), the rows of tiles A and B, the sequence's first key row and keys, row 0's position.
struct PackedItem {
  int q0, rows_a, rows_b, k0, kl, pos0;
};
constexpr int kPackGridY = 32768;

template <int D, bool F16, int T>
__global__ void __launch_bounds__(PackedShape<T>::kThreads, T == 2 ? 1 : 2) packed_attn_kernel(const __grid_constant__ PackedArgs g) {
  constexpr int kThreads = PackedShape<T>::kThreads, kRows = 128 * T;
  constexpr int kTile = 128 * D * 2;                 // bytes of a [128 x D] operand tile: D / 64 swizzled halves of 16 KB
  constexpr int kHalf = 128 * 64 * 2;
  constexpr uint32_t kTmem = 256 * T, kO = 128 * T;  // TMEM columns; S of tile t at 128 t, O at kO + 128 t
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = smem + T * kTile, *sV = smem + 2 * T * kTile;   // Q of each tile; T stages of K and of V
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + 3 * T * kTile);
  uint64_t *q_full = bars + 0, *drain = bars + 1;
  uint64_t *k_full = bars + 2, *v_full = bars + 4;   // 2 each
  uint64_t *k_empty = bars + 6, *v_empty = bars + 8; // 2 each
  uint64_t *s_full = bars + 10, *o_done = bars + 12; // per tile
  uint64_t *scan_full = bars + 14;                   // 2: v_full of the tiles that are scanned
  uint64_t *p_full = bars + 16;                      // per tile, one arrival per softmax warp
  uint64_t *v_clean = bars + 18;                     // 2, one arrival per scanning warp
  uint64_t *scanned = bars + 20;                     // the same, once, after the last scan
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 21);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  volatile int *dirty = abort_flag + 1;              // a noted non-finite value of V
  PackedItem *found = reinterpret_cast<PackedItem *>(tmem_slot + 4);
  int32_t *noted = reinterpret_cast<int32_t *>(smem + 3 * T * kTile + 256);   // first key of NaN, +inf, -inf: [3][D]
  int2 *lens = reinterpret_cast<int2 *>(noted + 3 * D);                   // queries and keys of each sequence past the 32nd

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t wl = g.stall ? kTestWaitUs : kWaitUs;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 21; ++i) sm100::mbar_init(&bars[i], i == 16 || i == 17 ? 4u : i >= 18 ? 2u : 1u);
    *abort_flag = 0;
    *dirty = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, kTmem);
    sm100::tmem_relinquish();
  }
  for (int i = threadIdx.x; i < 3 * D; i += kThreads) noted[i] = kPackNever;
  pdl_enter();   // set-up above overlaps the previous kernel's tail; global memory after

  // Warp 0 finds the item: the rank'th of a head's items in descending key tiles, sequences in order for equal ones.  A lane
  // looks after every 32nd sequence, the first of them in registers.  Then it asks for the first tiles at once; the other
  // warps meet it at the barrier below.
  const int head = int(blockIdx.x), rank = int(blockIdx.z) * kPackGridY + int(blockIdx.y);
  PackedItem it;
  if (warp == 0) {
    auto rows_of = [&](int s) {                          // queries and keys of sequence s
      const int a = g.cuq[s], b = g.cuq[s + 1], c = g.cuk[s], d = g.cuk[s + 1];
      const bool good = a >= 0 && b >= a && b <= g.q_tokens && c >= 0 && d >= c && d <= g.k_tokens;
      if (!good) record_status(PTSIM_E_OOB);
      return good ? make_int2(b - a, d - c) : make_int2(0, 0);
    };
    // Its items, and those with at least x key tiles: its last ones (item p's tiles end at key kl - ql + kRows (p + 1), or kl).
    auto items_of = [&](const int2 &len) { return (len.x + kRows - 1) / kRows; };
    auto with_tiles = [&](const int2 &len, int x) {
      const int np = items_of(len);
      if (x <= 0 || np == 0) return np;
      return x > (len.y + 127) >> 7 ? 0 : np - min(np - 1, max(0, ((x - 1) * 128 - len.y + len.x) >> (T == 2 ? 8 : 7)));
    };
    const int2 mine = lane < g.seqs ? rows_of(lane) : make_int2(0, 0);
    int most = mine.y, all = items_of(mine);
    for (int s = lane + 32; s < g.seqs; s += 32) {
      const int2 len = rows_of(s);
      lens[s] = len;
      most = max(most, len.y), all += items_of(len);
    }
    most = (__reduce_max_sync(0xffffffffu, most) + 127) >> 7, all = __reduce_add_sync(0xffffffffu, all);
    auto all_with = [&](int x) {
      int n = with_tiles(mine, x);
      for (int s = lane + 32; s < g.seqs; s += 32) n += with_tiles(lens[s], x);
      return __reduce_add_sync(0xffffffffu, n);
    };
    int seq = -1, p = 0;
    if (all > rank) {
      int lo = 0, hi = most + 1, above = 0;              // all_with(lo) > rank >= all_with(hi) = above
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, n = all_with(mid);
        if (n > rank) lo = mid;
        else hi = mid, above = n;
      }
      // Items of exactly lo tiles, sequence by sequence: the lane whose sequences' running count passes `left`.
      int left = rank - above;
      for (int s0 = 0; s0 < g.seqs; s0 += 32) {
        const int2 len = s0 == 0 ? mine : s0 + lane < g.seqs ? lens[s0 + lane] : make_int2(0, 0);
        const int more = with_tiles(len, lo + 1), n = with_tiles(len, lo) - more;
        int run = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
          const int up = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += up;
        }
        const uint32_t reached = __ballot_sync(0xffffffffu, run > left);
        if (reached) {
          const int at = __ffs(reached) - 1;
          seq = s0 + at;
          p = __shfl_sync(0xffffffffu, items_of(len) - 1 - more - (left - (run - n)), at);
          break;
        }
        left -= __shfl_sync(0xffffffffu, run, 31);
      }
    }
    it.q0 = -1;
    if (seq >= 0) {
      const int q0 = g.cuq[seq], ql = g.cuq[seq + 1] - q0, row0 = p * kRows;
      it.k0 = g.cuk[seq], it.kl = g.cuk[seq + 1] - it.k0;
      it.q0 = q0 + row0;
      it.pos0 = row0 + it.kl - ql;
      it.rows_a = min(128, ql - row0);
      it.rows_b = T == 2 ? max(0, min(128, ql - row0 - 128)) : 0;
    }
    if (lane == 0) {
      *found = it;
      const int last = it.pos0 + (it.rows_b > 0 ? 128 + it.rows_b : it.rows_a);   // keys that the item's last row sees
      if (seq >= 0 && last > 0) {
        const int kvh = head / g.per;
        // Only tiles that see a key: one that sees none has nothing to wait for before it stages its zeros over its Q.
        const int t0 = it.pos0 + it.rows_a > 0 ? 0 : 1, t1 = it.rows_b > 0 ? 2 : 1;
        sm100::mbar_arrive_expect_tx(q_full, (t1 - t0) * kTile);
        for (int t = t0; t < t1; ++t)
          for (int c = 0; c < D / 64; ++c)
            sm100::tma_load_3d(sQ + t * kTile + c * kHalf, &g.tq, q_full, c * 64, it.q0 + t * 128, head);
        sm100::mbar_arrive_expect_tx(&k_full[0], kTile);
        if (!(g.stall && head == 0 && rank == 0))          // test hook: K_0 armed, no copy in flight
          for (int c = 0; c < D / 64; ++c) sm100::tma_load_3d(sK + c * kHalf, &g.tk, &k_full[0], c * 64, it.k0, kvh);
      }
    }
    __syncwarp();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp != 0) it = *found;
  if (it.q0 < 0) {                         // the bound's spare CTAs (every thread of the CTA)
    if (warp == 1) sm100::tmem_dealloc(tmem, kTmem);
    return;
  }
  const int q0 = it.q0, k0 = it.k0, kl = it.kl, pos0 = it.pos0, rows_a = it.rows_a, rows_b = it.rows_b;
  const int nA = max(0, (pos0 + rows_a + 127) >> 7);                      // key tiles that some row sees
  const int nB = rows_b > 0 ? max(0, (pos0 + 128 + rows_b + 127) >> 7) : 0;
  const int n = max(nA, nB);
  const int first_scan = pos0 < 0 ? 0 : (pos0 + 1) >> 7;                  // tiles from here hold keys past row 0's position
  // Stage of tile j and the parity of its use.
  auto stage = [](int j) { return T == 2 ? j & 1 : 0; };
  auto parity = [](int j) { return uint32_t(T == 2 ? j >> 1 : j) & 1; };

  int kj = 0, vj = 0;   // (producer) K and V tiles whose stages were armed
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PackedShape<T>::kRegs0));
    if (warp == 0) {
      if (lane == 0 && n > 0) {
        const int kvh = head / g.per;
        for (int j = 0; j < n; ++j) {
          const int st = stage(j);
          if (j > 0) {                                     // Q and K_0 were asked for above
            if (!sm100::mbar_wait(&k_empty[st], parity(j) ^ 1, wl)) { *abort_flag = 1; break; }
            sm100::mbar_arrive_expect_tx(&k_full[st], kTile);
            for (int c = 0; c < D / 64; ++c)
              sm100::tma_load_3d(sK + st * kTile + c * kHalf, &g.tk, &k_full[st], c * 64, k0 + j * 128, kvh);
          }
          ++kj;
          if (!sm100::mbar_wait(&v_empty[st], parity(j) ^ 1, wl)) { *abort_flag = 1; break; }
          uint64_t *landed = j < first_scan ? &v_full[st] : &scan_full[st];
          sm100::mbar_arrive_expect_tx(landed, kTile);
          for (int c = 0; c < D / 64; ++c)
            sm100::tma_load_3d(sV + st * kTile + c * kHalf, &g.tv, landed, c * 64, k0 + j * 128, kvh);
          ++vj;
        }
      }
    } else if (warp == 1) {
      if (lane == 0 && n > 0) {
        constexpr uint32_t type = F16 ? 0u : (1u << 7) | (1u << 10);      // A and B formats
        constexpr uint32_t base = sm100::idesc_bf16_f32(128, 128, false, false) & ~((7u << 7) | (7u << 10));
        constexpr uint32_t idesc_s = base | type;
        constexpr uint32_t idesc_o = (sm100::idesc_bf16_f32(128, D, false, true) & ~((7u << 7) | (7u << 10))) | type;
        auto issue_s = [&](int t, int j) {
          const uint32_t k_addr = sm100::smem_u32(sK + stage(j) * kTile), q_addr = sm100::smem_u32(sQ + t * kTile);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
            sm100::mma_bf16_ss(tmem + t * 128, sm100::sw128_desc(q_addr + off, 16, 1024),
                               sm100::sw128_desc(k_addr + off, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
          }
          sm100::mma_commit(&s_full[t]);
        };
        auto issue_pv = [&](int t, int j) {
          const uint32_t v_addr = sm100::smem_u32(sV + stage(j) * kTile);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            sm100::mma_bf16_ts(tmem + kO + t * 128, tmem + t * 128 + k * 8,
                               sm100::sw128_desc(v_addr + k * 16 * 128, kHalf, 1024), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
          if (j == (t == 0 ? nA : nB) - 1) sm100::mma_commit(&o_done[t]);
        };
        // S_X(j + 1) overwrites P_X(j) in TMEM only after PV_X(j), issued before it, has read it (in-order execution).
        bool ok = sm100::mbar_wait(q_full, 0, wl) && sm100::mbar_wait(&k_full[0], 0, wl);
        if (ok) {
          sm100::tc_fence_after();
          if (nA > 0) issue_s(0, 0);
          if (T == 2 && nB > 0) issue_s(1, 0);
          sm100::mma_commit(&k_empty[0]);
        }
        for (int j = 0; ok && j < n; ++j) {
          const int st = stage(j);
          const bool next = j + 1 < n;
          // A scanned tile is complete once both scanning warps, which waited for its copies, have let it go.
          ok = j < first_scan ? sm100::mbar_wait(&v_full[st], parity(j), wl) : sm100::mbar_wait(&v_clean[st], parity(j - first_scan), wl);
          if (!ok) break;
          if (j < nA) {
            if (!(ok = sm100::mbar_wait(&p_full[0], j & 1, wl))) break;
            sm100::tc_fence_after();
            issue_pv(0, j);
          }
          if (T == 1) sm100::mma_commit(&v_empty[st]);
          if (next) {
            if (!(ok = sm100::mbar_wait(&k_full[stage(j + 1)], parity(j + 1), wl))) break;
            sm100::tc_fence_after();
            if (j + 1 < nA) issue_s(0, j + 1);
          }
          if (T == 2) {
            if (j < nB) {
              if (!(ok = sm100::mbar_wait(&p_full[1], j & 1, wl))) break;
              sm100::tc_fence_after();
              issue_pv(1, j);
            }
            sm100::mma_commit(&v_empty[st]);
            if (j + 1 < nB) issue_s(1, j + 1);
          }
          if (next) sm100::mma_commit(&k_empty[stage(j + 1)]);
        }
        if (!ok) *abort_flag = 1;
        sm100::mma_commit(drain);
        sm100::mbar_wait(drain, 0, wl);
      }
    } else {
      // Warps 2 and 3: V rows that some row of the item does not see (64 threads over 128 rows of D / 8 units).
      const int me = threadIdx.x - 64;
      for (int j = first_scan; j < n; ++j) {
        const int st = stage(j);
        if (!__all_sync(0xffffffffu, !*abort_flag && sm100::mbar_wait(&scan_full[st], parity(j - first_scan), wl))) {
          *abort_flag = 1;
          break;
        }
        uint8_t *v = sV + st * kTile;
        const int keys = min(128, kl - j * 128);
        uint32_t bad = 0;
#pragma unroll 8
        for (int i = 0; i < 128 * D / 8 / 64; ++i) {
          uint4 *u = reinterpret_cast<uint4 *>(v) + i * 64 + me;        // rows of 8 units within a half
          const int r = ((i * 64 + me) >> 3) & 127;
          if (r >= keys) *u = make_uint4(0, 0, 0, 0);
          else bad |= nonfinite8<F16>(*u);
        }
        if (bad) {                                                      // rare: go over this thread's units again, by value
          for (int i = 0; i < 128 * D / 8 / 64; ++i) {
            const int unit = i * 64 + me, r = (unit >> 3) & 127;
            uint16_t *h = reinterpret_cast<uint16_t *>(v) + unit * 8;
            if (r >= keys) continue;
            const int d0 = (unit >> 10) * 64 + (((unit & 7) ^ (r & 7)) << 3);
            for (int e = 0; e < 8; ++e) {
              const uint16_t x = h[e];
              const uint16_t ex = F16 ? 0x7c00 : 0x7f80;
              if ((x & ex) != ex) continue;
              const int what = (x & 0x7fff) != ex ? 0 : (x & 0x8000) ? 2 : 1;
              atomicMin(&noted[what * D + d0 + e], j * 128 + r);
              h[e] = 0;
            }
          }
          *dirty = 1;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&v_clean[st]);
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(scanned);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PackedShape<T>::kRegs1));
    const int t = (warp - 4) >> 2;           // tile
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;       // query row within the tile = TMEM lane
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + kO + t * 128 + lane_off;
    const int ntiles = t == 0 ? nA : nB, rows = t == 0 ? rows_a : rows_b;
    const int pos = pos0 + t * 128 + r;
    const int masked_from = pos0 + t * 128 < 0 ? 0 : (pos0 + t * 128 + 1) >> 7;   // tiles with keys past row 0 of this tile
    const float kLog2e = 1.4426950408889634f;
    const float sl = g.scale * kLog2e;
    // fp16 weights are kept 2^7 times larger (at most 2^15 with the lazy reference), so that small ones stay normal; l holds the same factor.
    constexpr float kBias = F16 ? 7.0f : 0.0f;
    float m = -INFINITY, l = 0.f;            // m in units of log2
    bool ok = true;
    // Tile j from its scores to its weights.  Masked: keys past a row's position get weight 0; the warp's rows see up to column
    // `low` of the tile (its first row) and `low + 31`.
    auto softmax = [&](int j, auto masked) {
      constexpr bool kMasked = decltype(masked)::value;
      const int low = kMasked ? pos - lane - j * 128 : 128;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) sm100::tmem_ld32(tS + c * 32, v[c]);
      sm100::tmem_wait_ld();
      if (kMasked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c * 32 + 31 <= low) continue;
          const int last = c * 32 > low + 31 ? -1 : low + lane;
#pragma unroll
          for (int q = 0; q < 32; ++q)
            if (c * 32 + q > last) v[c][q] = 0xff800000u;
        }
      }
      // Row maximum (scale > 0 keeps the arg max), eight independent chains.
      float mx8[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) mx8[q] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int q = 0; q < 32; ++q) mx8[q & 7] = fmaxf(mx8[q & 7], __uint_as_float(v[c][q]));
      const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                             fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
      // The reference moves only when the maximum passes it by more than 2^8: weights stay below 2^8 and O is rarely
      // rescaled; O / l does not depend on it.
      const float m_cand = fmaxf(m, mx * sl);
      const bool grow = m_cand - m > 8.0f;
      float alpha = 1.0f;
      if (grow) {
        alpha = ex2_fast(m - m_cand);
        m = m_cand;
      }
      const float off = (m == -INFINITY ? 0.f : -m) + kBias;
      const float2 a2 = make_float2(sl, sl), b2 = make_float2(off, off);
      float2 acc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
        if (kMasked && c * 32 > low + 31) {
#pragma unroll
          for (int q = 0; q < 16; ++q) pk[q] = 0;
        } else {
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 u = __ffma2_rn(make_float2(__uint_as_float(v[c][2 * q]), __uint_as_float(v[c][2 * q + 1])), a2, b2);
            const float p0 = ex2_fast(u.x), p1 = ex2_fast(u.y);
            acc[q & 3] = __fadd2_rn(acc[q & 3], make_float2(p0, p1));
            pk[q] = pack_16x2<F16>(p0, p1);
          }
        }
        sm100::tmem_st16(tS + c * 16, pk);
      }
      const float2 s2 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
      l = l * alpha + (s2.x + s2.y);
      // O already holds PV_X(j - 1): S_X(j) was issued after it.
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        const float2 al2 = make_float2(alpha, alpha);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          sm100::tmem_ld32(tO + c * 32, o);
          sm100::tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 x = __fmul2_rn(make_float2(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1])), al2);
            o[2 * q] = __float_as_uint(x.x);
            o[2 * q + 1] = __float_as_uint(x.y);
          }
          tmem_st32(tO + c * 32, o);
        }
      }
    };
    for (int j = 0; j < ntiles; ++j) {
      // The outcome is made the warp's: one lane must not leave a loop that others vote in.
      if (!(ok = __all_sync(0xffffffffu, !*abort_flag && sm100::mbar_wait(&s_full[t], j & 1, wl)))) break;
      sm100::tc_fence_after();
      if (j >= masked_from) softmax(j, std::true_type());
      else softmax(j, std::false_type());
      sm100::tmem_wait_st();
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&p_full[t]);
    }
    if (rows > 0) {
      if (ok && ntiles > 0)
        ok = __all_sync(0xffffffffu, !*abort_flag && sm100::mbar_wait(&o_done[t], 0, wl) && sm100::mbar_wait(scanned, 0, wl));
      if (ok) {
        sm100::tc_fence_after();
        const float inv = pos < 0 ? 0.f : 1.0f / l;
        // The warp's 32 rows, staged over Q (every product that reads this tile's is done, or the tile was never loaded), 16-byte
        // units exchanged by row.
        constexpr int kUnits = D / 8;
        uint8_t *mine = sQ + t * kTile + quarter * (kTile / 4);
        uint32_t v[D / 32][32];
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          if (ntiles > 0) sm100::tmem_ld32(tO + c * 32, v[c]);
        sm100::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float x[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) x[q] = pos < 0 ? 0.f : __uint_as_float(v[c][q]) * inv;   // no key: zeros
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(mine + lane * (D * 2) + (((c * 4 + q) ^ (lane & 7)) << 4)) =
                make_uint4(pack_16x2<F16>(x[q * 8], x[q * 8 + 1]), pack_16x2<F16>(x[q * 8 + 2], x[q * 8 + 3]),
                           pack_16x2<F16>(x[q * 8 + 4], x[q * 8 + 5]), pack_16x2<F16>(x[q * 8 + 6], x[q * 8 + 7]));
        }
        if (*dirty)                                            // noted values of V that the row sees
          for (int d = 0; d < D; ++d) {
            float add = 0.f;
            if (pos >= noted[D + d]) add += INFINITY;
            if (pos >= noted[2 * D + d]) add -= INFINITY;
            if (pos >= noted[d]) add = __uint_as_float(0x7fc00000u);
            uint16_t *e = reinterpret_cast<uint16_t *>(mine + lane * (D * 2) + (((d >> 3) ^ (lane & 7)) << 4)) + (d & 7);
            if (add != 0.f) {
              float x;
              if (F16) asm("cvt.f32.f16 %0, %1;" : "=f"(x) : "h"(*e));
              else x = bf16_bits_to_f32(*e);
              *e = uint16_t(pack_16x2<F16>(x + add, 0.f));
            }
          }
        __syncwarp();
        uint16_t *obase = g.o + int64_t(q0 + t * 128 + quarter * 32) * g.o_row + int64_t(head) * g.o_head;
        const int unit = lane % kUnits;
#pragma unroll 8
        for (int i = 0; i < kUnits; ++i) {
          const int row = i * (32 / kUnits) + lane / kUnits;
          if (quarter * 32 + row < rows)
            *reinterpret_cast<uint4 *>(obase + row * g.o_row + unit * 8) =
                *reinterpret_cast<const uint4 *>(mine + row * (D * 2) + ((unit ^ (row & 7)) << 4));
        }
      } else {
        *abort_flag = 1;
      }
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  // After an abort (final at the barrier above) the producer waits, bounded, for Q and the last fill of
  // each K and V stage, so no copy still lands in shared memory once the CTA has exited.
  if (warp == 0 && lane == 0 && *abort_flag && n > 0) {
    sm100::mbar_wait(q_full, 0, wl);
    for (int i = max(0, kj - T); i < kj; ++i) sm100::mbar_wait(&k_full[stage(i)], parity(i), wl);
    for (int i = max(0, vj - T); i < vj; ++i) {
      if (i < first_scan) sm100::mbar_wait(&v_full[stage(i)], parity(i), wl);
      else sm100::mbar_wait(&scan_full[stage(i)], parity(i - first_scan), wl);
    }
  }
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, kTmem);
  }
}

template <int D, bool F16, int T>
static int run_packed(const PackedArgs &g, const LaunchCtx &c) {
  constexpr auto kern = packed_attn_kernel<D, F16, T>;
  using Shape = PackedShape<T>;
  PTSIM_CUDA((smem_limit_once<kern>(packed_smem<D, T>(PTSIM_PACKED_SEQS), c.device)));
  // setmaxnreg.inc waits until the registers it asks for are free, so the warpgroups' shares must fit the registers the
  // block is launched with; refuse (rather than wait forever) if the build disagrees.
  static std::atomic<int> regs_ok{0};   // 0 unknown, 1 fits, 2 does not
  if (regs_ok.load() == 0) {
    cudaFuncAttributes fa;
    PTSIM_CUDA(cudaFuncGetAttributes(&fa, kern));
    regs_ok.store(fa.numRegs * Shape::kThreads >= 128 * Shape::kRegs0 + 128 * T * Shape::kRegs1 ? 1 : 2);
  }
  if (regs_ok.load() != 1) return fail(PTSIM_E_RESOURCE, "attention register split does not fit this build's registers");
  // floor(tokens / 128 T) full items and at most one more a sequence; heads of an item together.
  const int64_t most = int64_t(g.q_tokens) / (128 * T) + g.seqs, y = most < kPackGridY ? most : kPackGridY;
  PTSIM_CUDA(launch_pdl(kern, dim3(unsigned(g.hq), unsigned(y), unsigned(ceil_div(most, kPackGridY))), dim3(Shape::kThreads), packed_smem<D, T>(g.seqs), c.stream, g));
  return PTSIM_OK;
}

// Tiles of a CTA, by the average number of keys of a sequence (the lengths themselves are on the device).  Time of 148 heads
// (us) with one and with two tiles, dim 128, sequences of n: 64 3.97 / 6.76, 128 5.24 / 7.55, 256 11.0 / 12.8, 512 26.6 / 26.9,
// 1024 73.7 / 68.6; 256 queries behind 2048 keys 44.9 / 40.7.  Dim 64 (half the products, as many exponentials): 128 3.84 /
// 5.89, 512 20.7 / 23.8, 1024 57.1 / 60.9, 2048 176 / 180; 256 queries behind 4096 keys 67.6 / 66.8.  All of them batches of one
// length; of a skewed one (a long prompt beside many short ones, empty sequences, rows of no sequence) the average says little, and
// neither form has been measured on it.
static int packed_tiles(const PackedArgs &g, int dim) {
  return int64_t(g.k_tokens) < int64_t(g.seqs) * (dim == 64 ? 4096 : 768) ? 1 : 2;
}

template <int D, bool F16>
static int run_packed(const PackedArgs &g, const LaunchCtx &c) {
  return packed_tiles(g, D) == 2 ? run_packed<D, F16, 2>(g, c) : run_packed<D, F16, 1>(g, c);
}

int launch_packed(const ptsim_desc &d, void *const *ptrs, const LaunchCtx &c) {
  const ptsim_pattn_params &a = d.p.pattn;
  if (a.q_tokens == 0 || a.seqs == 0) return PTSIM_OK;
  PackedArgs g;
  memset(&g, 0, sizeof(g));
  auto at = [&](int arg, int64_t off) { return static_cast<uint16_t *>(ptrs[arg]) + off; };
  int rc = make_tmap_heads(&g.tq, at(a.q_arg, a.q_off), a.dim, a.q_tokens, a.hq, a.q_row, a.q_head, 64, 128);
  if (rc) return rc;
  // Without keys no K or V tile is loaded; the maps then stand over q.
  const bool keys = a.k_tokens > 0;
  if ((rc = make_tmap_heads(&g.tk, keys ? at(a.k_arg, a.k_off) : at(a.q_arg, a.q_off), a.dim, keys ? a.k_tokens : 1, a.hkv,
                            keys ? a.k_row : a.q_row, keys ? a.k_head : a.q_head, 64, 128)))
    return rc;
  if ((rc = make_tmap_heads(&g.tv, keys ? at(a.v_arg, a.v_off) : at(a.q_arg, a.q_off), a.dim, keys ? a.k_tokens : 1, a.hkv,
                            keys ? a.v_row : a.q_row, keys ? a.v_head : a.q_head, 64, 128)))
    return rc;
  g.o = at(a.o_arg, a.o_off);
  if (reinterpret_cast<uintptr_t>(g.o) % 16 != 0) return fail(PTSIM_E_ARGS, "the attention output is not 16-byte aligned");
  g.cuq = static_cast<const int32_t *>(ptrs[a.cuq_arg]);
  g.cuk = static_cast<const int32_t *>(ptrs[a.cuk_arg]);
  g.o_row = a.o_row;
  g.o_head = a.o_head;
  g.q_tokens = int(a.q_tokens);
  g.k_tokens = int(a.k_tokens);
  g.seqs = int(a.seqs);
  g.hq = int(a.hq);
  g.per = int(a.hq / a.hkv);
  g.scale = a.scale;
  g.stall = (d.flags & PTSIM_FLAG_TEST_STALL) ? 1 : 0;
  const bool f16 = d.arg_dtype[a.q_arg] == PTSIM_DT_F16;
  if (a.dim == 64) return f16 ? run_packed<64, true>(g, c) : run_packed<64, false>(g, c);
  return f16 ? run_packed<128, true>(g, c) : run_packed<128, false>(g, c);
}

}  // namespace ptsim
