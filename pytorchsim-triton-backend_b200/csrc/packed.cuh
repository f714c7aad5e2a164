// Causal GQA attention of prompts of different lengths packed back to back (PTSIM_KIND_ATTN_PACKED); no counterpart in
// the reference, whose prefill program has one length (attention.cuh).
//
// Query i of a sequence with ql queries and kl keys sits at position p = i + kl - ql and sees keys j <= p.  With z_j =
// scale q.k_j the row's result is sum_j e^(z_j - m) v_j / sum_j e^(z_j - m) for any reference m: key tiles are visited once, the
// row keeps m, l = sum e^(z_j - m) and O = sum e^(z_j - m) v_j, and O and l are rescaled when m moves.
//
// One CTA per (256 query rows of a sequence, head): two 128-row tiles A and B share each 128-key tile, as in
// attn2_fwd_kernel, whose hand-offs this kernel keeps (warp 0 TMA, warp 1 tcgen05.mma, warps 4-7 and 8-11 the softmax of A
// and B, S, P and O in TMEM).  What is different:
//   - the lengths are known on the device only, so the grid is the bound floor(tokens / 256) + seqs tile pairs a head and
//     a CTA finds its pair from the tables: pairs go in descending row index over all sequences (the longest rows first,
//     so the last CTAs to start are the short ones), found by a binary search on sum_s max(0, pairs_s - p);
//   - masks: a tile past a row's position is masked by comparison, so tiles need no alignment with the lengths;
//   - a V row that some row of the pair does not see would still meet that row's P = 0, and 0 * NaN is NaN.  Warps 2 and 3
//     go over the V tiles that hold such rows (the last one to three of a pair) before the MMA reads them: rows of the
//     next sequence are cleared, and a non-finite value within the sequence is cleared and noted per column with its first
//     key; the epilogue adds it to the rows that do see it.  The scan overlaps S = Q K^T and the first softmax.
// P is rounded to the inputs' 16-bit type for the tensor core (half a step, 2^-9 of each weight for bf16, 2^-12 for fp16),
// as the prefill program does; z, m, l and O are fp32.
#pragma once
#include "attention.cuh"

namespace ptsim {

constexpr int kPackRows = 256;                       // query rows of a CTA
constexpr int kPackThreads = 384;
constexpr int kPackRegs0 = 56, kPackRegs1 = 224;     // registers a thread: first warpgroup, softmax warpgroups
static_assert(128 * kPackRegs0 + 256 * kPackRegs1 <= kPackThreads * 168, "register split above the launch's registers");
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

template <int D>
constexpr int packed_smem(int seqs) {
  return 6 * 128 * D * 2 + 1024 + 256 + 3 * D * 4 + seqs * 4;
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

template <int D, bool F16>
__global__ void __launch_bounds__(kPackThreads, 1) packed_attn_kernel(const __grid_constant__ PackedArgs g) {
  constexpr int kTile = 128 * D * 2;                 // bytes of a [128 x D] operand tile: D / 64 swizzled halves of 16 KB
  constexpr int kHalf = 128 * 64 * 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem, *sK = smem + 2 * kTile, *sV = smem + 4 * kTile;   // Q_A, Q_B; K and V two stages each
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + 6 * kTile);
  uint64_t *q_full = bars + 0;
  uint64_t *k_full = bars + 1, *v_full = bars + 3;   // 2 each
  uint64_t *k_empty = bars + 5, *v_empty = bars + 7; // 2 each
  uint64_t *s_full = bars + 9, *o_done = bars + 11;  // [A, B]
  uint64_t *p_full = bars + 13;                      // [A, B], one arrival per softmax warp
  uint64_t *v_clean = bars + 15;                     // 2, one arrival per scanning warp
  uint64_t *scanned = bars + 17;                     // the same, once, after the last scan
  uint64_t *drain = bars + 18;
  uint64_t *scan_full = bars + 19;                   // 2: v_full of the tiles that are scanned
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 21);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  volatile int *dirty = abort_flag + 1;              // a noted non-finite value of V
  int32_t *noted = reinterpret_cast<int32_t *>(smem + 6 * kTile + 256);   // first key of NaN, +inf, -inf: [3][D]
  int32_t *pairs = noted + 3 * D;                    // 256-row tiles of each sequence

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t wl = g.stall ? kTestWaitUs : kWaitUs;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 21; ++i)
      sm100::mbar_init(&bars[i], (i == 13 || i == 14) ? 4u : (i >= 15 && i <= 17) ? 2u : 1u);
    *abort_flag = 0;
    *dirty = 0;
    sm100::fence_barrier_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, 512);
    sm100::tmem_relinquish();
  }
  for (int i = threadIdx.x; i < 3 * D; i += kPackThreads) noted[i] = kPackNever;
  pdl_enter();   // set-up above overlaps the previous kernel's tail; global memory after
  for (int s = threadIdx.x; s < g.seqs; s += kPackThreads) {
    const int q0 = g.cuq[s], q1 = g.cuq[s + 1], k0 = g.cuk[s], k1 = g.cuk[s + 1];
    const bool good = q0 >= 0 && q1 >= q0 && q1 <= g.q_tokens && k0 >= 0 && k1 >= k0 && k1 <= g.k_tokens;
    if (!good) record_status(PTSIM_E_OOB);
    pairs[s] = good ? int(ceil_div(q1 - q0, kPackRows)) : 0;
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // This CTA's pair: item i of the pairs in descending row index p, sequences in order for equal p.  Every warp searches.
  const int item = int(blockIdx.x) / g.hq, head = int(blockIdx.x) % g.hq;
  int p = -1, seq = 0;
  {
    // past(x) = the pairs with index >= x, over all sequences; the largest p with past(p) > item.
    auto past = [&](int x) {
      int n = 0;
      for (int s = lane; s < g.seqs; s += 32) n += max(0, pairs[s] - x);
      return __reduce_add_sync(0xffffffffu, n);
    };
    int most = 0;
    for (int s = lane; s < g.seqs; s += 32) most = max(most, pairs[s]);
    most = __reduce_max_sync(0xffffffffu, most);
    if (past(0) > item) {
      int lo = 0, hi = most;               // past(lo) > item >= past(hi)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (past(mid) > item) lo = mid;
        else hi = mid;
      }
      p = lo;
      int left = item - past(p + 1);       // the left-th sequence with more than p pairs
      for (int s0 = 0; s0 < g.seqs; s0 += 32) {
        const uint32_t has = __ballot_sync(0xffffffffu, s0 + lane < g.seqs && pairs[s0 + lane < g.seqs ? s0 + lane : 0] > p);
        const int n = __popc(has);
        if (left < n) {
          seq = s0 + __fns(has, 0, left + 1);
          break;
        }
        left -= n;
      }
    }
  }
  if (p < 0) {                             // the bound's spare CTAs (every thread of the CTA)
    if (warp == 1) sm100::tmem_dealloc(tmem, 512);
    return;
  }
  const int q0 = g.cuq[seq], ql = g.cuq[seq + 1] - q0;
  const int k0 = g.cuk[seq], kl = g.cuk[seq + 1] - k0;
  const int row0 = p * kPackRows, pos0 = row0 + kl - ql;                  // row 0 of tile A and its position
  const int rows_a = min(128, ql - row0), rows_b = max(0, min(128, ql - row0 - 128));
  const int nA = max(0, (pos0 + rows_a + 127) >> 7);                      // key tiles that some row sees
  const int nB = rows_b > 0 ? max(0, (pos0 + 128 + rows_b + 127) >> 7) : 0;
  const int n = max(nA, nB);
  const int first_scan = pos0 < 0 ? 0 : (pos0 + 1) >> 7;                  // tiles from here hold keys past row 0's position

  int kj = 0, vj = 0;   // (producer) K and V tiles whose stages were armed
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPackRegs0));
    if (warp == 0) {
      if (lane == 0 && n > 0) {
        const int kvh = head / g.per;
        sm100::mbar_arrive_expect_tx(q_full, rows_b > 0 ? 2 * kTile : kTile);
        for (int t = 0; t < (rows_b > 0 ? 2 : 1); ++t)
          for (int c = 0; c < D / 64; ++c)
            sm100::tma_load_3d(sQ + t * kTile + c * kHalf, &g.tq, q_full, c * 64, q0 + row0 + t * 128, head);
        for (int j = 0; j < n; ++j) {
          const int st = j & 1;
          if (!sm100::mbar_wait(&k_empty[st], ((j >> 1) & 1) ^ 1, wl)) { *abort_flag = 1; break; }
          sm100::mbar_arrive_expect_tx(&k_full[st], kTile);
          if (!(g.stall && blockIdx.x == 0 && j == 0))   // test hook: K_0 armed, no copy in flight
            for (int c = 0; c < D / 64; ++c)
              sm100::tma_load_3d(sK + st * kTile + c * kHalf, &g.tk, &k_full[st], c * 64, k0 + j * 128, kvh);
          ++kj;
          if (!sm100::mbar_wait(&v_empty[st], ((j >> 1) & 1) ^ 1, wl)) { *abort_flag = 1; break; }
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
          const uint32_t k_addr = sm100::smem_u32(sK + (j & 1) * kTile), q_addr = sm100::smem_u32(sQ + t * kTile);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
            sm100::mma_bf16_ss(tmem + t * 128, sm100::sw128_desc(q_addr + off, 16, 1024),
                               sm100::sw128_desc(k_addr + off, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
          }
          sm100::mma_commit(&s_full[t]);
        };
        auto issue_pv = [&](int t, int j) {
          const uint32_t v_addr = sm100::smem_u32(sV + (j & 1) * kTile);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            sm100::mma_bf16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8,
                               sm100::sw128_desc(v_addr + k * 16 * 128, kHalf, 1024), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
          if (j == (t == 0 ? nA : nB) - 1) sm100::mma_commit(&o_done[t]);
        };
        // S_X(j + 1) overwrites P_X(j) in TMEM only after PV_X(j), issued before it, has read it (in-order execution).
        bool ok = sm100::mbar_wait(q_full, 0, wl) && sm100::mbar_wait(&k_full[0], 0, wl);
        if (ok) {
          sm100::tc_fence_after();
          if (nA > 0) issue_s(0, 0);
          if (nB > 0) issue_s(1, 0);
          sm100::mma_commit(&k_empty[0]);
        }
        for (int j = 0; ok && j < n; ++j) {
          const int st = j & 1;
          // A scanned tile is complete once both scanning warps, which waited for its copies, have let it go.
          ok = j < first_scan ? sm100::mbar_wait(&v_full[st], (j >> 1) & 1, wl)
                              : sm100::mbar_wait(&v_clean[st], ((j - first_scan) >> 1) & 1, wl);
          if (!ok) break;
          if (j < nA) {
            if (!(ok = sm100::mbar_wait(&p_full[0], j & 1, wl))) break;
            sm100::tc_fence_after();
            issue_pv(0, j);
          }
          if (j + 1 < n) {
            if (!(ok = sm100::mbar_wait(&k_full[st ^ 1], ((j + 1) >> 1) & 1, wl))) break;
            sm100::tc_fence_after();
            if (j + 1 < nA) issue_s(0, j + 1);
          }
          if (j < nB) {
            if (!(ok = sm100::mbar_wait(&p_full[1], j & 1, wl))) break;
            sm100::tc_fence_after();
            issue_pv(1, j);
          }
          sm100::mma_commit(&v_empty[st]);
          if (j + 1 < n) {
            if (j + 1 < nB) issue_s(1, j + 1);
            sm100::mma_commit(&k_empty[st ^ 1]);
          }
        }
        if (!ok) *abort_flag = 1;
        sm100::mma_commit(drain);
        sm100::mbar_wait(drain, 0, wl);
      }
    } else {
      // Warps 2 and 3: V rows that some row of the pair does not see (64 threads over 128 rows of D / 8 units).
      const int me = threadIdx.x - 64;
      for (int j = first_scan; j < n; ++j) {
        const int st = j & 1;
        if (*abort_flag || !sm100::mbar_wait(&scan_full[st], ((j - first_scan) >> 1) & 1, wl)) { *abort_flag = 1; break; }
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPackRegs1));
    const int t = (warp - 4) >> 2;           // 0: tile A, 1: tile B
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;       // query row within the tile = TMEM lane
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    const int ntiles = t == 0 ? nA : nB, rows = t == 0 ? rows_a : rows_b;
    const int pos = pos0 + t * 128 + r;
    const int masked_from = pos0 + t * 128 < 0 ? 0 : (pos0 + t * 128 + 1) >> 7;   // tiles with keys past row 0 of this tile
    const float kLog2e = 1.4426950408889634f;
    const float sl = g.scale * kLog2e;
    // fp16 weights are kept 2^7 times larger (at most 2^15 with the lazy reference), so that small ones stay normal; l holds the same factor.
    constexpr float kBias = F16 ? 7.0f : 0.0f;
    float m = -INFINITY, l = 0.f;            // m in units of log2
    bool ok = true;
    for (int j = 0; j < ntiles; ++j) {
      if (*abort_flag || !sm100::mbar_wait(&s_full[t], j & 1, wl)) { ok = false; break; }
      sm100::tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) sm100::tmem_ld32(tS + c * 32, v[c]);
      sm100::tmem_wait_ld();
      if (j >= masked_from) {
        const int last = pos - j * 128;      // keys past it become -inf: they never win the maximum and their weight is 0
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int q = 0; q < 32; ++q)
            if (c * 32 + q > last) v[c][q] = 0xff800000u;
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
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float2 u = __ffma2_rn(make_float2(__uint_as_float(v[c][2 * q]), __uint_as_float(v[c][2 * q + 1])), a2, b2);
          const float p0 = ex2_fast(u.x), p1 = ex2_fast(u.y);
          acc[q & 3] = __fadd2_rn(acc[q & 3], make_float2(p0, p1));
          pk[q] = pack_16x2<F16>(p0, p1);
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
      sm100::tmem_wait_st();
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&p_full[t]);
    }
    if (rows > 0) {
      if (ok && !*abort_flag && (ntiles == 0 || (sm100::mbar_wait(&o_done[t], 0, wl) && sm100::mbar_wait(scanned, 0, wl)))) {
        sm100::tc_fence_after();
        const float inv = pos < 0 ? 0.f : 1.0f / l;
        uint16_t *orow = g.o + int64_t(q0 + row0 + t * 128 + r) * g.o_row + int64_t(head) * g.o_head;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          if (ntiles > 0) {
            sm100::tmem_ld32(tO + c * 32, v);
            sm100::tmem_wait_ld();
          }
          float x[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) x[q] = pos < 0 ? 0.f : __uint_as_float(v[q]) * inv;   // no key: zeros
          if (*dirty) {
#pragma unroll
            for (int q = 0; q < 32; ++q) {
              const int d = c * 32 + q;
              if (pos >= noted[D + d]) x[q] += INFINITY;
              if (pos >= noted[2 * D + d]) x[q] -= INFINITY;
              if (pos >= noted[d]) x[q] += __uint_as_float(0x7fc00000u);
            }
          }
          if (r < rows)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              reinterpret_cast<uint4 *>(orow + c * 32)[q] =
                  make_uint4(pack_16x2<F16>(x[q * 8], x[q * 8 + 1]), pack_16x2<F16>(x[q * 8 + 2], x[q * 8 + 3]),
                             pack_16x2<F16>(x[q * 8 + 4], x[q * 8 + 5]), pack_16x2<F16>(x[q * 8 + 6], x[q * 8 + 7]));
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
    for (int i = (kj - 2 < 0 ? 0 : kj - 2); i < kj; ++i) sm100::mbar_wait(&k_full[i & 1], (i >> 1) & 1, wl);
    for (int i = (vj - 2 < 0 ? 0 : vj - 2); i < vj; ++i) {
      if (i < first_scan) sm100::mbar_wait(&v_full[i & 1], (i >> 1) & 1, wl);
      else sm100::mbar_wait(&scan_full[i & 1], ((i - first_scan) >> 1) & 1, wl);
    }
  }
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 512);
  }
}

template <int D, bool F16>
static int run_packed(const PackedArgs &g, const LaunchCtx &c) {
  constexpr auto kern = packed_attn_kernel<D, F16>;
  PTSIM_CUDA((smem_limit_once<packed_attn_kernel<D, F16>>(packed_smem<D>(PTSIM_PACKED_SEQS), c.device)));
  // setmaxnreg.inc waits until the registers it asks for are free, so the warpgroups' shares must fit the registers the
  // block is launched with; refuse (rather than wait forever) if the build disagrees.
  static std::atomic<int> regs_ok{0};   // 0 unknown, 1 fits, 2 does not
  if (regs_ok.load() == 0) {
    cudaFuncAttributes fa;
    PTSIM_CUDA(cudaFuncGetAttributes(&fa, kern));
    regs_ok.store(fa.numRegs * kPackThreads >= 128 * kPackRegs0 + 256 * kPackRegs1 ? 1 : 2);
  }
  if (regs_ok.load() != 1) return fail(PTSIM_E_RESOURCE, "attention register split does not fit this build's registers");
  const int64_t grid = (int64_t(g.q_tokens) / kPackRows + g.seqs) * g.hq;
  if (grid >= (int64_t(1) << 31)) return fail(PTSIM_E_UNSUPPORTED, "packed attention over more than 2^31 tiles");
  PTSIM_CUDA(launch_pdl(kern, dim3(unsigned(grid)), dim3(kPackThreads), packed_smem<D>(g.seqs), c.stream, g));
  return PTSIM_OK;
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
