// Page bookkeeping of a paged cache (PTSIM_KIND_PAGES): grow, fork, copy, free, compact.  No counterpart in the reference,
// whose programs hold each tensor whole.
//
// The state is three int32 tensors (table, lens, refs); a page is free where refs is 0, so there is no list of free pages to
// keep and the k-th page a launch takes is the k-th lowest free one: results depend on the state alone.  Everything
// that decides is a few thousand integers, bound by latency, and runs in one CTA (pages_plan_kernel): checks first, then the
// scan of refs that ranks free pages (compaction: holes and movers) by block-wide prefix sums, 4096 pages a step and no
// further than the pages asked for, then the tables, unless a check failed.  What moves bytes, and the rows
// of tables that forks share, is a second kernel over the whole GPU (pages_apply_kernel, a programmatic dependent): a warp per
// 2 KB of a page, four 16-byte loads in flight a lane; its bound is HBM, each moved byte read and written once.  32 forks: 18 us
// for free, plan and copy (14 captured); 56 MB moved by a compaction between a free and a grow: 23 us for the four kernels,
// of which the copy is 14 (its bytes take 9).
#pragma once
#include "common.cuh"

namespace ptsim {

constexpr int kPagesThreads = 1024;
constexpr int kPagesSegment = 2048;   // bytes of a page that a warp copies at once

struct PagesArgs {
  const int32_t *ids, *aux;
  int32_t *table, *lens, *refs;
  uint8_t *pool;
  int32_t *halt;                      // nonzero: change nothing; or null
  int32_t *head, *from, *to, *remap;  // workspace: [0] pages to copy (-1: refused or halted), [1] used pages; [pages] each
  int64_t page_bytes;
  int32_t op, n, slots, pages, page_size, max_pages, layers;
};

// Does the halt word (null: none) stop this launch?  Every launch that it stops records why, so a synchronisation after any of them
// fails.
__device__ __forceinline__ bool halted(const int32_t *halt) {
  const int why = halt == nullptr ? 0 : *halt;
  if (why != 0 && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) record_status(why);
  return why != 0;
}
__device__ __forceinline__ int pages_held(const PagesArgs &g, int len) { return (len + g.page_size - 1) / g.page_size; }
__device__ __forceinline__ bool pages_len_ok(const PagesArgs &g, int len) {
  return len >= 0 && len <= int64_t(g.max_pages) * g.page_size;
}

// Exclusive prefix sum of x over the CTA's 1024 threads; *total gets the sum.  `sums` is 33 shared ints.
__device__ __forceinline__ int block_scan(int x, int *sums, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  __syncthreads();                     // the previous scan's sums have been read
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    sums[lane] = s;
  }
  __syncthreads();
  *total = sums[31];
  return v - x + (warp > 0 ? sums[warp - 1] : 0);
}

// Four consecutive counts from page p (0 past the pool where `past` says used, so a missing page is not free).
__device__ __forceinline__ int4 pages_refs4(const PagesArgs &g, int p) {
  if (p + 3 < g.pages && (reinterpret_cast<uintptr_t>(g.refs) & 15) == 0) return *reinterpret_cast<const int4 *>(g.refs + p);
  return make_int4(p < g.pages ? g.refs[p] : 1, p + 1 < g.pages ? g.refs[p + 1] : 1, p + 2 < g.pages ? g.refs[p + 2] : 1,
                   p + 3 < g.pages ? g.refs[p + 3] : 1);
}

__global__ void __launch_bounds__(kPagesThreads) pages_plan_kernel(const __grid_constant__ PagesArgs g) {
  __shared__ int ids[PTSIM_PAGES_IDS], aux[PTSIM_PAGES_IDS], base[PTSIM_PAGES_IDS], first[PTSIM_PAGES_IDS];
  __shared__ int sums[33], refused;
  __shared__ unsigned long long asked;
  const int i = threadIdx.x;
  if (i == 0) refused = 0, asked = 0;
  pdl_enter();
  if (halted(g.halt)) {
    if (i == 0) g.head[0] = -1;
    return;
  }
  if (g.op == PTSIM_PAGES_COMPACT) {
    // Used pages, then the k-th hole below their number and the k-th used page from it on.
    int used = 0, total;
    for (int p = 4 * i; p < g.pages; p += 4 * kPagesThreads) {
      const int4 r = pages_refs4(g, p);
      used += (r.x > 0) + (p + 1 < g.pages && r.y > 0) + (p + 2 < g.pages && r.z > 0) + (p + 3 < g.pages && r.w > 0);
    }
    block_scan(used, sums, &total);
    const int live = total;
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < g.pages; p0 += 4 * kPagesThreads) {
      const int p = p0 + 4 * i;
      const int4 r = pages_refs4(g, p);
      const int c[4] = {r.x, r.y, r.z, r.w};
      int mine = 0;                    // holes in the low half, movers in the high one (at most 4096 of each a step)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (p + e < g.pages) mine += p + e < live ? (c[e] <= 0 ? 1 : 0) : (c[e] > 0 ? 1 << 16 : 0);
      int at = block_scan(mine, sums, &total);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (p + e < g.pages) {
          if (p + e < live) {
            if (c[e] <= 0) g.to[holes + (at++ & 0xffff)] = p + e;
          } else if (c[e] > 0) {
            g.from[movers + (at >> 16)] = p + e;
            at += 1 << 16;
          } else {
            g.remap[p + e] = p + e;
          }
        }
      holes += total & 0xffff;
      movers += total >> 16;
    }
    __syncthreads();
    for (int k = i; k < movers; k += kPagesThreads) {
      const int a = g.from[k], b = g.to[k];
      g.remap[a] = b;
      g.refs[b] = g.refs[a];
      g.refs[a] = 0;
    }
    if (i == 0) g.head[0] = movers, g.head[1] = live;
    return;
  }

  // Checks; the pages entry i asks for.
  int code = 0, need = 0, len = 0;
  int4 ahead = pages_refs4(g, 4 * i);     // the first 4096 counts come in beside the lists
  if (i < g.n) {
    ids[i] = g.ids[i];
    aux[i] = g.aux[i];
  }
  __syncthreads();
  const bool grow = g.op == PTSIM_PAGES_GROW;
  if (i < g.n) {
    const int a = ids[i], b = aux[i];
    if (a < 0 || a >= g.slots || (!grow && (b < 0 || b >= g.slots))) {
      code = PTSIM_E_OOB;
    } else if (!pages_len_ok(g, len = g.lens[a])) {
      code = PTSIM_E_OOB;
    } else if (grow) {
      const int64_t want = (int64_t(len) + b + g.page_size - 1) / g.page_size;
      if (b < 0) code = PTSIM_E_ARGS;
      else if (want > g.max_pages || int64_t(len) + b > 0x7fffffff) code = PTSIM_E_RESOURCE;
      else need = int(want) - pages_held(g, len);
      first[i] = pages_held(g, len);
    } else {
      if (g.lens[b] != 0) code = PTSIM_E_ARGS;
      first[i] = g.op == PTSIM_PAGES_COPY ? 0 : len / g.page_size;
      need = pages_held(g, len) - first[i];
    }
    for (int j = 0; j < g.n && code == 0; ++j)
      if ((j < i && (grow ? ids[j] == a : aux[j] == b)) || (!grow && ids[j] == b)) code = PTSIM_E_ARGS;
  }
  if (need > 0) atomicAdd(&asked, (unsigned long long)need);      // the scan's 32 bits could wrap
  if (code) atomicOr(&refused, code == PTSIM_E_OOB ? 1 : code == PTSIM_E_ARGS ? 2 : 4);
  int total, found = 0;
  const int at = block_scan(code ? 0 : need, sums, &total);   // its barriers make `refused` everyone's
  if (i < g.n) base[i] = at;
  const bool oob = refused & 1, args = refused & 2;
  bool short_ = (refused & 4) || asked > (unsigned long long)g.pages;
  if (!args && !oob && !short_) {
    // The `total` lowest free pages, in order.
    for (int p0 = 0; p0 < g.pages && found < total; p0 += 4 * kPagesThreads) {
      const int p = p0 + 4 * i;
      const int4 r = ahead;
      if (p0 + 4 * kPagesThreads < g.pages) ahead = pages_refs4(g, p + 4 * kPagesThreads);
      const int c[4] = {r.x, r.y, r.z, r.w};
      int sum, k = found + block_scan((c[0] <= 0) + (c[1] <= 0) + (c[2] <= 0) + (c[3] <= 0), sums, &sum);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c[e] <= 0) {
          if (k < total) g.to[k] = p + e;
          ++k;
        }
      found += sum;
    }
    short_ = found < total;
  }
  if (args || oob || short_) {
    if (i == 0) {
      const int why = oob ? PTSIM_E_OOB : args ? PTSIM_E_ARGS : PTSIM_E_RESOURCE;
      record_status(why);
      if (g.halt != nullptr) *g.halt = why;
      g.head[0] = -1;
    }
    return;
  }
  __syncthreads();
  for (int t = i; t < total; t += kPagesThreads) {
    int lo = 0, hi = g.n;              // the last entry with base <= t (entries that need nothing share their base with the next)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (base[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int64_t place = first[lo] + (t - base[lo]);
    const int page = g.to[t];
    if (!grow) {
      const int src = g.table[int64_t(ids[lo]) * g.max_pages + place];
      const bool good = src >= 0 && src < g.pages;
      if (!good) record_status(PTSIM_E_OOB);
      g.from[t] = good ? src : -1;
    }
    g.table[int64_t(grow ? ids[lo] : aux[lo]) * g.max_pages + place] = page;
    g.refs[page] = 1;
  }
  if (i < g.n) g.lens[grow ? ids[i] : aux[i]] = grow ? len + aux[i] : len;
  if (i == 0) g.head[0] = total;
}

__global__ void __launch_bounds__(256) pages_apply_kernel(const __grid_constant__ PagesArgs g) {
  pdl_enter();
  const int count = g.head[0];
  if (count < 0) return;
  if (g.op == PTSIM_PAGES_COMPACT) {
    const int live = g.head[1];
    for (int64_t s = blockIdx.x; s < g.slots; s += gridDim.x) {
      const int len = g.lens[s];
      if (!pages_len_ok(g, len)) {
        if (threadIdx.x == 0) record_status(PTSIM_E_OOB);
        continue;
      }
      int32_t *row = g.table + s * g.max_pages;
      for (int k = threadIdx.x; k < pages_held(g, len); k += 256) {
        const int p = row[k];
        if (p < 0 || p >= g.pages) record_status(PTSIM_E_OOB);
        else if (p >= live) row[k] = g.remap[p];
      }
    }
  } else if (g.op == PTSIM_PAGES_FORK) {
    // Full pages, counted once more, 1024 entries of one target at a time.
    const int segments = int(ceil_div(g.max_pages, 1024));
    for (int64_t u = blockIdx.x; u < int64_t(g.n) * segments; u += gridDim.x) {
      const int i = int(u / segments), full = g.lens[g.ids[i]] / g.page_size, k0 = int(u % segments) * 1024;
      const int32_t *src = g.table + int64_t(g.ids[i]) * g.max_pages;
      int32_t *dst = g.table + int64_t(g.aux[i]) * g.max_pages;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = k0 + e * 256 + int(threadIdx.x);
        if (k >= full) continue;
        const int p = src[k];
        dst[k] = p;
        if (p >= 0 && p < g.pages) atomicAdd(&g.refs[p], 1);
        else record_status(PTSIM_E_OOB);
      }
    }
  }
  const int lane = threadIdx.x & 31;
  const int64_t segments = ceil_div(g.page_bytes, kPagesSegment), units = int64_t(count) * g.layers * segments;
  for (int64_t u = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); u < units; u += int64_t(gridDim.x) * 8) {
    const int k = int(u / (segments * g.layers));
    const int64_t rest = u % (segments * g.layers), layer = rest / segments, off = rest % segments * kPagesSegment + lane * 16;
    const int a = g.from[k], b = g.to[k];
    if (a < 0) continue;
    const uint8_t *src = g.pool + (layer * g.pages + a) * g.page_bytes + off;
    uint8_t *dst = g.pool + (layer * g.pages + b) * g.page_bytes + off;
    uint4 w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (off + e * 512 < g.page_bytes) w[e] = *reinterpret_cast<const uint4 *>(src + e * 512);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (off + e * 512 < g.page_bytes) *reinterpret_cast<uint4 *>(dst + e * 512) = w[e];
  }
}

// One CTA per listed slot.
__global__ void __launch_bounds__(256) pages_free_kernel(const __grid_constant__ PagesArgs g) {
  pdl_enter();
  if (halted(g.halt)) return;
  const int id = g.ids[blockIdx.x];
  bool again = false;
  for (int j = threadIdx.x; j < int(blockIdx.x); j += 256) again |= g.ids[j] == id;
  if (id < 0 || id >= g.slots) {
    if (threadIdx.x == 0) record_status(PTSIM_E_OOB);
    return;
  }
  if (__syncthreads_or(again)) return;
  const int len = g.lens[id];
  if (!pages_len_ok(g, len)) {
    if (threadIdx.x == 0) record_status(PTSIM_E_OOB);
    return;
  }
  int32_t *row = g.table + int64_t(id) * g.max_pages;
  for (int k = threadIdx.x; k < pages_held(g, len); k += 256) {
    const int p = row[k];
    if (p >= 0 && p < g.pages) atomicSub(&g.refs[p], 1);
    else record_status(PTSIM_E_OOB);
    row[k] = -1;
  }
  __syncthreads();                     // every thread has read the length
  if (threadIdx.x == 0) g.lens[id] = 0;
}

int64_t pages_workspace(const ptsim_desc &d) {
  return d.p.pages.op == PTSIM_PAGES_FREE ? 0 : 4 * (4 + 3 * d.p.pages.pages);
}

int launch_pages(const ptsim_desc &d, void *const *ptrs, void *ws, size_t ws_bytes, const LaunchCtx &c) {
  const ptsim_pages_params &p = d.p.pages;
  if (p.op != PTSIM_PAGES_COMPACT && p.n == 0) return PTSIM_OK;
  PagesArgs g;
  memset(&g, 0, sizeof(g));
  auto ints = [&](int arg) { return arg < 0 ? nullptr : static_cast<int32_t *>(ptrs[arg]); };
  g.ids = ints(p.ids_arg);
  g.aux = ints(p.aux_arg);
  g.table = ints(p.table_arg);
  g.lens = ints(p.lens_arg);
  g.refs = ints(p.refs_arg);
  g.pool = p.pool_arg < 0 ? nullptr : static_cast<uint8_t *>(ptrs[p.pool_arg]);
  g.halt = ints(p.halt_arg_p1 - 1);
  if (reinterpret_cast<uintptr_t>(g.pool) % 16 != 0) return fail(PTSIM_E_ARGS, "the pool is not 16-byte aligned");
  g.page_bytes = p.page_bytes;
  g.op = p.op;
  g.n = int(p.n);
  g.slots = int(p.slots);
  g.pages = int(p.pages);
  g.page_size = int(p.page_size);
  g.max_pages = int(p.max_pages);
  g.layers = int(p.layers);
  if (p.op == PTSIM_PAGES_FREE) {
    PTSIM_CUDA(launch_pdl(pages_free_kernel, dim3(unsigned(p.n)), dim3(256), 0, c.stream, g));
    return PTSIM_OK;
  }
  const int64_t need = pages_workspace(d);
  if (ws == nullptr || int64_t(ws_bytes) < need)
    return fail(PTSIM_E_RESOURCE, "page bookkeeping needs %lld bytes of workspace, got %zu", (long long)need, ws_bytes);
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0) return fail(PTSIM_E_ARGS, "workspace is not 16-byte aligned");
  g.head = static_cast<int32_t *>(ws);
  g.from = g.head + 4;
  g.to = g.from + g.pages;
  g.remap = g.to + g.pages;
  PTSIM_CUDA(launch_pdl(pages_plan_kernel, dim3(1), dim3(kPagesThreads), 0, c.stream, g));
  if (p.op != PTSIM_PAGES_GROW)
    PTSIM_CUDA(launch_pdl(pages_apply_kernel, dim3(unsigned(c.sm_count * 4)), dim3(256), 0, c.stream, g));
  return PTSIM_OK;
}

}  // namespace ptsim
