// Paged key / value cache: the step plan (block tables, positions, slot map), the scatter of new rows into pages, and
// attention of the new rows over their sequences' pages.
//
// A pool holds pages [num_pages, Hkv, page_size, D] per layer for keys and for values; a sequence's pages are the ids in
// its row of the block table.  Bad ids, slots and lengths come from the device and cannot be refused on the host: the
// kernels check every index before they use it, skip the access and set kStatusPagePlanInvalid.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda.h>

#include <atomic>

#include "common.cuh"
#include "tc.cuh"

namespace tb200 {
int* status_word_ptr();

namespace paged {

constexpr int kMaxSeqs = 4096;          // sequences of one step: their offsets live in shared memory
constexpr int kMaxSlots = 65536;        // rows of the block table: one bit each in shared memory
constexpr int kMaxCols = 1 << 20;       // columns of the block table and rows of a step: a block's scan stays inside 32 bits
constexpr int kMaxRows = 1 << 22;
constexpr int kMaxLength = 1 << 30;     // tokens of one sequence
constexpr int kMaxLine = 1 << 30;       // tiles of a step over all key heads
constexpr int kMinTiles = 2;            // a CTA's stretch is at least this long: shorter ones cost more to join than they save

// Inclusive scan over the block; `part` needs 33 entries.
__device__ __forceinline__ int block_scan(int v, int* part, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int p = lane < n ? part[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += u;
    }
    part[lane] = p;
  }
  __syncthreads();
  total = part[n - 1];
  return v + (warp > 0 ? part[warp - 1] : 0);
}

// Largest i in [0, n) with start[i] <= x, where start[0] = 0 <= x < start[n].
__device__ __forceinline__ int find_segment(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The same by a whole warp: 32 probes at a time, so one round of dependent loads per factor of 32.
__device__ __forceinline__ int find_segment_warp(const int* start, int n, int x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && start[at] <= x);
    const int k = 31 - __clz((int)below);        // lane 0 is always below
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

struct PlanParams {
  const int *cached, *fresh, *slots, *pages, *mapped;   // [B], [B], [B], [F], [B] or null
  int* table;                                           // [S, W]
  int B, S, W, F, ps, R, num_pages;
  int* row_start;                                       // [B + 1]
  int64_t *positions, *slot_map;                        // [R]
  int* status;
};

// Every block scans the (few) request lengths itself, so that no block waits for another, and then writes its share of
// the rows and of the newly handed out table entries.  A page that is needed for a row of this step is taken from the
// hand-out list, not from the table, which another block may still be writing.  Latency bound: a launch, one scan and
// one round of dependent loads: 6 us for 9 sequences, 8 us for 500 sequences with 50 thousand rows, launch included.
// The work list (work_kernel) is a launch of its own per step and window.
__global__ void __launch_bounds__(256) plan_kernel(const PlanParams p) {
  extern __shared__ int sm[];
  int* row_start = sm;                 // [B + 1]
  int* page_start = sm + p.B + 1;      // [B + 1]
  unsigned* seen = reinterpret_cast<unsigned*>(sm + 2 * (p.B + 1));   // bit per slot (block 0)
  __shared__ int part[33];
  bool bad = false;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < (p.S + 31) / 32; i += blockDim.x) seen[i] = 0u;
  __syncthreads();
  int rows = 0, need_sum = 0;
  for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    int n = 0, need = 0;
    if (b < p.B) {
      const int slot = p.slots[b], c = p.cached[b];
      n = p.fresh[b];
      if (c < 0 || c > kMaxLength || n < 0 || slot < 0 || slot >= p.S) {
        bad = true;
        n = 0;
      } else {
        const int64_t end = ((int64_t)c + n + p.ps - 1) / p.ps;
        const int have = p.mapped != nullptr ? max(0, p.mapped[b]) : (int)(((int64_t)c + p.ps - 1) / p.ps);
        bad |= end > p.W || (p.mapped != nullptr && p.mapped[b] < 0);
        need = (int)max((int64_t)0, min(end, (int64_t)p.W) - have);
        if (blockIdx.x == 0) bad |= (atomicOr(&seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31)) & 1u;   // the same slot twice
      }
      bad |= n > p.R;
      n = min(n, p.R);
    }
    int t1, t2;
    const int e1 = block_scan(n, part, t1);
    const int e2 = block_scan(need, part, t2);
    if (b < p.B) {
      row_start[b] = min(rows + e1 - n, p.R);
      page_start[b] = need_sum + e2 - need;
    }
    bad |= rows + t1 > p.R;
    rows = min(rows + t1, p.R);          // rows past the caller's count are left out
    need_sum = min(need_sum + t2, 1 << 30);   // beyond any hand-out list: only device data that is flagged gets there
  }
  if (threadIdx.x == 0) {
    row_start[p.B] = rows;
    page_start[p.B] = need_sum;
  }
  bad |= need_sum > p.F;
  __syncthreads();
  const int tid = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  for (int e = tid; e < need_sum; e += step) {
    const int b = find_segment(page_start, p.B, e);
    const int have = p.mapped != nullptr ? max(0, p.mapped[b]) : (p.cached[b] + p.ps - 1) / p.ps;
    int page = e < p.F ? p.pages[e] : -1;
    if (page < 0 || page >= p.num_pages) {
      page = -1;
      bad = true;
    }
    p.table[(int64_t)p.slots[b] * p.W + have + e - page_start[b]] = page;
  }
  for (int r = tid; r < p.R; r += step) {
    int64_t pos = 0, slot = -1;
    if (r < rows) {
      const int b = find_segment(row_start, p.B, r);
      pos = (int64_t)p.cached[b] + r - row_start[b];
      const int64_t col = pos / p.ps;
      if (col < p.W) {
        const int have = p.mapped != nullptr ? max(0, p.mapped[b]) : (p.cached[b] + p.ps - 1) / p.ps;
        const int64_t e = page_start[b] + col - have;
        const int page = col < have ? p.table[(int64_t)p.slots[b] * p.W + col] : (e < p.F ? p.pages[e] : -1);
        if (page >= 0 && page < p.num_pages) slot = (int64_t)page * p.ps + pos % p.ps;
        else bad = true;
      }
    }
    p.positions[r] = pos;
    p.slot_map[r] = slot;
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= p.B; b += blockDim.x) p.row_start[b] = row_start[b];
  if (bad) atomicOr(p.status, kStatusPagePlanInvalid);
}

// ----------------------------------------------------------------------------------------------------------------- write
struct WriteParams {
  const char *k, *v;                      // [T, H, D], strides in bytes
  int64_t k_row, k_head, v_row, v_head;
  char *kp, *vp;                          // [num_pages, H, page_size, D], strides in bytes
  int64_t kp_page, kp_head, kp_slot, vp_page, vp_head, vp_slot;
  const int64_t* slot_map;
  int64_t T, num_slots;
  int H, vecs, ps;                        // vecs: 16-byte vectors per head
  int* status;
};

// A copy: one 16-byte vector of a key and of the value beside it per thread and step.  16001 rows of 8 heads of 128: 25 us
// for 131 MB (5.3 TB/s).
__global__ void __launch_bounds__(256) write_kernel(const WriteParams p) {
  const int per_row = p.H * p.vecs;
  const int64_t total = p.T * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / per_row;
    const int c = (int)(i % per_row);
    const int h = c / p.vecs, v = c % p.vecs;
    const int64_t slot = p.slot_map[t];
    if (slot < 0 || slot >= p.num_slots) {
      if (slot != -1) atomicOr(p.status, kStatusPagePlanInvalid);
      continue;
    }
    const int64_t page = slot / p.ps;
    const int off = (int)(slot % p.ps);
    const uint4 a = *reinterpret_cast<const uint4*>(p.k + t * p.k_row + h * p.k_head + v * 16);
    const uint4 b = *reinterpret_cast<const uint4*>(p.v + t * p.v_row + h * p.v_head + v * 16);
    *reinterpret_cast<uint4*>(p.kp + page * p.kp_page + h * p.kp_head + off * p.kp_slot + v * 16) = a;
    *reinterpret_cast<uint4*>(p.vp + page * p.vp_page + h * p.vp_head + off * p.vp_slot + v * 16) = b;
  }
}

// ------------------------------------------------------------------------------------------------------------- attention
// Work.  A *source* is a set of neighbouring rows that all look at one key range of one table row: the rows of a sequence
// on what follows its group's prefix, or all rows of a group on the prefix.  Its (row, query head of one key head) pairs
// are cut into *units*, a unit's keys into tiles.  The tiles of all units and key heads form one line that is cut into
// equal stretches, one per CTA, whatever the lengths are: a CTA works through the *pieces* of units that fall into its
// stretch.  A piece that covers its unit is finished where it is; the others leave (max, sum, unnormalised fp32 output)
// behind, at most two per CTA (the first and the last of a stretch), which the finish kernel joins in the order of the
// line, so results do not depend on scheduling.  A group's two sources are joined there as well.
//
// There are two lists with a line each: units of 16 pairs for the kernel on mma.sync, units of up to 128 pairs (whole rows)
// for the one on tcgen05, both with 64-key tiles.  A source of more than kFewPairs pairs is *large*: it is in both lists,
// behind the small ones in the first, and runs from the second where that kernel is launched.  A 16-pair unit is the most
// that reads its keys once on the first kernel; beyond it each further unit reads them again, which the second kernel
// does not: 32 sequences of 4000 tokens, 8 key heads of 128, 4 / 12 / 20 / 32 / 64 / 128 pairs a key head: 111 / 115 / 195 /
// 197 / 319 / 638 us on the first, 125 / 125 / 131 / 135 us from 20 pairs on the second (floor 80 us).
constexpr int kRowsA = 16, kTileA = 64;
constexpr int kRowsB = 128, kTileB = 64;
constexpr int kFewPairs = 16;

struct __align__(16) Unit {
  int row0, pairs, pair0, slot;                  // first row and pair count of the source, first pair of the unit, table row
  int key_lo, key_hi, base, shared;              // keys [lo, hi); position of the source's first row, or -1 for a prefix;
                                                 // number of that row among the rows of sharing groups, -1 = not one
};

// Layout of the int32 work buffer (one per window), from the sizes that the host knows.
struct WorkLayout {
  int64_t seq_group, shared, group_row, src_a, src_b, tiles_a, tiles_b, units_a, units_b, size;
  // header: [0, 1] units and tiles (of one key head) of the small sources in list A, [2, 3] of all, [4, 5] of list B, [6] whether
  // a sequence that shares nothing has several rows
  __host__ __device__ WorkLayout(int64_t B, int64_t NG, int64_t max_a, int64_t max_b) {
    seq_group = 8;
    shared = seq_group + B;                      // rows of the groups that share, as running counts
    group_row = shared + NG + 1;                 // first row of each group
    src_a = group_row + NG;                      // first unit of each source, -1 = none
    src_b = src_a + B + NG;
    tiles_a = src_b + B + NG;                    // running tile counts
    tiles_b = tiles_a + max_a + 1;
    units_a = (tiles_b + max_b + 1 + 3) / 4 * 4;
    units_b = units_a + 8 * max_a;
    size = units_b + 8 * max_b;
  }
};

struct WorkParams {
  const int *cached, *row_start, *slots, *group_start, *group_prefix;
  int B, NG, W, ps, G, Hkv, window, max_a, max_b, rows_b;   // rows_b: token rows of a unit in list B
  int max_shared;                                // rows of sharing groups that the caller has room for
  int* work;
  int* status;
};

// One block, because a unit's place follows from a scan over all sources and then all units; latency bound.  Device time of a
// replayed graph beside the tables' kernel: 4 us for 9 or 61 single rows, 10 us for 4 prefixes of 16 sequences, 24 us for a
// prompt of 32768 rows (8200 units of 16 pairs), 39 us for 500 sequences of up to 200 rows.
__global__ void __launch_bounds__(1024) work_kernel(const WorkParams p) {
  extern __shared__ int sm[];
  const int n_src = p.B + p.NG;
  int* start = sm;                               // [n_src + 1] first unit of each source in the list at hand
  int* prefix = start + n_src + 1;               // [NG] tokens of the group's prefix, as used
  int* leader = prefix + p.NG;                   // [NG] first sequence with rows
  __shared__ int part[33];
  const WorkLayout lay(p.B, p.NG, p.max_a, p.max_b);
  int* seq_group = p.work + lay.seq_group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool bad = false;
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) seq_group[b] = -1;
  __syncthreads();
  // groups: one warp each.  The prefix ends at the shortest member, and a group with one live sequence shares nothing.
  for (int g = warp; g < p.NG; g += blockDim.x / 32) {
    const int a = min(max(p.group_start[g], 0), p.B), e = min(max(p.group_start[g + 1], a), p.B);
    bad |= a != p.group_start[g] || e != p.group_start[g + 1];
    int live = 0, shortest = INT_MAX, first = INT_MAX;
    for (int b = a + lane; b < e; b += 32) {
      if (p.row_start[b + 1] == p.row_start[b]) continue;
      ++live;
      shortest = min(shortest, p.cached[b]);
      first = min(first, b);
    }
    live = __reduce_add_sync(0xffffffffu, live);
    shortest = __reduce_min_sync(0xffffffffu, shortest);
    first = __reduce_min_sync(0xffffffffu, first);
    const int use = live > 1 ? max(0, min(p.group_prefix[g], shortest)) : 0;
    if (lane == 0) { prefix[g] = use; leader[g] = first; }
    if (use > 0)
      for (int b = a + lane; b < e; b += 32) seq_group[b] = g;
  }
  // Offsets out of order are flagged and nothing is shared: a sequence of two groups would be joined twice, and running
  // row counts would leave 32 bits.
  if (__syncthreads_or(bad)) {
    for (int g = threadIdx.x; g < p.NG; g += blockDim.x) prefix[g] = 0;
    for (int b = threadIdx.x; b < p.B; b += blockDim.x) seq_group[b] = -1;
    __syncthreads();
  }
  {
    int* shared = p.work + lay.shared;           // running row counts of the groups that share a prefix
    int rows = 0, kept = 0;
    for (int g0 = 0; g0 < p.NG; g0 += blockDim.x) {
      const int g = g0 + threadIdx.x;
      int n = 0, a = 0, e = 0;
      if (g < p.NG) {
        a = min(max(p.group_start[g], 0), p.B);
        e = min(max(p.group_start[g + 1], 0), p.B);
        if (prefix[g] > 0) n = max(0, p.row_start[e] - p.row_start[a]);
        p.work[lay.group_row + g] = p.row_start[a];
      }
      int total;
      const int upto = rows + block_scan(n, part, total);
      rows += total;
      if (upto > p.max_shared && n > 0) {        // no room: the group is attended to without sharing
        n = 0;
        prefix[g] = 0;
        for (int b = a; b < e; ++b) seq_group[b] = -1;
      }
      const int upto_kept = kept + block_scan(n, part, total);
      if (g < p.NG) shared[g] = upto_kept - n;
      kept += total;
    }
    if (threadIdx.x == 0) shared[p.NG] = kept;
  }
  bool several = false;
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) several |= p.row_start[b + 1] - p.row_start[b] > 1 && seq_group[b] < 0;
  several = __syncthreads_or(several);
  if (threadIdx.x == 0) p.work[6] = several;
  auto source_rows = [&](int s, int& r0, int& r1) {
    if (s < p.B) {
      r0 = p.row_start[s];
      r1 = p.row_start[s + 1];
    } else {
      const int g = s - p.B;
      r0 = r1 = 0;
      if (prefix[g] > 0) {
        r0 = p.row_start[min(max(p.group_start[g], 0), p.B)];
        r1 = p.row_start[min(max(p.group_start[g + 1], 0), p.B)];
      }
    }
  };
  int *src_a = p.work + lay.src_a, *src_b = p.work + lay.src_b, *tiles_a = p.work + lay.tiles_a, *tiles_b = p.work + lay.tiles_b;
  Unit *units_a = reinterpret_cast<Unit*>(p.work + lay.units_a), *units_b = reinterpret_cast<Unit*>(p.work + lay.units_b);
  // Appends the units of the small or the large sources to a list that has `n0` units and `t0` tiles already.
  auto list = [&](bool large, int rows, int tile, int max_units, int* src, int* tiles, Unit* units, int& n0, int& t0) {
    int n_units = 0;
    for (int s0 = 0; s0 < n_src; s0 += blockDim.x) {
      const int s = s0 + threadIdx.x;
      int n = 0;
      bool mine = false;
      if (s < n_src) {
        int r0, r1;
        source_rows(s, r0, r1);
        const int64_t pairs = (int64_t)max(0, r1 - r0) * p.G;
        mine = (pairs > kFewPairs) == large;
        if (mine) n = (int)((pairs + rows - 1) / rows);
      }
      int total;
      const int e = block_scan(n, part, total);
      if (s < n_src) {
        start[s] = n_units + e - n;
        if (mine) src[s] = n > 0 ? n0 + n_units + e - n : -1;
        else if (src == src_b) src[s] = -1;
      }
      n_units += total;
    }
    if (threadIdx.x == 0) start[n_src] = n_units;
    if (n_units > max_units - n0) {              // no step comes near: a row belongs to at most two sources
      bad = true;
      n_units = max_units - n0;
    }
    __syncthreads();
    int n_tiles = 0;
    for (int u0 = 0; u0 < n_units; u0 += blockDim.x) {
      const int u = u0 + threadIdx.x;
      int n = 0;
      if (u < n_units) {
        const int s = find_segment(start, n_src, u);
        int r0, r1;
        source_rows(s, r0, r1);
        Unit w;
        w.row0 = r0;
        w.pairs = (r1 - r0) * p.G;
        w.pair0 = (u - start[s]) * rows;
        const int last = min(w.pair0 + rows, w.pairs) - 1;
        const int64_t room = (int64_t)p.W * p.ps;
        if (s < p.B) {
          const int g = seq_group[s], c = p.cached[s];
          w.slot = p.slots[s];
          w.base = c;
          w.shared = g < 0 ? -1 : p.work[lay.shared + g] + r0 - p.work[lay.group_row + g];
          w.key_lo = g < 0 ? 0 : prefix[g];
          if (p.window > 0) w.key_lo = max(w.key_lo, c + w.pair0 / p.G - p.window + 1);
          w.key_hi = (int)min((int64_t)c + last / p.G + 1, room);
        } else {
          const int g = s - p.B;
          w.slot = p.slots[min(leader[g], p.B - 1)];
          w.base = -1;
          w.shared = p.work[lay.shared + g];
          // the smallest position of the group's rows bounds the window of all of them
          int from = 0;
          if (p.window > 0) {
            from = INT_MAX;
            const int a = min(max(p.group_start[g], 0), p.B), e = min(max(p.group_start[g + 1], a), p.B);
            for (int b = a; b < e; ++b)
              if (p.row_start[b + 1] > p.row_start[b]) from = min(from, p.cached[b]);
            from = max(0, from - p.window + 1);
          }
          w.key_lo = from;
          w.key_hi = (int)min((int64_t)prefix[g], room);
        }
        n = w.key_hi > w.key_lo ? (w.key_hi - 1) / tile - w.key_lo / tile + 1 : 0;
        if (n > kMaxLine / 1024) {               // a block's scan stays inside 32 bits
          bad = true;
          n = 0;
        }
        units[n0 + u] = w;
      }
      int total;
      const int e = block_scan(n, part, total);
      if (u < n_units) tiles[n0 + u] = t0 + n_tiles + e - n;
      n_tiles = min(n_tiles + total, kMaxLine + 1 - t0);
    }
    if ((t0 + (int64_t)n_tiles) * p.Hkv > kMaxLine) {      // no real step comes near: lengths that are flagged, no work
      bad = true;
      n_units = n_tiles = 0;
    }
    n0 += n_units;
    t0 += n_tiles;
    if (threadIdx.x == 0) tiles[n0] = t0;
    __syncthreads();
  };
  int n = 0, t = 0;
  list(false, kRowsA, kTileA, p.max_a, src_a, tiles_a, units_a, n, t);
  if (threadIdx.x == 0) { p.work[0] = n; p.work[1] = t; }
  list(true, kRowsA, kTileA, p.max_a, src_a, tiles_a, units_a, n, t);
  if (threadIdx.x == 0) { p.work[2] = n; p.work[3] = t; }
  n = t = 0;
  if (p.rows_b > 0) list(true, p.rows_b * p.G, kTileB, p.max_b, src_b, tiles_b, units_b, n, t);
  if (threadIdx.x == 0) { p.work[4] = n; p.work[5] = t; }
  if (bad) atomicOr(p.status, kStatusPagePlanInvalid);
}

// One kernel's view of its list.
struct List {
  const int* tiles;
  const Unit* units;
  int n_units, n_tiles, ctas;
  // Tiles of a CTA's stretch.
  __device__ __forceinline__ int stretch(int Hkv) const { return max(kMinTiles, (n_tiles * Hkv + ctas - 1) / ctas); }
};

// What a CTA leaves for the finish kernel: the unit that its stretch begins and does not end, when it shares nothing.
struct __align__(16) Cut {
  int parts, row0, pairs, pair0, head;
};

struct AttnParams {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  __nv_bfloat16* out;                            // [R, Hq, D]
  const float* sinks;                            // [Hq] or null
  const int *table, *slots, *cached, *row_start, *work;
  const __nv_bfloat16 *kp, *vp;                  // pages; strides in elements
  int64_t kp_page, kp_head, kp_slot, vp_page, vp_head, vp_slot;
  int B, NG, W, R, Hq, Hkv, G, ps, num_pages, window, max_a, max_b, ctas_a, ctas_b, rows_b, ps_shift, max_shared;
  float scale_log2;
  bool zero_tail, use_b;                         // use_b: large sources run on the tcgen05 kernel
  float *part_a, *part_a_ml;                     // [ctas_a, 2, kRowsA, D], [ctas_a, 2, kRowsA, 2]: pieces
  float *part_b, *part_b_ml;                     // [ctas_b, 2, kRowsB, D], [ctas_b, 2, kRowsB, 2]
  float *row_o, *row_ml;                         // [2, max_shared, Hq, D], [.., 2]: whole units of groups (own keys, prefix)
  Cut* cuts;                                     // [ctas_a + ctas_b]
  int* status;

  // Where a whole unit of a group leaves a (row, query head): `pr` pairs behind the source's first; -1 without room.
  __device__ __forceinline__ int64_t shared_at(const Unit& u, int pr, int head) const {
    const int row = u.shared + pr / G;
    return row < max_shared ? ((int64_t)(u.base < 0) * max_shared + row) * Hq + head * G + pr % G : -1;
  }

  // SMs that work on list B while the others work on list A, where both have work: in proportion to the time that the
  // lists take.  In units of an SM's time for a 64-key tile of list A (0.5 us: two CTAs, memory latency) a unit there costs 3
  // more (its queries, its join) and a tile of list B 2 (the issuing thread).  Against one list after the other on all SMs:
  // 4 prefixes of 8192 with 16 sequences of up to 1000 tokens behind each 69.6 -> 61.4 us, 2 of 32768 with 64 of up to 4000
  // behind each 297 -> 262, a prompt of 512 rows beside 60 sequences of up to 8000 tokens 227 -> 209 (L2 cold).  It can lose: 4
  // prefixes of 65536 with 32 sequences behind each 233.5 -> 241.7.  The weights were found with heads of 128.
  __device__ __forceinline__ int sms_b() const {
    const int64_t a = (int64_t)work[1] + 3 * (int64_t)work[0], b = 2 * (int64_t)work[5];
    return work[1] == 0 || b == 0 ? ctas_b : max(1, min(ctas_b - 1, (int)((ctas_b * b + (a + b) / 2) / (a + b))));
  }
  __device__ __forceinline__ List list_a(const WorkLayout& lay) const {
    const int h = use_b ? 0 : 2;
    const int ctas = use_b && work[1] > 0 && work[5] > 0 ? ctas_a / ctas_b * (ctas_b - sms_b()) : ctas_a;      // some per SM
    return {work + lay.tiles_a, reinterpret_cast<const Unit*>(work + lay.units_a), work[h], work[h + 1], ctas};
  }
  __device__ __forceinline__ List list_b(const WorkLayout& lay) const {
    return {work + lay.tiles_b, reinterpret_cast<const Unit*>(work + lay.units_b), work[4], work[5], sms_b()};
  }
};

template <int D>
struct Cfg {
  static constexpr int kStages = D == 64 ? 4 : D == 128 ? 3 : 2;
  static constexpr int kCtasPerSm = D == 256 ? 1 : 2;            // a third CTA or longer rings at 64 gained nothing
  static constexpr uint32_t kHalfBytes = kTileA * D * 2;         // keys (or values) of a tile
  static constexpr uint32_t kStageBytes = 2 * kHalfBytes;
  static constexpr uint32_t kExchange = 2 * kRowsA * D * 4;   // two fp32 output tiles
  static constexpr uint32_t kSmem = kStages * kStageBytes + kExchange + 4 * kRowsA * 2 * 4 + 16 * kStages + 16;
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2bf(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ bool any_nan(const float4& v) { return v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w; }
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The same, true for all when any thread brings true.
__device__ __forceinline__ bool consumer_any(bool v) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.or.pred b, 1, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)v) : "memory");
  return r != 0;
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

// Programmatic launches.  The three kernels of a call are chained: each lets the next one start while it runs, and a
// kernel that needs what came before waits for it here (all memory of the earlier grids is visible then).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A bounded wait whose outcome is the same for all lanes, so that a warp leaves as one.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort_flag));
}

// After an abort, whichever role it came from and however far the producer had got: the copies of the last tiles are waited
// for (with a limit) before the block may end.
template <typename F>
__device__ __forceinline__ void drain(int it, int stages, F full) {
  volatile int quiet = 0;
  for (int j = max(0, it - stages); j < it; ++j) tc::mbar_wait(full(j % stages), (j / stages) & 1, &quiet);
}

// A CTA's walk over its stretch of the line.
struct Walk {
  const int* tiles;
  int Hkv;
  int at, end, per;
  int u, head, first, count;                     // current piece: unit, key head, first tile of the unit, tiles
  int unit_tiles;

  __device__ __forceinline__ Walk(const List& l, int Hkv_, int cta) : tiles(l.tiles), Hkv(Hkv_) {
    const int line = l.n_tiles * Hkv;
    per = l.stretch(Hkv);
    at = (int)min((int64_t)line, (int64_t)cta * per);
    end = min(line, at + per);
    u = at < end ? find_segment_warp(tiles, l.n_units, at / Hkv) : 0;
  }
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    int from = tiles[u], to = tiles[u + 1];
    while (to * Hkv <= at) {
      from = to;
      to = tiles[++u + 1];
    }
    unit_tiles = to - from;
    const int in = at - from * Hkv;
    head = in / unit_tiles;
    first = in - head * unit_tiles;
    count = min(unit_tiles - first, end - at);
    at += count;
    return true;
  }
  // After the last piece of the stretch: how many CTAs the unit is spread over if it begins here and goes on, else 0.
  __device__ __forceinline__ Cut cut(const Unit& unit) const {
    Cut c{0, unit.row0, unit.pairs, unit.pair0, head};
    if (first == 0 && count < unit_tiles && unit.shared < 0) c.parts = 2 + (unit_tiles - count - 1) / per;
    return c;
  }
};

// Few rows (a unit of 16 pairs), bound by the bytes of the keys and values: 16 rows of tensor work per key are far below
// what mma.sync sustains, so the design is about keeping TMA loads in flight.  One producer warp streams 64-key tiles of K
// and V (a 128-byte swizzled box per page) through a ring; each of four consumer warps takes 16 keys of every tile and
// keeps its own running maximum, sum and output in registers, so no warp waits for another inside a piece.  The four are
// joined at the end of a piece.  Two CTAs an SM (10 warps: at most 168 registers a thread, which is what holding the
// queries of the next piece during the join, or joining by halves, would not fit).  One sequence of 100000 tokens, 8 key
// heads of 128: 64 us for 410 MB (6.4 TB/s); 61 sequences of 30 to 8000 tokens: 167 us for 1 GB (6.0 TB/s).
template <int D>
__global__ void __launch_bounds__(160, Cfg<D>::kCtasPerSm)
attn_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const AttnParams p) {
  using C = Cfg<D>;
  using namespace tc;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  float* exch = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
  float* ml = exch + C::kExchange / 4;                                   // [4][kRowsA][2]
  const uint32_t bars = base + C::kStages * C::kStageBytes + C::kExchange + 4 * kRowsA * 2 * 4;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + (bars - base) + 16 * C::kStages);
  auto full = [&](int s) { return bars + 16u * s; };
  auto empty = [&](int s) { return bars + 16u * s + 8u; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_start();
  const List list = p.list_a(WorkLayout(p.B, p.NG, p.max_a, p.max_b));
  if (blockIdx.x > 0 && (int)blockIdx.x >= list.ctas) {           // block 0 waits for the other kernel below in any case
    if (threadIdx.x == 0) p.cuts[blockIdx.x] = Cut{0, 0, 0, 0, 0};
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  Walk walk(list, p.Hkv, blockIdx.x);
  int it = 0;

  if (warp == 4) {
    // ---------------------------------------------------------------------------------------------------- producer
    const int box = min(p.ps, kTileA), subs = kTileA / box;
    const int loads = 2 * subs;                  // at most 8: one lane each
    const int kv = lane / subs, sub = lane % subs;
    const CUtensorMap* map = kv ? &tmap_v : &tmap_k;
    bool ok = true;
    while (ok && walk.next()) {
      const Unit u = list.units[walk.u];
      const int* row = p.table + (int64_t)u.slot * p.W;
      const int t0 = u.key_lo / kTileA + walk.first;
      auto entry = [&](int t) {                  // page of this lane's box of tile t, -1 when no key of it is needed
        const int key = t * kTileA + sub * box;
        return lane < loads && key < u.key_hi ? row[key >> p.ps_shift] : INT_MIN;
      };
      int page = entry(t0), page1 = walk.count > 1 ? entry(t0 + 1) : INT_MIN;
      for (int i = 0; i < walk.count; ++i, ++it) {
        const int st = it % C::kStages;
        const int t = t0 + i;
        const int page2 = i + 2 < walk.count ? entry(t + 2) : INT_MIN;      // fetched two tiles ahead
        if (!warp_wait(empty(st), ((it / C::kStages) & 1) ^ 1, abort_flag)) { ok = false; break; }
        const int need = __popc(__ballot_sync(0xffffffffu, page != INT_MIN));
        if (lane == 0) mbar_expect_tx(full(st), need * box * D * 2);
        __syncwarp();
        if (page != INT_MIN) {
          if (page < 0 || page >= p.num_pages) {  // out of range: the load fills zeros
            atomicOr(p.status, kStatusPagePlanInvalid);
            page = p.num_pages;
          }
          const int key = t * kTileA + sub * box;
          tma_load_5d(base + st * C::kStageBytes + kv * C::kHalfBytes + sub * box * D * 2, map, full(st), 0, key & (p.ps - 1), 0, walk.head, page);
        }
        page = page1;
        page1 = page2;
      }
    }
  } else {
    // ---------------------------------------------------------------------------------------------------- consumers
    const int quad = lane & 3, r_lo = lane >> 2;                         // this thread's rows: r_lo and r_lo + 8
    // a page's box is [64-column block][key][128 bytes]; this warp's 16 keys lie in one box
    const int box = min(p.ps, kTileA);
    const uint32_t block = box * 128, mine = (warp * 16) / box * (box * D * 2) + (warp * 16) % box * 128;
    if (threadIdx.x == 0) p.cuts[blockIdx.x] = Cut{0, 0, 0, 0, 0};       // each piece writes it again
    bool ok = true;
    while (ok && walk.next()) {
      const Unit u = list.units[walk.u];
      // rows: queries as A fragments, visible key range
      uint32_t qf[D / 16][4];
      int lo[2], hi[2];
      int lo_min = INT_MAX, lo_max = 0, hi_min = INT_MAX, hi_max = -1;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int pr = u.pair0 + r_lo + 8 * j;
        const bool live = pr < u.pairs;
        const int i = live ? pr / p.G : 0;
        const __nv_bfloat16* qr = p.q + (int64_t)(u.row0 + i) * p.q_row + (int64_t)(walk.head * p.G + (live ? pr % p.G : 0)) * p.q_head + quad * 2;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[k][j] = live ? *reinterpret_cast<const uint32_t*>(qr + k * 16) : 0u;
          qf[k][2 + j] = live ? *reinterpret_cast<const uint32_t*>(qr + k * 16 + 8) : 0u;
        }
        lo[j] = u.key_lo;
        hi[j] = u.key_hi - 1;
        if (live) {
          if (u.base >= 0) {
            hi[j] = min(hi[j], u.base + i);
            if (p.window > 0) lo[j] = max(lo[j], u.base + i - p.window + 1);
          } else if (p.window > 0) {
            const int b = find_segment(p.row_start, p.B, u.row0 + i);
            lo[j] = max(lo[j], p.cached[b] + u.row0 + i - p.row_start[b] - p.window + 1);
          }
          lo_min = min(lo_min, lo[j]);
          lo_max = max(lo_max, lo[j]);
          hi_min = min(hi_min, hi[j]);
          hi_max = max(hi_max, hi[j]);
        }
      }
      lo_min = __reduce_min_sync(0xffffffffu, lo_min);
      lo_max = __reduce_max_sync(0xffffffffu, lo_max);
      hi_min = __reduce_min_sync(0xffffffffu, hi_min);
      hi_max = __reduce_max_sync(0xffffffffu, hi_max);
      float o[D / 8][4];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

      const int t0 = u.key_lo / kTileA + walk.first;
      for (int i = 0; i < walk.count; ++i, ++it) {
        const int st = it % C::kStages;
        if (!warp_wait(full(st), (it / C::kStages) & 1, abort_flag)) { ok = false; break; }
        const uint32_t ks = base + st * C::kStageBytes, vs = ks + C::kHalfBytes;
        const int k0 = (t0 + i) * kTileA + warp * 16;                     // this warp's first key
        if (k0 <= hi_max && k0 + 15 >= lo_min) {
          // S = Q K^T
          float s[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
          {
            const int key = ((lane >> 4) << 3) + (lane & 7);
            const uint32_t rowa = ks + mine + key * 128;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const int chunk = (k & 3) * 2 + ((lane >> 3) & 1);
              uint32_t b[4];
              ldmatrix4(rowa + (k >> 2) * block + ((chunk ^ (key & 7)) << 4), b);
              mma16816(s[0], qf[k], b[0], b[1]);
              mma16816(s[1], qf[k], b[2], b[3]);
            }
          }
          const bool edge = k0 + 15 > hi_min || k0 < lo_max;
          if (edge) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = k0 + n * 8 + quad * 2 + (e & 1);
                if (key < lo[e >> 1] || key > hi[e >> 1]) s[n][e] = -INFINITY;
              }
            // values outside every row's range may be anything, and a zero weight does not silence an infinity
            if (k0 + 15 > hi_max || k0 < lo_min) {
              for (int c = lane; c < 16 * (D / 8); c += 32) {
                const int key = c / (D / 8), ch = c % (D / 8);
                if (k0 + key > hi_max || k0 + key < lo_min)
                  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs + mine + (ch >> 3) * block + key * 128 + (((ch & 7) ^ (key & 7)) << 4)),
                               "r"(0) : "memory");
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
          // running maximum: raised only when it grew by more than 2^8, P = exp2(S scale - m) stays in bf16's range
          float mt[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mt[j] = fmaxf(fmaxf(s[0][2 * j], s[0][2 * j + 1]), fmaxf(s[1][2 * j], s[1][2 * j + 1]));
            mt[j] = fmaxf(mt[j], __shfl_xor_sync(0xffffffffu, mt[j], 1));
            mt[j] = fmaxf(mt[j], __shfl_xor_sync(0xffffffffu, mt[j], 2)) * p.scale_log2;
          }
          if (__any_sync(0xffffffffu, mt[0] > m[0] + 8.f || mt[1] > m[1] + 8.f)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float mn = fmaxf(m[j], mt[j]);
              const float a = m[j] == -INFINITY ? 0.f : exp2f(m[j] - mn);
              m[j] = mn;
              l[j] *= a;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                o[n][2 * j] *= a;
                o[n][2 * j + 1] *= a;
              }
            }
          }
          uint32_t pf[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float neg = m[j] == -INFINITY ? 0.f : -m[j];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const float a = exp2f(fmaf(s[n][2 * j], p.scale_log2, neg)), b = exp2f(fmaf(s[n][2 * j + 1], p.scale_log2, neg));
              l[j] += a + b;
              pf[2 * n + j] = pack2bf(a, b);
            }
          }
          // O += P V
          {
            const int key = (((lane >> 3) & 1) << 3) + (lane & 7);
            const uint32_t rowa = vs + mine + key * 128;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
              const int chunk = (n & 3) * 2 + (lane >> 4);
              uint32_t b[4];
              ldmatrix4_t(rowa + (n >> 2) * block + ((chunk ^ (key & 7)) << 4), b);
              mma16816(o[2 * n], pf, b[0], b[1]);
              mma16816(o[2 * n + 1], pf, b[2], b[3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(st));
      }
      // ---- join the four warps
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
        if (quad == 0) {
          ml[(warp * kRowsA + r_lo + 8 * j) * 2] = m[j];
          ml[(warp * kRowsA + r_lo + 8 * j) * 2 + 1] = l[j];
        }
      }
      if (consumer_any(!ok)) break;              // a wait ran out: all four leave together
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mm = -INFINITY;
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[(w * kRowsA + r_lo + 8 * j) * 2]);
        const float f = m[j] == -INFINITY ? 0.f : exp2f(m[j] - mm);
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * j] *= f;
          o[n][2 * j + 1] *= f;
        }
      }
      const int live_rows = min(kRowsA, u.pairs - u.pair0);
      const bool tall = live_rows > 8;           // a decode step of up to eight heads a key head has nothing in the upper rows
      // an fp32 tile in shared memory: column blocks of eight are spread over the banks by the row
      auto slot = [&](int which, int row, int c) { return exch + which * (kRowsA * D) + row * D + (c ^ ((row & 7) << 3)); };
      auto put = [&](int which) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j == 1 && !tall) break;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(slot(which, r_lo + 8 * j, n * 8 + quad * 2)) = make_float2(o[n][2 * j], o[n][2 * j + 1]);
        }
      };
      auto add = [&](int which) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j == 1 && !tall) break;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const float2 v = *reinterpret_cast<const float2*>(slot(which, r_lo + 8 * j, n * 8 + quad * 2));
            o[n][2 * j] += v.x;
            o[n][2 * j + 1] += v.y;
          }
        }
      };
      if (warp & 1) put(warp >> 1);
      consumer_sync();
      if (!(warp & 1)) add(warp >> 1);
      if (warp == 2) put(1);
      consumer_sync();
      if (warp == 0) {
        add(1);
        put(0);
      }
      consumer_sync();
      const bool whole = walk.count == walk.unit_tiles;
      const int which = walk.first > 0 ? 0 : 1;
      if (threadIdx.x == 0) p.cuts[blockIdx.x] = walk.cut(u);
      const int64_t cta = blockIdx.x;
      for (int c = threadIdx.x; c < live_rows * (D / 4); c += 128) {
        const int row = c / (D / 4), d = (c % (D / 4)) * 4;
        const int pr = u.pair0 + row;
        const float4 v = *reinterpret_cast<const float4*>(slot(0, row, d));
        float mm = -INFINITY, ll = 0.f;
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[(w * kRowsA + row) * 2]);
        for (int w = 0; w < 4; ++w) {
          const float mw = ml[(w * kRowsA + row) * 2];
          ll += (mw == -INFINITY ? 1.f : exp2f(mw - mm)) * ml[(w * kRowsA + row) * 2 + 1];   // without a maximum: 0, or NaN
        }
        const int64_t rh = (int64_t)(u.row0 + pr / p.G) * p.Hq + walk.head * p.G + pr % p.G;
        if (whole && u.shared < 0) {
          float den = ll;
          float f = 1.f;
          if (p.sinks != nullptr) {
            const float sk = p.sinks[rh % p.Hq] * 1.4426950408889634f, top = fmaxf(sk, mm);
            f = mm == -INFINITY ? 0.f : exp2f(mm - top);
            den = ll * f + (sk == -INFINITY ? 0.f : exp2f(sk - top));
          }
          f = den == 0.f ? 0.f : f / den;        // a NaN stays one
          *reinterpret_cast<uint2*>(p.out + rh * D + d) = make_uint2(pack2bf(v.x * f, v.y * f), pack2bf(v.z * f, v.w * f));
        } else if (whole) {
          const int64_t at = p.shared_at(u, pr, walk.head);
          if (at < 0) continue;
          *reinterpret_cast<float4*>(p.row_o + at * D + d) = v;
          if (d == 0) *reinterpret_cast<float2*>(p.row_ml + at * 2) = make_float2(mm, ll);
        } else {
          const int64_t at = (cta * 2 + which) * kRowsA + row;
          *reinterpret_cast<float4*>(p.part_a + at * D + d) = v;
          if (d == 0) *reinterpret_cast<float2*>(p.part_a_ml + at * 2) = make_float2(mm, ll);
        }
      }
      consumer_sync();
    }
  }
  wait_for_earlier();                            // the tcgen05 kernel runs at the same time; what follows needs both
  __syncthreads();
  if (*abort_flag) {
    if (warp == 4) drain(it, C::kStages, full);
    if (threadIdx.x == 0) atomicOr(p.status, kStatusPagedWaitTimedOut);
  }
}

// Many rows behind one key range (a prefix with the rows of its group, the rows of a prompt chunk): tcgen05.
//
// A unit is up to 128 pairs (whole rows), one TMEM lane each; 64-key tiles alternate between two softmax warpgroups, which
// keep their own running maximum, sum and output accumulator, so neither waits for the other, and each has two score
// buffers, so that the softmax of one tile runs under the MMAs of the next.  Per tile: S = Q K^T into tensor memory,
// P = exp2(S - m) written over S as bf16, O += P V with P read from tensor memory.  Behind every P V the issuer puts the S
// of the tile four later, into the same buffer, and a commit (a bare one at the end), so "the next S of a buffer is there"
// also says that its P V is done: a warpgroup that has to rescale its accumulator waits for that of its other buffer.
// Queries come by TMA too (boxes of rows x heads of the key head), the next piece's as soon as the last S is done.
// The exponentials (64 x 128 per tile on a 16-per-clock unit) and the MMAs take 512 clocks a tile each; the issuing thread's
// own work (two waits, twelve MMAs of 60 to 75 clocks, three commits) takes some 1700 and bounds the kernel: 4 groups of
// 16 sequences behind 65536 tokens, 4 key heads: 139 us for 537 MB (3.9 TB/s); one group of 64: 586 TFLOP/s; 512 rows behind
// 8192 tokens, 32 + 8 heads of 128: 128 us (555 TFLOP/s).  A prompt is slower: 4096 rows alone take 437 us, 315 TFLOP/s counted
// over the keys that a row sees, some 3500 clocks a tile, which the issuing thread does not explain; what does has not been
// measured (its units are short, 32 tiles in the mean, with one buffer for the queries and an output to drain each).  The flash
// forward, which keeps two query tiles per tile of keys, takes 157 us.
// P is rounded to bf16 before it meets V, as in the flash kernels: the tensor cores take the values' type.
//   warp 0: TMA producer    warp 1: TMEM, MMA issue    warps 2..5, 6..9: softmax of even / odd tiles, then the output
// Tensor memory: score buffer b (of warpgroup b % 2) at column 64 b, accumulator of warpgroup g at 256 + 128 g.
template <int D>
struct CfgB {
  static constexpr int kStages = D == 64 ? 10 : 5;               // tiles of keys and of values in flight: 160 KB
  static constexpr uint32_t kQBytes = kRowsB * D * 2;
  static constexpr uint32_t kTileBytes = kTileB * D * 2;
  static constexpr uint32_t kStage = kQBytes + 2 * kStages * kTileBytes;         // fp32 rows on their way out, 2 KB a warp
  static constexpr uint32_t kBars = kStage + 8 * 2048;
  static constexpr int kNumBars = 4 * kStages + 13;
  static constexpr uint32_t kMl = kBars + 8 * kNumBars + 8;      // TMEM address, abort flag
  static constexpr uint32_t kSmem = kMl + 2 * kRowsB * 2 * 4;
};

// Named barrier of the eight softmax warps; true for all when any thread brings true.
__device__ __forceinline__ bool softmax_any(bool v) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.or.pred b, 2, 256, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)v) : "memory");
  return r != 0;
}
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <int D>
__global__ void __launch_bounds__(320, 1)
attn_block_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const AttnParams p) {
  using C = CfgB<D>;
  using namespace tc;
  constexpr uint32_t kQCol = kRowsB * 128, kCol = kTileB * 128;   // one 64-column block of the queries, of a tile
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t q_smem = base;
  auto k_smem = [&](int s) { return base + C::kQBytes + C::kTileBytes * (2 * s); };
  auto v_smem = [&](int s) { return base + C::kQBytes + C::kTileBytes * (2 * s + 1); };
  const uint32_t bars = base + C::kBars;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (C::kStages + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * C::kStages + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * C::kStages + s); };
  auto s_full = [&](int b) { return bars + 8u * (4 * C::kStages + b); };
  auto p_ready = [&](int b) { return bars + 8u * (4 * C::kStages + 4 + b); };
  const uint32_t q_full = bars + 8u * (4 * C::kStages + 8), q_empty = q_full + 8u, o_full = q_full + 16u, o_free = q_full + 24u, quit = q_full + 32u;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + C::kBars + 8 * C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  float* ml = reinterpret_cast<float*>(smem + C::kMl);            // [2][kRowsB][2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  let_next_start();
  const List list = p.list_b(WorkLayout(p.B, p.NG, p.max_a, p.max_b));
  Walk walk(list, p.Hkv, blockIdx.x);
  if (walk.at >= walk.end) {                                      // the same for the whole block
    if (threadIdx.x == 64) p.cuts[p.ctas_a + blockIdx.x] = Cut{0, 0, 0, 0, 0};
    return;
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(s_full(b), 1);
      mbar_init(p_ready(b), 4);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_full, 1);
    mbar_init(o_free, 8);
    mbar_init(quit, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_ptr), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  int issued_k = 0, issued_v = 0, issued_q = 0;  // the producer's copies

  if (warp == 0) {
    // ---------------------------------------------------------------------------------------------------- producer
    const int box = min(p.ps, kTileB), subs = kTileB / box;
    // A tile is [64-column block][key][128 bytes]: one box where a page holds the whole tile, else one per page and block
    const int loads = subs == 1 ? 1 : (D / 64) * subs;            // at most 2 * 4 per operand: lanes 0..15 keys, 16..31 values
    const uint32_t bytes = box * 128 * (subs == 1 ? D / 64 : 1);
    const int kv = lane >> 4, li = lane & 15, col = li / subs, sub = li % subs;
    const CUtensorMap* map = kv ? &tmap_v : &tmap_k;
    const uint32_t q_bytes = (uint32_t)(p.rows_b * p.G) * D * 2;   // a whole box: rows behind the tensor are filled with zeros
    bool ok = true;
    int it = 0, piece = 0;
    while (ok && walk.next()) {
      const Unit u = list.units[walk.u];
      const int* row = p.table + (int64_t)u.slot * p.W;
      const int t0 = u.key_lo / kTileB + walk.first;
      auto entry = [&](int t) {
        const int key = t * kTileB + sub * box;
        return li < loads && key < u.key_hi ? row[key >> p.ps_shift] : INT_MIN;
      };
      int page = entry(t0), page1 = walk.count > 1 ? entry(t0 + 1) : INT_MIN;
      if (!warp_wait(q_empty, (piece & 1) ^ 1, abort_flag)) break;   // the last S of the piece before is done
      if (lane == 0) {
        mbar_expect_tx(q_full, q_bytes);
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(q_smem + c * kQCol, &tmap_q, q_full, c * 64, walk.head * p.G, u.row0 + u.pair0 / p.G);
      }
      issued_q = ++piece;
      for (int i = 0; i < walk.count; ++i, ++it) {
        const int st = it % C::kStages;
        const uint32_t parity = ((it / C::kStages) & 1) ^ 1;
        const int t = t0 + i;
        const int page2 = i + 2 < walk.count ? entry(t + 2) : INT_MIN;      // fetched two tiles ahead
        const bool wanted = page != INT_MIN;
        const int need = __popc(__ballot_sync(0xffffffffu, wanted) & 0xffffu);
        if (wanted && (page < 0 || page >= p.num_pages)) {        // out of range: the load fills zeros
          atomicOr(p.status, kStatusPagePlanInvalid);
          page = p.num_pages;
        }
        const int slot = (t * kTileB + sub * box) & (p.ps - 1);
        const uint32_t off = col * kCol + sub * box * 128;
        if (!warp_wait(k_empty(st), parity, abort_flag)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(k_full(st), need * bytes);
        __syncwarp();
        if (wanted && kv == 0) tma_load_5d(k_smem(st) + off, map, k_full(st), 0, slot, col, walk.head, page);
        issued_k = it + 1;
        if (!warp_wait(v_empty(st), parity, abort_flag)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(v_full(st), need * bytes);
        __syncwarp();
        if (wanted && kv == 1) tma_load_5d(v_smem(st) + off, map, v_full(st), 0, slot, col, walk.head, page);
        issued_v = it + 1;
        page = page1;
        page1 = page2;
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------------------------------------------- MMA issue
    // This thread's own instructions are on the critical path of every tile: stages and parities are counted up, not
    // divided out, and a barrier that is there already costs one poll.
    if (lane == 0) {
      const uint32_t idesc_s = make_idesc(false, false, kRowsB, kTileB);
      const uint32_t idesc_pv = make_idesc(false, true, kRowsB, D);       // values are [keys, D]: MN-major
      // an operand's descriptor is its base plus 16-byte units
      const uint64_t q_desc = make_desc(q_smem, 16, 1024), k_desc = make_desc(k_smem(0), 16, 1024), v_desc = make_desc(v_smem(0), kCol, 1024);
      auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || mbar_wait(bar, parity, abort_flag); };
      int piece = 0, ks = 0, vs = 0;             // next stages of the two rings
      uint32_t kp = 0, vp = 0, ready = 0;        // their parities, and those of p_ready (one bit per buffer)
      bool ok = true;
      while (ok && walk.next()) {
        const int n = walk.count;
        auto issue_s = [&](int j) {
          if (!wait(k_full(ks), kp)) return false;
          tc_fence_after();
          const uint64_t kd = k_desc + ks * (2 * C::kTileBytes >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16<1>(tmem + 64 * (j & 3), q_desc + (((k >> 2) * kQCol + (k & 3) * 32u) >> 4), kd + (((k >> 2) * kCol + (k & 3) * 32u) >> 4), idesc_s, k != 0);
          umma_commit(s_full(j & 3));
          umma_commit(k_empty(ks));
          if (j == n - 1) umma_commit(q_empty);
          if (++ks == C::kStages) {
            ks = 0;
            kp ^= 1;
          }
          return true;
        };
        ok = wait(q_full, piece & 1);
        for (int j = 0; j < min(n, 4) && ok; ++j) ok = issue_s(j);
        // the output of the piece before has been read
        ok = ok && (piece == 0 || wait(o_free, (piece - 1) & 1));
        for (int j = 0; j < n && ok; ++j) {
          const int b = j & 3, g = j & 1;
          ok = wait(v_full(vs), vp) && wait(p_ready(b), (ready >> b) & 1);
          if (!ok) break;
          ready ^= 1u << b;
          tc_fence_after();
          const uint64_t vd = v_desc + vs * (2 * C::kTileBytes >> 4);
#pragma unroll
          for (int k = 0; k < kTileB / 16; ++k)  // 16 keys: 8 packed columns of P, 16 rows of V
            umma_bf16_ts(tmem + 256 + 128 * g, tmem + 64 * b + k * 8, vd + k * (2048 >> 4), idesc_pv, j >= 2 || k != 0);
          umma_commit(v_empty(vs));
          if (++vs == C::kStages) {
            vs = 0;
            vp ^= 1;
          }
          if (j + 4 < n) ok = issue_s(j + 4);
          else umma_commit(s_full(b));
        }
        if (ok) umma_commit(o_full);
        ++piece;
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------------------------------------------- softmax
    const int g = (warp - 2) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;           // this thread's pair in the unit, and its TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_t = lane_base + 256;
    float* stage = reinterpret_cast<float*>(smem + C::kStage + (warp - 2) * 2048);
    int it = 0, piece = 0;
    if (threadIdx.x == 64) p.cuts[p.ctas_a + blockIdx.x] = Cut{0, 0, 0, 0, 0};   // each piece writes it again
    uint32_t full = 0;                           // parities of s_full, one bit per buffer
    bool ok = true;
    while (ok && walk.next()) {
      const Unit u = list.units[walk.u];
      const int n = walk.count;
      // visible keys of this pair
      const int pr = u.pair0 + r;
      const bool live = pr < u.pairs && r < p.rows_b * p.G;
      int lo = u.key_lo, hi = u.key_hi - 1;
      if (live) {
        const int row = u.row0 + pr / p.G;
        if (u.base >= 0) {
          hi = min(hi, u.base + row - u.row0);
          if (p.window > 0) lo = max(lo, u.base + row - u.row0 - p.window + 1);
        } else if (p.window > 0) {
          const int b = find_segment(p.row_start, p.B, row);
          lo = max(lo, p.cached[b] + row - p.row_start[b] - p.window + 1);
        }
      }
      const bool warp_live = __any_sync(0xffffffffu, live);
      float m = -INFINITY, l = 0.f;
      for (int j = g; j < n; j += 2) {
        const int b = j & 3;
        const uint32_t s_t = lane_base + 64 * b;
        if (!warp_wait(s_full(b), (full >> b) & 1, abort_flag)) { ok = false; break; }
        full ^= 1u << b;
        tc_fence_after();
        const int c0 = (u.key_lo / kTileB + walk.first + j) * kTileB;
        if (warp_live) {
          uint32_t x[2][32];
          tmem_ld32(s_t, x[0]);
          tmem_ld32(s_t + 32, x[1]);
          tmem_ld_wait();
          const int rlo = lo - c0, rhi = hi - c0;
          if (rhi < kTileB - 1 || rlo > 0) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (c * 32 + e > rhi || c * 32 + e < rlo) x[c][e] = __float_as_uint(-INFINITY);
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(x[c][e]));
          const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2);
          if (__any_sync(0xffffffffu, m_new > m + 8.f)) {
            const float alpha = m == -INFINITY ? 0.f : exp2f(m - m_new);
            l *= alpha;
            if (j >= 2) {
              // P V of this warpgroup's previous tile is done once the next commit of that buffer has come (see above)
              const int ob = (j + 2) & 3;
              if (!warp_wait(s_full(ob), (full >> ob) & 1, abort_flag)) { ok = false; break; }
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(o_t + 128 * g + c * 16, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st16(o_t + 128 * g + c * 16, o);
              }
            }
            m = m_new;
          }
          const float neg = m == -INFINITY ? 0.f : -m;
          const uint64_t sc2 = pack_f2(p.scale_log2, p.scale_log2), neg2 = pack_f2(neg, neg);
          uint64_t ls[2] = {pack_f2(0.f, 0.f), pack_f2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float a, d;
              unpack_f2(fma_f2(pack_f2(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), sc2, neg2), a, d);
              a = exp2f(a);
              d = exp2f(d);
              ls[e & 1] = add_f2(ls[e & 1], pack_f2(a, d));
              pk[e] = pack2bf(a, d);
            }
            tmem_st16(s_t + c * 16, pk);
          }
          float a0, a1, b0, b1;
          unpack_f2(ls[0], a0, a1);
          unpack_f2(ls[1], b0, b1);
          l += (a0 + a1) + (b0 + b1);
          tmem_st_wait();
        }
        // values outside the keys of the unit may be anything, and a zero weight does not silence an infinity
        if (c0 + kTileB > u.key_hi || c0 < u.key_lo) {
          const int st = (it + j) % C::kStages;
          if (!warp_wait(v_full(st), ((it + j) / C::kStages) & 1, abort_flag)) { ok = false; break; }
          const int from = max(0, u.key_hi - c0), before = max(0, u.key_lo - c0);
          for (int key = r / (D / 8); key < kTileB; key += 128 / (D / 8)) {
            const int ch = r % (D / 8);
            if (key >= from || key < before)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_smem(st) + (ch >> 3) * kCol + key * 128 + (((ch & 7) ^ (key & 7)) << 4)),
                           "r"(0) : "memory");
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(b));
      }
      // every buffer that was used this piece has one more commit behind its last P V
      for (int b = g; b < min(n, 4); b += 2) full ^= 1u << b;
      it += n;
      // ---- join the two warpgroups; each writes half of the columns of every row
      ok = ok && warp_wait(o_full, piece & 1, abort_flag);
      ml[(g * kRowsB + r) * 2] = m;
      ml[(g * kRowsB + r) * 2 + 1] = l;
      if (softmax_any(!ok)) break;
      tc_fence_after();
      const float m0 = ml[r * 2], m1 = n > 1 ? ml[(kRowsB + r) * 2] : -INFINITY;
      const float mm = fmaxf(m0, m1);
      float f0 = m0 == -INFINITY ? 0.f : exp2f(m0 - mm), f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mm);
      const float ll = f0 * ml[r * 2 + 1] + f1 * ml[(kRowsB + r) * 2 + 1];
      const bool whole = walk.count == walk.unit_tiles;
      const bool last = whole && u.shared < 0;
      const int64_t rh = live ? (int64_t)(u.row0 + pr / p.G) * p.Hq + walk.head * p.G + pr % p.G : 0;
      if (last) {
        float den = ll, f = 1.f;
        if (p.sinks != nullptr) {
          const float sk = p.sinks[rh % p.Hq] * 1.4426950408889634f, top = fmaxf(sk, mm);
          f = mm == -INFINITY ? 0.f : exp2f(mm - top);
          den = ll * f + (sk == -INFINITY ? 0.f : exp2f(sk - top));
        }
        f = den == 0.f ? 0.f : f / den;          // a NaN stays one
        f0 *= f;
        f1 *= f;
      }
      if (warp_live) {
        // 16 columns of the warp's 32 rows at a time go through shared memory, so that four lanes write the 64 bytes of a row
        const int64_t at = last ? 0 : !whole ? ((int64_t)blockIdx.x * 2 + (walk.first > 0 ? 0 : 1)) * kRowsB + r : live ? p.shared_at(u, pr, walk.head) : 0;
        if (!last && live && g == 0 && at >= 0) *reinterpret_cast<float2*>((whole ? p.row_ml : p.part_b_ml) + at * 2) = make_float2(mm, ll);
        const int sub = lane >> 2, quad = lane & 3;
        char* mine = !live || at < 0 ? nullptr : last ? reinterpret_cast<char*>(p.out + rh * D) : reinterpret_cast<char*>((whole ? p.row_o : p.part_b) + at * D);
        char* dst[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          dst[k] = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, (unsigned long long)mine, k * 8 + sub));
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          const int col = g * (D / 2) + c * 16;
          uint32_t a[16], b[16];
          tmem_ld16(o_t + col, a);
          tmem_ld16(o_t + 128 + col, b);         // with one tile the second accumulator is not read below
          tmem_ld_wait();
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = f0 * __uint_as_float(a[4 * e + i]) + (n > 1 ? f1 * __uint_as_float(b[4 * e + i]) : 0.f);
            *reinterpret_cast<float4*>(stage + lane * 16 + ((e ^ (lane >> 1)) & 3) * 4) = make_float4(v[0], v[1], v[2], v[3]);
          }
          __syncwarp();
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(stage + (k * 8 + sub) * 16 + ((quad ^ ((k * 8 + sub) >> 1)) & 3) * 4);
          if (last) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (dst[k] != nullptr) *reinterpret_cast<uint2*>(dst[k] + (col + quad * 4) * 2) = make_uint2(pack2bf(v[k].x, v[k].y), pack2bf(v[k].z, v[k].w));
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (dst[k] != nullptr) *reinterpret_cast<float4*>(dst[k] + (col + quad * 4) * 4) = v[k];
          }
        }
      }
      tc_fence_before();
      if (softmax_any(false)) break;             // ml is read before the next piece writes it
      if (lane == 0) mbar_arrive(o_free);
      ++piece;
      if (threadIdx.x == 64) p.cuts[p.ctas_a + blockIdx.x] = walk.cut(u);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (warp == 0) {
      drain(issued_k, C::kStages, k_full);
      drain(issued_v, C::kStages, v_full);
      drain(issued_q, 1, [&](int) { return q_full; });
    } else if (warp == 1 && lane == 0) {         // and the MMAs, before their accumulators are given back
      volatile int quiet = 0;
      umma_commit(quit);
      mbar_wait(quit, 0, &quiet);
    }
    if (threadIdx.x == 0) atomicOr(p.status, kStatusPagedWaitTimedOut);
    __syncwarp();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One row and query head, key by key, by a warp: for rows that have a NaN in their output.  Where the scores are numbers, that comes
// from values that are not finite: one that the row sees, or one that only other rows of its unit see, since 0 * inf is a NaN
// in the products above.  Looking for such values in every tile that some rows see and others do not cost a prompt of
// 4096 rows 15 % (418 -> 483 us), and a test in the attention kernels' store loops 6 to 20 %, because it changed how their loops
// over the tiles were compiled.  Looking at the outputs here costs 2 % of a prompt of 4096 rows (427 -> 437 us) and nothing of a
// step of single rows.  A value that is not finite counts whatever its probability rounds to.
template <int D>
__device__ __noinline__ void attend_row(const AttnParams& p, int row, int h) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int b = find_segment_warp(p.row_start, p.B, row);
  const int pos = p.cached[b] + row - p.row_start[b];
  const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int last = (int)min((int64_t)pos, (int64_t)p.W * p.ps - 1);
  const int* table = p.table + (int64_t)p.slots[b] * p.W;
  const __nv_bfloat16* k0 = p.kp + (h / p.G) * p.kp_head;
  const __nv_bfloat16* v0 = p.vp + (h / p.G) * p.vp_head + lane * N;
  const uint32_t* q0 = reinterpret_cast<const uint32_t*>(p.q + (int64_t)row * p.q_row + (int64_t)h * p.q_head);
  float o[N];
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int base = first; base <= last; base += 32) {             // a key a lane
    const int key = base + lane, slot = key & (p.ps - 1);
    const int page = key <= last ? table[key >> p.ps_shift] : -1;
    const bool there = page >= 0 && page < p.num_pages;          // else zeros, as in the kernels above
    const uint4* k = reinterpret_cast<const uint4*>(k0 + page * p.kp_page + slot * p.kp_slot);
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      const uint4 v = there ? k[c] : make_uint4(0, 0, 0, 0);
      const uint32_t kw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t qw = q0[4 * c + i];
        s = fmaf(__uint_as_float(qw << 16), __uint_as_float(kw[i] << 16), s);
        s = fmaf(__uint_as_float(qw & 0xffff0000u), __uint_as_float(kw[i] & 0xffff0000u), s);
      }
    }
    s = key <= last ? s * p.scale_log2 : -INFINITY;
    if (__any_sync(0xffffffffu, s != s)) {       // so is the sum, and every output
      l = s = __uint_as_float(0x7fffffffu);
      break;
    }
    const float top = fmaxf(m, warp_max(s));
    if (top == -INFINITY) continue;
    const float a = m == -INFINITY ? 0.f : exp2f(m - top), w = exp2f(s - top);
    m = top;
    l = l * a + warp_sum(w);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (fabsf(o[e]) < INFINITY) o[e] *= a;
    const int64_t at = there ? page * p.vp_page + slot * p.vp_slot : -1;
    unsigned seen = __ballot_sync(0xffffffffu, s > -INFINITY && there);
    while (seen != 0u) {
      float wj[4], v[4][N];
#pragma unroll
      for (int j = 0; j < 4; ++j) {              // four values in flight
        const int k = seen != 0u ? __ffs(seen) - 1 : -1;
        seen &= seen - 1;
        wj[j] = k < 0 ? 0.f : __shfl_sync(0xffffffffu, w, k);
        const int64_t row_at = k < 0 ? -1 : __shfl_sync(0xffffffffu, at, k);
#pragma unroll
        for (int e = 0; e < N; ++e) v[j][e] = k < 0 ? 0.f : __bfloat162float(v0[row_at + e]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = fabsf(v[j][e]) < INFINITY ? fmaf(wj[j], v[j][e], o[e]) : o[e] + v[j][e];
    }
  }
  float f = 1.f;
  if (p.sinks != nullptr) {
    const float sk = p.sinks[h] * 1.4426950408889634f, top = fmaxf(sk, m);
    f = m == -INFINITY ? 0.f : exp2f(m - top);
    l = l * f + (sk == -INFINITY ? 0.f : exp2f(sk - top));
  }
  f = l == 0.f ? 0.f : f / l;
  __nv_bfloat16* out = p.out + ((int64_t)row * p.Hq + h) * D + lane * N;
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (f != f || !(fabsf(o[e]) >= INFINITY)) o[e] *= f;         // an infinity stays one unless the sum is a NaN
#pragma unroll
  for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2bf(o[e], o[e + 1]);
}
// The same for the rows of 32 adjacent vectors of the output, from vector `c0`, where a lane saw a NaN: those that the attention
// kernels finished.  A row that this kernel joins may not be there yet; it is looked at where it is joined.
template <int D>
__device__ __noinline__ void attend_again(const AttnParams& p, int64_t c0, bool nan) {
  constexpr int kV = D / 8;
  const int lane = threadIdx.x & 31;
  const int* seq_group = p.work + WorkLayout(p.B, p.NG, p.max_a, p.max_b).seq_group;
  for (unsigned left = __ballot_sync(0xffffffffu, nan); left != 0u;) {
    const int k = (__ffs(left) - 1) / kV * kV;   // first lane of the row
    left &= ~((kV == 32 ? 0xffffffffu : (1u << (kV & 31)) - 1u) << k);
    const int64_t rh = (c0 + k) / kV;
    const int row = (int)(rh / p.Hq), h = (int)(rh % p.Hq);
    const int b = find_segment_warp(p.row_start, p.B, row);
    const int pr = (row - p.row_start[b]) * p.G + h % p.G;
    bool joined = seq_group[b] >= 0;
    for (int i = lane; i < p.ctas_a + (p.use_b ? p.ctas_b : 0); i += 32) {
      const Cut u = p.cuts[i];
      joined |= u.parts > 0 && u.row0 == p.row_start[b] && u.head == h / p.G && pr >= u.pair0 && pr < u.pair0 + (i < p.ctas_a ? kRowsA : p.rows_b * p.G);
    }
    if (!__any_sync(0xffffffffu, joined)) attend_row<D>(p, row, h);
  }
}
__device__ __forceinline__ bool any_nan(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) nan |= (w[i] & 0x7fffu) > 0x7f80u || (w[i] & 0x7fff0000u) > 0x7f800000u;
  return nan;
}
// Block `block` of `blocks` looks at its share of the output.  Only where a sequence has several rows: the pairs of one row see
// the same keys, and values outside those are cleared above.
template <int D>
__device__ __forceinline__ void look_for_nan(const AttnParams& p, int last_row, int block, int blocks) {
  const int64_t n = (int64_t)last_row * p.Hq * (D / 8), step = (int64_t)blocks * 128;
  const uint4* out = reinterpret_cast<const uint4*>(p.out);
  const int lane = threadIdx.x & 31;
  for (int64_t c = (int64_t)block * 128 + threadIdx.x - lane; c < n; c += 4 * step) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i * step + lane < n ? out[c + i * step + lane] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (__any_sync(0xffffffffu, any_nan(v[i]))) attend_again<D>(p, c + i * step, any_nan(v[i]));
  }
}

// Joins what the attention kernels left in parts.  Blocks [0, cuts): a sequence that shares nothing is in parts where a
// stretch boundary cuts one of its units; a CTA has at most one cut unit that begins in its stretch and goes on behind it
// and left its description, and the block(s) of that CTA join it.  The other blocks: a (row, query head) of a group that
// shares always has two sources; a warp joins the parts of both, those of the prefix first.  All orders are fixed.  Rows
// behind the last sequence are cleared on the way.  Latency bound: a few dependent loads.
constexpr int kSlices = 8;                       // blocks that share a cut unit of 128 pairs

template <int D>
__global__ void __launch_bounds__(128, 8) finish_kernel(const __grid_constant__ AttnParams p) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const WorkLayout lay(p.B, p.NG, p.max_a, p.max_b);
  const int cuts = p.ctas_a + (p.use_b ? p.ctas_b * kSlices : 0);
  const int last_row = p.row_start[p.B];
  const bool several = p.work[6] != 0;
  auto finish = [&](int64_t rh, float m, float l) {              // 1 / denominator, with the head's sink
    float f = 1.f;
    if (p.sinks != nullptr) {
      const float sk = p.sinks[rh % p.Hq] * 1.4426950408889634f, top = fmaxf(sk, m);
      f = m == -INFINITY ? 0.f : exp2f(m - top);
      l = l * f + (sk == -INFINITY ? 0.f : exp2f(sk - top));
    }
    return l == 0.f ? 0.f : f / l;               // a NaN stays one
  };
  if ((int)blockIdx.x < cuts) {
    const bool big = (int)blockIdx.x >= p.ctas_a;
    const int c0 = big ? (blockIdx.x - p.ctas_a) / kSlices : blockIdx.x;
    const int row0 = big ? (blockIdx.x - p.ctas_a) % kSlices * (kRowsB / kSlices) : 0;      // this block's rows of the unit
    const int rows = big ? kRowsB : kRowsA;
    wait_for_earlier();
    if (several) look_for_nan<D>(p, last_row, blockIdx.x, cuts);
    const Cut unit = p.cuts[big ? p.ctas_a + c0 : c0];
    const int parts = min(unit.parts, (big ? p.ctas_b : p.ctas_a) - c0), head = unit.head;
    if (p.zero_tail) {
      const int64_t n = (int64_t)(p.R - last_row) * p.Hq * D / 8;
      uint4* tail = reinterpret_cast<uint4*>(p.out + (int64_t)last_row * p.Hq * D);
      for (int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x; i < n; i += (int64_t)cuts * 128) tail[i] = make_uint4(0, 0, 0, 0);
    }
    if (parts == 0) return;
    const float* po = big ? p.part_b : p.part_a;
    const float* pml = big ? p.part_b_ml : p.part_a_ml;
    auto part = [&](int i, int row) { return i == 0 ? ((int64_t)c0 * 2 + 1) * rows + row : (int64_t)(c0 + i) * 2 * rows + row; };
    const int live = min(big ? min(row0 + kRowsB / kSlices, p.rows_b * p.G) : rows, unit.pairs - unit.pair0);
    bool again = false;
    for (int c = threadIdx.x; c < (live - row0) * (D / 4); c += 128) {
      const int row = row0 + c / (D / 4), d = (c % (D / 4)) * 4;
      // eight parts at a time, all their loads in flight together
      float m = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i0 = 0; i0 < parts; i0 += 8) {
        float2 v[8];
        float4 q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t at = part(min(i0 + i, parts - 1), row);
          v[i] = *reinterpret_cast<const float2*>(pml + at * 2);
          q[i] = *reinterpret_cast<const float4*>(po + at * D + d);
          if (i0 + i >= parts) v[i] = make_float2(-INFINITY, 0.f);
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) mn = fmaxf(mn, v[i].x);
        const float a = m == -INFINITY ? 1.f : exp2f(m - mn);    // there was no output before: o is 0, l is 0 or NaN
        m = mn;
        l *= a;
        o.x *= a; o.y *= a; o.z *= a; o.w *= a;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (v[i].x == -INFINITY) {             // without a visible key the output may be anything and the sum is 0,
            l += v[i].y;                         // without a score but NaN it is NaN
            continue;
          }
          const float w = exp2f(v[i].x - mn);
          l += v[i].y * w;
          o.x += q[i].x * w; o.y += q[i].y * w; o.z += q[i].z * w; o.w += q[i].w * w;
        }
      }
      const int pr = unit.pair0 + row;
      const int64_t rh = (int64_t)(unit.row0 + pr / p.G) * p.Hq + head * p.G + pr % p.G;
      const float f = finish(rh, m, l);
      const float4 y = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
      again |= any_nan(y) && l == l;
      *reinterpret_cast<uint2*>(p.out + rh * D + d) = make_uint2(pack2bf(y.x, y.y), pack2bf(y.z, y.w));
    }
    if (__syncthreads_or(again))                 // all of the block's rows, which are few
      for (int pr = unit.pair0 + row0 + (threadIdx.x >> 5); pr < unit.pair0 + live; pr += 4)
        attend_row<D>(p, unit.row0 + pr / p.G, head * p.G + pr % p.G);
    return;
  }

  const int* shared = p.work + lay.shared;
  const int n_rows = min(shared[p.NG], p.max_shared), stride = (gridDim.x - cuts) * 4;
  const List list_a = p.list_a(lay), list_b = p.list_b(lay);
  bool waited = false;
  for (int64_t i = (blockIdx.x - cuts) * 4 + (threadIdx.x >> 5); i < (int64_t)n_rows * p.Hq; i += stride) {
    const int in = (unsigned)i / (unsigned)p.Hq, h = (int)i - in * p.Hq;
    const int g = find_segment_warp(shared, p.NG, in);
    const int r = p.work[lay.group_row + g] + in - shared[g];
    const int64_t rh = (int64_t)r * p.Hq + h;
    const int b = find_segment_warp(p.row_start, p.B, r);
    // where the parts of the two sources are: part 0, the others `step` apart
    struct Parts {
      const float *o, *ml;
      int64_t at0, at1;
      int step, n;
    };
    auto locate = [&](bool prefix) {
      Parts q{p.row_o, p.row_ml, ((int64_t)prefix * p.max_shared + in) * p.Hq + h, 0, 0, 0};
      const int s = prefix ? p.B + g : b;
      const int ua = p.work[lay.src_a + s], ub = p.use_b ? p.work[lay.src_b + s] : -1;
      const bool big = ub >= 0;
      const List list = big ? list_b : list_a;
      const int u0 = big ? ub : ua;
      if (u0 < 0 || u0 >= list.n_units) return q;
      const int rows = big ? kRowsB : kRowsA, per_unit = big ? p.rows_b * p.G : kRowsA;
      const int pr = (r - list.units[u0].row0) * p.G + h % p.G;
      const int u = u0 + pr / per_unit;
      if (u >= list.n_units) return q;
      const int t = list.tiles[u], nt = list.tiles[u + 1] - t;
      if (nt == 0) return q;
      const int per = list.stretch(p.Hkv), t0 = t * p.Hkv + (h / p.G) * nt;
      const int c0 = t0 / per, c1 = (t0 + nt - 1) / per;
      q.n = c1 - c0 + 1;
      if (c0 < c1) {
        q.o = big ? p.part_b : p.part_a;
        q.ml = big ? p.part_b_ml : p.part_a_ml;
        q.at0 = ((int64_t)c0 * 2 + 1) * rows + pr % per_unit;
        q.at1 = (int64_t)(c0 + 1) * 2 * rows + pr % per_unit;
        q.step = 2 * rows;
      }
      return q;
    };
    const Parts own = locate(false), pre = locate(true);
    if (!waited) wait_for_earlier();
    waited = true;
    float o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const int total = pre.n + own.n;
    for (int i0 = 0; i0 < total; i0 += 32) {     // the lanes fetch the maxima and sums of 32 parts at once
      const int mine = i0 + lane;
      float pm = -INFINITY, pl = 0.f;
      const float* src = p.row_o;
      if (mine < total) {
        const bool first = mine < pre.n;
        const int j = first ? mine : mine - pre.n;
        const int64_t at = j == 0 ? (first ? pre.at0 : own.at0) : (first ? pre.at1 : own.at1) + (int64_t)(j - 1) * (first ? pre.step : own.step);
        const float2 v = *reinterpret_cast<const float2*>((first ? pre.ml : own.ml) + at * 2);
        pm = v.x;
        pl = v.y;
        src = (first ? pre.o : own.o) + at * D;
      }
      const float mn = fmaxf(m, warp_max(pm));
      if (mn == -INFINITY) {                     // sums of nothing, or NaN where the scores are
        l += warp_sum(pl);
        continue;
      }
      const float a = m == -INFINITY ? 1.f : exp2f(m - mn);      // there was no output before: l is 0 or NaN
      const float w = pm == -INFINITY ? 0.f : exp2f(pm - mn);
      m = mn;
      l = l * a + warp_sum(pl * w);
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] *= a;
      const int cnt = min(32, total - i0);
      for (int j0 = 0; j0 < cnt; j0 += 4) {      // four parts' outputs in flight
        float wi[4], v[4][N];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = min(j0 + j, cnt - 1);
          wi[j] = j0 + j < cnt ? __shfl_sync(0xffffffffu, w, k) : 0.f;
          const float* q = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)src, k)) + lane * N;
#pragma unroll
          for (int e = 0; e < N; ++e) v[j][e] = q[e];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (wi[j] > 0.f) {                     // a part without a visible key may hold anything
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] += v[j][e] * wi[j];
          }
      }
    }
    const float f = finish(rh, m, l);
    __nv_bfloat16* out = p.out + rh * D + lane * N;
    bool again = false;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float a = o[e] * f, c = o[e + 1] * f;
      again |= a != a || c != c;
      *reinterpret_cast<uint32_t*>(out + e) = pack2bf(a, c);
    }
    if (__any_sync(0xffffffffu, again && l == l)) attend_row<D>(p, r, h);
  }
  if (!waited) wait_for_earlier();               // a block without a row still ends behind the earlier kernels
}

}  // namespace paged

static const int* int_vector(const at::Tensor& t, int64_t n, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1 && t.numel() == n,
              "page_plan: ", name, " must be a contiguous int32 vector of ", n, " elements on ", dev);
  return t.data_ptr<int>();
}

// Returns row_start [B + 1] int32, positions [R] int64, slot_map [R] int64; extends the rows of `block_table` in place.
std::tuple<at::Tensor, at::Tensor, at::Tensor> page_plan(const at::Tensor& cached, const at::Tensor& fresh, at::Tensor table,
                                                         const at::Tensor& slots, const at::Tensor& pages,
                                                         const c10::optional<at::Tensor>& mapped, int64_t page_size,
                                                         int64_t total_rows, int64_t num_pages) {
  TORCH_CHECK(table.is_cuda() && table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous(),
              "page_plan: block_table must be a contiguous int32 CUDA matrix");
  const auto dev = table.device();
  const int64_t B = cached.numel();
  TORCH_CHECK(pages.numel() <= (1 << 30), "page_plan: too many pages");
  TORCH_CHECK(B <= paged::kMaxSeqs, "page_plan: at most ", paged::kMaxSeqs, " sequences, got ", B);
  TORCH_CHECK(table.size(0) <= paged::kMaxSlots && table.size(1) <= paged::kMaxCols,
              "page_plan: the block table has at most ", paged::kMaxSlots, " rows and ", paged::kMaxCols, " columns");
  TORCH_CHECK(page_size > 0 && page_size <= (1 << 20), "page_plan: bad page size ", page_size);
  TORCH_CHECK(total_rows >= 0 && total_rows <= paged::kMaxRows && num_pages >= 0 && num_pages <= INT32_MAX, "page_plan: bad row or page count");
  c10::cuda::CUDAGuard guard(dev);
  paged::PlanParams p{};
  p.cached = int_vector(cached, B, dev, "cached");
  p.fresh = int_vector(fresh, B, dev, "new");
  p.slots = int_vector(slots, B, dev, "slots");
  p.pages = int_vector(pages, pages.numel(), dev, "pages");
  p.mapped = mapped.has_value() ? int_vector(*mapped, B, dev, "mapped") : nullptr;
  p.table = table.data_ptr<int>();
  p.B = (int)B; p.S = (int)table.size(0); p.W = (int)table.size(1); p.F = (int)pages.numel();
  p.ps = (int)page_size; p.R = (int)total_rows; p.num_pages = (int)num_pages;
  p.status = status_word_ptr();
  auto i32 = table.options();
  auto row_start = at::empty({B + 1}, i32);
  auto positions = at::empty({total_rows}, i32.dtype(at::kLong)), slot_map = at::empty({total_rows}, i32.dtype(at::kLong));
  p.row_start = row_start.data_ptr<int>();
  p.positions = positions.data_ptr<int64_t>();
  p.slot_map = slot_map.data_ptr<int64_t>();
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((std::max<int64_t>(total_rows, p.F) + 255) / 256, num_sms()));
  const size_t smem = sizeof(int) * (2 * (B + 1) + (p.S + 31) / 32);
  paged::plan_kernel<<<grid, 256, smem, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {row_start, positions, slot_map};
}

static void check_pages(const at::Tensor& k, const at::Tensor& v, const char* who) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && v.sizes() == k.sizes() && v.device() == k.device() && v.scalar_type() == k.scalar_type(),
              who, ": pages must be CUDA tensors [num_pages, Hkv, page_size, D] of one shape and type");
  const int64_t e = k.element_size();
  for (const at::Tensor* t : {&k, &v}) {
    TORCH_CHECK(t->stride(3) == 1 && (t->size(3) * e) % 16 == 0 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                who, ": page vectors must be contiguous and 16-byte aligned");
    for (int i = 0; i < 3; ++i)
      TORCH_CHECK((t->stride(i) * e) % 16 == 0 && t->stride(i) > 0, who, ": page strides must be positive multiples of 16 bytes");
  }
  TORCH_CHECK(k.size(0) <= INT32_MAX, who, ": too many pages");
}

void paged_write(const at::Tensor& k, const at::Tensor& v, at::Tensor k_pages, at::Tensor v_pages, const at::Tensor& slot_map) {
  check_pages(k_pages, v_pages, "paged_write");
  const auto dev = k_pages.device();
  const int64_t e = k_pages.element_size(), D = k_pages.size(3), H = k_pages.size(1);
  TORCH_CHECK(k_pages.scalar_type() == at::kBFloat16 || k_pages.scalar_type() == at::kFloat, "paged_write: unsupported dtype ", k_pages.scalar_type());
  TORCH_CHECK(slot_map.device() == dev && slot_map.scalar_type() == at::kLong && slot_map.is_contiguous() && slot_map.dim() == 1,
              "paged_write: slot_map must be a contiguous int64 vector on the pages' device");
  const int64_t T = slot_map.numel();
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->device() == dev && t->scalar_type() == k_pages.scalar_type() && t->dim() == 3 && t->size(0) == T && t->size(1) == H &&
                    t->size(2) == D && t->stride(2) == 1 && (t->stride(0) * e) % 16 == 0 && (t->stride(1) * e) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "paged_write: keys and values must be [T, Hkv, D] of the pages' type with 16-byte aligned vectors");
  if (T == 0 || H == 0) return;
  c10::cuda::CUDAGuard guard(dev);
  paged::WriteParams p{};
  p.k = (const char*)k.data_ptr(); p.v = (const char*)v.data_ptr();
  p.k_row = k.stride(0) * e; p.k_head = k.stride(1) * e; p.v_row = v.stride(0) * e; p.v_head = v.stride(1) * e;
  p.kp = (char*)k_pages.data_ptr(); p.vp = (char*)v_pages.data_ptr();
  p.kp_page = k_pages.stride(0) * e; p.kp_head = k_pages.stride(1) * e; p.kp_slot = k_pages.stride(2) * e;
  p.vp_page = v_pages.stride(0) * e; p.vp_head = v_pages.stride(1) * e; p.vp_slot = v_pages.stride(2) * e;
  p.slot_map = slot_map.data_ptr<int64_t>();
  p.T = T; p.ps = (int)k_pages.size(2); p.num_slots = k_pages.size(0) * k_pages.size(2);
  p.H = (int)H; p.vecs = (int)(D * e / 16);
  p.status = status_word_ptr();
  const int64_t total = T * H * p.vecs;
  const int grid = (int)std::min<int64_t>((total + 255) / 256, (int64_t)num_sms() * 32);
  paged::write_kernel<<<grid, 256, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Units of a step at most: one per source and one more per so many pairs; every row belongs to at most two sources.
static int64_t max_units(int64_t B, int64_t NG, int64_t R, int64_t G, int64_t rows) {
  const int64_t n = B + NG + (NG > 0 ? 2 : 1) * R * G / rows + 1;
  TORCH_CHECK(n < (1 << 26), "paged attention: too many rows");
  return n;
}

// The attention work list of a step for one window (see "Work" above).
at::Tensor paged_work(const at::Tensor& cached, const at::Tensor& row_start, const at::Tensor& slots, const c10::optional<at::Tensor>& group_start,
                      const c10::optional<at::Tensor>& group_prefix, int64_t table_cols, int64_t page_size,
                      int64_t total_rows, int64_t hq, int64_t hkv, int64_t window, int64_t shared_rows) {
  TORCH_CHECK(cached.is_cuda(), "paged_work: CUDA tensors expected");
  const auto dev = cached.device();
  c10::cuda::CUDAGuard guard(dev);
  const int64_t B = cached.numel();
  TORCH_CHECK(hkv > 0 && hq > 0 && hq % hkv == 0, "paged_work: ", hq, " query heads on ", hkv, " key heads");
  TORCH_CHECK(group_start.has_value() == group_prefix.has_value(), "paged_work: group_start and group_prefix come together");
  TORCH_CHECK(window >= 0 && window <= INT32_MAX, "paged_work: bad window");
  TORCH_CHECK(shared_rows >= 0 && shared_rows <= total_rows, "paged_work: bad count of shared rows");
  paged::WorkParams p{};
  p.cached = int_vector(cached, B, dev, "cached");
  p.row_start = int_vector(row_start, B + 1, dev, "row_start");
  p.slots = int_vector(slots, B, dev, "slots");
  int64_t NG = 0;
  if (group_start.has_value()) {
    NG = group_prefix->numel();
    TORCH_CHECK(NG <= paged::kMaxSeqs, "page_plan: at most ", paged::kMaxSeqs, " groups");
    p.group_prefix = int_vector(*group_prefix, NG, dev, "group_prefix");
    p.group_start = int_vector(*group_start, NG + 1, dev, "group_start");
  }
  p.B = (int)B; p.NG = (int)NG; p.W = (int)table_cols; p.ps = (int)page_size;
  p.G = (int)(hq / hkv); p.Hkv = (int)hkv; p.window = (int)window; p.max_shared = (int)shared_rows;
  p.max_a = (int)max_units(B, NG, total_rows, p.G, paged::kRowsA);
  p.rows_b = paged::kRowsB / p.G;
  p.max_b = (int)max_units(B, NG, total_rows, p.G, p.rows_b > 0 ? p.rows_b * p.G : paged::kRowsB);
  auto work = at::empty({paged::WorkLayout(B, NG, p.max_a, p.max_b).size}, cached.options());
  p.work = work.data_ptr<int>();
  p.status = status_word_ptr();
  const int smem = (int)(sizeof(int) * (B + NG + 1 + 2 * NG));
  if (smem > 48 * 1024) C10_CUDA_CHECK(cudaFuncSetAttribute(paged::work_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  paged::work_kernel<<<1, 1024, smem, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return work;
}

// Pages as [page, head, 64-column block, slot, 64 columns], fetched in 128-byte swizzled boxes of up to 64 slots of one page
// and head and `blocks` column blocks.
static CUtensorMap page_map(const at::Tensor& t, int blocks) {
  CUtensorMap map;
  const uint64_t e = 2;
  const cuuint64_t dims[5] = {64, (cuuint64_t)t.size(2), (cuuint64_t)t.size(3) / 64, (cuuint64_t)t.size(1), (cuuint64_t)t.size(0)};
  const cuuint64_t strides[4] = {(cuuint64_t)t.stride(2) * e, 128, (cuuint64_t)t.stride(1) * e, (cuuint64_t)t.stride(0) * e};
  const cuuint32_t box[5] = {64, (cuuint32_t)std::min<int64_t>(t.size(2), 64), (cuuint32_t)blocks, 1, 1};
  const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
  const CUresult r = cuTensorMapEncodeTiled(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, t.data_ptr(), dims, strides, box, elem,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (pages) failed with code ", (int)r);
  return map;
}

// Queries [R, Hq, D] as 128-byte wide, swizzled boxes of `rows` rows x the query heads of one key head.
static CUtensorMap query_map(const at::Tensor& q, int group, int rows) {
  CUtensorMap map;
  const cuuint64_t dims[3] = {(cuuint64_t)q.size(2), (cuuint64_t)q.size(1), (cuuint64_t)q.size(0)};
  const cuuint64_t strides[2] = {(cuuint64_t)q.stride(1) * 2, (cuuint64_t)q.stride(0) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)rows};
  const cuuint32_t elem[3] = {1, 1, 1};
  const CUresult r = cuTensorMapEncodeTiled(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q.data_ptr(), dims, strides, box, elem,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (queries) failed with code ", (int)r);
  return map;
}

void paged_attention(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                     const at::Tensor& slots, const at::Tensor& cached, const at::Tensor& row_start, const at::Tensor& work, int64_t groups, int64_t max_rows, int64_t shared_rows,
                     double scale, int64_t window, const c10::optional<at::Tensor>& sinks, at::Tensor out, bool zero_tail) {
  check_pages(k_pages, v_pages, "paged_attention");
  const auto dev = k_pages.device();
  const int64_t R = q.size(0), D = k_pages.size(3), ps = k_pages.size(2);
  TORCH_CHECK(q.device() == dev && q.dim() == 3 && q.scalar_type() == at::kBFloat16 && k_pages.scalar_type() == at::kBFloat16 &&
                  q.size(2) == D && k_pages.size(1) > 0 && q.size(1) > 0 && q.size(1) % k_pages.size(1) == 0,
              "paged_attention: q must be bf16 [R, Hq, D] beside bf16 pages");
  TORCH_CHECK(q.stride(2) == 1 && q.stride(1) % 2 == 0 && q.stride(0) % 2 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 4 == 0,
              "paged_attention: query vectors must be contiguous and 4-byte aligned");
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "paged_attention: unsupported head dimension ", D);
  TORCH_CHECK(ps >= 16 && ps <= 256 && (ps & (ps - 1)) == 0, "paged_attention: unsupported page size ", ps);
  TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == dev &&
                  reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "paged_attention: out must be a contiguous, 16-byte aligned bf16 tensor of q's shape");
  if (sinks.has_value())
    TORCH_CHECK(sinks->device() == dev && sinks->scalar_type() == at::kFloat && sinks->is_contiguous() && sinks->numel() == q.size(1),
                "paged_attention: sinks must be a contiguous fp32 vector [Hq]");
  TORCH_CHECK(table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous());
  TORCH_CHECK(shared_rows >= 0 && shared_rows <= R, "paged_attention: bad count of shared rows");
  c10::cuda::CUDAGuard guard(dev);
  if (R == 0) return;
  const int64_t B = cached.numel();
  paged::AttnParams p{};
  p.q = (const __nv_bfloat16*)q.data_ptr(); p.q_row = q.stride(0); p.q_head = q.stride(1);
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.sinks = sinks.has_value() ? sinks->data_ptr<float>() : nullptr;
  p.table = table.data_ptr<int>();
  p.slots = int_vector(slots, B, dev, "slots");
  p.kp = (const __nv_bfloat16*)k_pages.data_ptr(); p.vp = (const __nv_bfloat16*)v_pages.data_ptr();
  p.kp_page = k_pages.stride(0); p.kp_head = k_pages.stride(1); p.kp_slot = k_pages.stride(2);
  p.vp_page = v_pages.stride(0); p.vp_head = v_pages.stride(1); p.vp_slot = v_pages.stride(2);
  p.cached = int_vector(cached, B, dev, "cached");
  p.row_start = int_vector(row_start, B + 1, dev, "row_start");
  p.B = (int)B; p.NG = (int)groups; p.W = (int)table.size(1); p.R = (int)R;
  p.Hq = (int)q.size(1); p.Hkv = (int)k_pages.size(1); p.G = p.Hq / p.Hkv; p.ps = (int)ps; p.num_pages = (int)k_pages.size(0);
  p.ps_shift = __builtin_ctz((unsigned)ps);
  p.window = (int)window; p.scale_log2 = (float)(scale * 1.4426950408889634); p.zero_tail = zero_tail;
  p.max_shared = groups > 0 ? (int)shared_rows : 0;
  p.max_a = (int)max_units(B, groups, R, p.G, paged::kRowsA);
  p.rows_b = paged::kRowsB / p.G;
  p.max_b = (int)max_units(B, groups, R, p.G, p.rows_b > 0 ? p.rows_b * p.G : paged::kRowsB);
  p.work = int_vector(work, paged::WorkLayout(B, groups, p.max_a, p.max_b).size, dev, "work (made for other heads, rows or groups?)");
  p.status = status_word_ptr();
  // 256-wide heads would need more tensor memory than there is for two accumulators, and a unit holds whole rows of up
  // to 128 query heads per key head: the rest stays on the first kernel.
  p.use_b = D <= 128 && p.rows_b > 0 && max_rows * p.G > paged::kFewPairs;
  p.ctas_a = num_sms() * (D == 256 ? paged::Cfg<256>::kCtasPerSm : paged::Cfg<128>::kCtasPerSm);
  p.ctas_b = num_sms();
  if (p.use_b)
    TORCH_CHECK(q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
                "paged_attention: query vectors must be 16-byte aligned");
  const auto f32 = q.options().dtype(at::kFloat);
  const int64_t na = (int64_t)p.ctas_a * 2 * paged::kRowsA, nb = p.use_b ? (int64_t)p.ctas_b * 2 * paged::kRowsB : 0;
  const int64_t nr = 2 * (int64_t)p.max_shared * p.Hq;
  const int64_t n_cuts = p.ctas_a + p.ctas_b;
  auto scratch = at::empty({(na + nb + nr) * (D + 2) + 4 + n_cuts * (int64_t)(sizeof(paged::Cut) / sizeof(float))}, f32);
  p.part_a = scratch.data_ptr<float>();
  p.part_b = p.part_a + na * D;
  p.row_o = p.part_b + nb * D;
  p.part_a_ml = p.row_o + nr * D;
  p.part_b_ml = p.part_a_ml + na * 2;
  p.row_ml = p.part_b_ml + nb * 2;
  p.cuts = reinterpret_cast<paged::Cut*>(reinterpret_cast<uintptr_t>(p.row_ml + nr * 2 + 3) & ~(uintptr_t)15);
  const int blocks = (int)(D / 64);
  const CUtensorMap mk = page_map(k_pages, blocks), mv = page_map(v_pages, blocks);
  const CUtensorMap mq = p.use_b ? query_map(q, p.G, p.rows_b) : mk;
  const bool split = p.use_b && ps < paged::kTileB && blocks > 1;      // the second kernel's tiles are not whole boxes
  const CUtensorMap bk = split ? page_map(k_pages, 1) : mk, bv = split ? page_map(v_pages, 1) : mv;
  auto stream = at::cuda::getCurrentCUDAStream();
  auto run = [&](auto kernel, int64_t grid, int threads, int smem, bool chained, auto... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = chained ? 1 : 0;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
  };
  auto launch = [&](auto dim) {
    constexpr int kD = decltype(dim)::value;
    static std::atomic<uint64_t> ready{0};       // the shared memory sizes are set once per head dimension and device
    const uint64_t bit = 1ull << (dev.index() & 63);
    if (!(ready.load() & bit)) {
      C10_CUDA_CHECK(cudaFuncSetAttribute(paged::attn_rows_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, paged::Cfg<kD>::kSmem));
      if constexpr (kD <= 128)
        C10_CUDA_CHECK(cudaFuncSetAttribute(paged::attn_block_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, paged::CfgB<kD>::kSmem));
      ready.fetch_or(bit);
    }
    if constexpr (kD <= 128)
      if (p.use_b) run(paged::attn_block_kernel<kD>, p.ctas_b, 320, paged::CfgB<kD>::kSmem, false, mq, bk, bv, p);
    run(paged::attn_rows_kernel<kD>, p.ctas_a, 160, paged::Cfg<kD>::kSmem, p.use_b, mk, mv, p);
    const int64_t row_blocks = std::min<int64_t>(((int64_t)p.max_shared * p.Hq + 3) / 4, (int64_t)num_sms() * 8);
    run(paged::finish_kernel<kD>, p.ctas_a + (p.use_b ? p.ctas_b * paged::kSlices : 0) + row_blocks, 128, 0, true, p);
  };
  if (D == 64) launch(std::integral_constant<int, 64>{});
  else if (D == 128) launch(std::integral_constant<int, 128>{});
  else launch(std::integral_constant<int, 256>{});
}

}  // namespace tb200
