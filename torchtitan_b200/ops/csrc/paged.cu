// Paged key / value cache: the step plan (block tables, positions, slot map), the scatter of new rows into pages, and
// attention of the new rows over their sequences' pages.
//
// A pool holds pages [num_pages, Hkv, page_size, D] per layer for keys and for values; a sequence's pages are the ids in
// its row of the block table.  Bad ids, slots and lengths come from the device and cannot be refused on the host: the
// kernels check every index before they use it, skip the access and set kStatusPagePlanInvalid.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace tb200 {
int* status_word_ptr();

namespace paged {

constexpr int kMaxSeqs = 4096;          // sequences of one step: their offsets live in shared memory
constexpr int kMaxSlots = 65536;        // rows of the block table: one bit each in shared memory
constexpr int kMaxCols = 1 << 20;       // columns of the block table and rows of a step: a block's scan stays inside 32 bits
constexpr int kMaxRows = 1 << 22;
constexpr int kMaxLength = 1 << 30;     // tokens of one sequence

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
// one round of dependent loads.
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
        bad |= end > p.W;
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

// A copy: one 16-byte vector of a key and of the value beside it per thread and step.
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
struct SimpleParams {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  const __nv_bfloat16 *kp, *vp;
  int64_t kp_page, kp_head, kp_slot, vp_page, vp_head, vp_slot;   // in elements
  const int *table, *slots, *cached, *row_start;
  const float* sinks;
  __nv_bfloat16* out;                     // [R, Hq, D]
  int B, S, W, R, Hq, Hkv, D, ps, num_pages, window;
  float scale;
  bool zero_tail;
  int* status;
};

// One block of four warps per (row, query head); a warp takes every fourth key, its lanes hold D / 32 elements each.
__global__ void __launch_bounds__(128) simple_kernel(const SimpleParams p) {
  __shared__ float sm_m[4], sm_l[4], sm_o[4][256];
  const int r = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = p.D / 32;
  __nv_bfloat16* out = p.out + ((int64_t)r * p.Hq + h) * p.D;
  if (r >= p.row_start[p.B]) {
    if (p.zero_tail)
      for (int d = threadIdx.x; d < p.D; d += 128) out[d] = __float2bfloat16_rn(0.f);
    return;
  }
  const int b = find_segment(p.row_start, p.B, r);
  const int slot = p.slots[b];
  const int pos = p.cached[b] + r - p.row_start[b];
  const int kv = h / (p.Hq / p.Hkv);
  float q[8], o[8];
  for (int i = 0; i < 8; ++i) {
    o[i] = 0.f;
    q[i] = i < per ? __bfloat162float(p.q[r * p.q_row + h * p.q_head + lane * per + i]) : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int64_t last = min((int64_t)pos, (int64_t)p.W * p.ps - 1);
  for (int64_t j = (p.window > 0 ? max(0, pos - p.window + 1) : 0) + warp; j <= last; j += 4) {
    const int page = p.table[(int64_t)slot * p.W + j / p.ps];
    if (page < 0 || page >= p.num_pages) {
      atomicOr(p.status, kStatusPagePlanInvalid);
      continue;
    }
    const __nv_bfloat16* k = p.kp + page * p.kp_page + kv * p.kp_head + (j % p.ps) * p.kp_slot + lane * per;
    const __nv_bfloat16* v = p.vp + page * p.vp_page + kv * p.vp_head + (j % p.ps) * p.vp_slot + lane * per;
    float s = 0.f;
    for (int i = 0; i < per; ++i) s += q[i] * __bfloat162float(k[i]);
    s = warp_sum(s) * p.scale;
    const float mn = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(s - mn);
    m = mn;
    l = l * a + w;
    for (int i = 0; i < per; ++i) o[i] = o[i] * a + w * __bfloat162float(v[i]);
  }
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
  for (int i = 0; i < per; ++i) sm_o[warp][lane * per + i] = o[i];
  __syncthreads();
  float mm = p.sinks != nullptr ? p.sinks[h] : -INFINITY;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm_m[w]);
  float den = p.sinks != nullptr && mm != -INFINITY ? expf(p.sinks[h] - mm) : 0.f;
  float f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = sm_m[w] == -INFINITY ? 0.f : expf(sm_m[w] - mm);
    den += f[w] * sm_l[w];
  }
  for (int d = threadIdx.x; d < p.D; d += 128) {
    float s = 0.f;
    for (int w = 0; w < 4; ++w) s += f[w] * sm_o[w][d];
    out[d] = __float2bfloat16_rn(den > 0.f ? s / den : 0.f);
  }
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

void paged_attention_simple(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                            const at::Tensor& slots, const at::Tensor& cached, const at::Tensor& row_start, double scale, int64_t window,
                            const c10::optional<at::Tensor>& sinks, at::Tensor out, bool zero_tail) {
  check_pages(k_pages, v_pages, "paged_attention");
  const auto dev = k_pages.device();
  TORCH_CHECK(q.device() == dev && q.dim() == 3 && q.scalar_type() == at::kBFloat16 && k_pages.scalar_type() == at::kBFloat16 &&
                  q.size(2) == k_pages.size(3) && q.stride(2) == 1 && q.size(1) % k_pages.size(1) == 0,
              "paged_attention: q must be bf16 [R, Hq, D] beside bf16 pages");
  TORCH_CHECK(q.size(2) % 32 == 0 && q.size(2) <= 256, "paged_attention: unsupported head dimension ", q.size(2));
  TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == dev);
  c10::cuda::CUDAGuard guard(dev);
  if (q.numel() == 0) return;
  paged::SimpleParams p{};
  p.q = (const __nv_bfloat16*)q.data_ptr(); p.q_row = q.stride(0); p.q_head = q.stride(1);
  p.kp = (const __nv_bfloat16*)k_pages.data_ptr(); p.vp = (const __nv_bfloat16*)v_pages.data_ptr();
  p.kp_page = k_pages.stride(0); p.kp_head = k_pages.stride(1); p.kp_slot = k_pages.stride(2);
  p.vp_page = v_pages.stride(0); p.vp_head = v_pages.stride(1); p.vp_slot = v_pages.stride(2);
  p.table = table.data_ptr<int>(); p.slots = slots.data_ptr<int>(); p.cached = cached.data_ptr<int>(); p.row_start = row_start.data_ptr<int>();
  p.sinks = sinks.has_value() ? sinks->data_ptr<float>() : nullptr;
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.B = (int)slots.numel(); p.S = (int)table.size(0); p.W = (int)table.size(1); p.R = (int)q.size(0);
  p.Hq = (int)q.size(1); p.Hkv = (int)k_pages.size(1); p.D = (int)q.size(2); p.ps = (int)k_pages.size(2);
  p.num_pages = (int)k_pages.size(0); p.window = (int)window; p.scale = (float)scale; p.zero_tail = zero_tail;
  p.status = status_word_ptr();
  paged::simple_kernel<<<p.R * p.Hq, 128, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace tb200
