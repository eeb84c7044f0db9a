// Per-head RMSNorm of queries and keys and the rotary embedding in one pass, forward and backward.
//
//   n = x * rsqrt(mean(x^2) + eps) * (w + gain) * scale        y = R(position) n on the first `rot` elements
//   backward: dn = R^T dy, xh = x * r, g = dn (w + gain) scale, dx = r (g - xh mean(g xh)), dw = sum scale dn xh
//
// Bound by HBM: a few flops per byte, every q / k element is read once and written once (the backward recomputes
// the row's rsqrt from x, which it has to read anyway, so the forward stores nothing for it).  A head vector lies
// on kGroup lanes with 8 elements each (16-byte loads), so the sum of squares is log2(kGroup) shuffles and the
// rotate-half partner is one shuffle away.  One warp takes one token and kHeads * (32 / kGroup) of its heads:
// the token's cos / sin values (and the weights) stay in registers for all of them, which keeps table reads at
// one row per warp instead of one per head, and the kHeads independent loads hide latency.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace tb200 {
int* status_word_ptr();

namespace qkn {

constexpr int kE = 8;          // elements per lane
constexpr int kThreads = 256;

struct Params {
  const void* x;               // [T, Hq + 2 Hkv, D], row stride xs
  int64_t xs;
  const void *qw, *kw;         // [D] or null
  const float* table;          // [P, rot] cos | sin, or null (no rotation)
  const int64_t* pos;          // [axes, T]
  const int* axes;             // [rot / 2] axis of each frequency, or null (one axis)
  int n_axes;
  int64_t T;
  int Hq, Hkv, D, rot, P;
  bool interleaved;
  float eps, gain, q_scale;
  int* status;
  // forward
  void *q, *k;                 // [T, Hq, D], [T, Hkv, D]
  // backward
  const void *dq, *dk, *dv;    // row strides below, head stride D; dv may be null (zero)
  int64_t dqs, dks, dvs;
  void* dx;                    // [T, Hq + 2 Hkv, D]
  float* dw_partial;           // [blocks, 2, D] or null
};

// 8 consecutive elements as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[kE]);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&f)[kE]) {
  unpack8(*reinterpret_cast<const bf16x8*>(p), f);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&f)[kE]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[kE]);
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&f)[kE]) {
  *reinterpret_cast<bf16x8*>(p) = pack8(f);
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&f)[kE]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// cos / sin of this lane's 8 elements for one token.  Rotate-half: element e pairs with e +- rot / 2, the lane keeps
// eight values.  Interleaved: pairs (2i, 2i + 1), the lane keeps four.  `sin` carries the sign of the element's own
// combination, so that y = c * self + s * partner in both styles.
struct Turn {
  float c[kE], s[kE];
  bool on;                     // this lane's elements rotate
};

__device__ __forceinline__ int64_t position(const Params& p, int axis, int64_t t) {
  const bool bad_axis = axis < 0 || axis >= p.n_axes;
  int64_t at = bad_axis ? -1 : p.pos[(int64_t)axis * p.T + t];
  if (at < 0 || at >= p.P) {
    atomicOr(p.status, kStatusRopePositionOutOfRange);
    at = at < 0 ? 0 : p.P - 1;
  }
  return at;
}

__device__ __forceinline__ void load_turn(const Params& p, int64_t t, int e0, float sign, Turn& r) {
  const int half = p.rot / 2;
  r.on = p.table != nullptr && e0 < p.rot;
  if (!r.on) return;
  if (p.interleaved) {
    const int f0 = e0 / 2;
    float c[4], s[4];
    if (p.axes == nullptr) {
      const float* row = p.table + position(p, 0, t) * p.rot;
#pragma unroll
      for (int j = 0; j < 4; ++j) { c[j] = row[f0 + j]; s[j] = row[half + f0 + j]; }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* row = p.table + position(p, p.axes[f0 + j], t) * p.rot;
        c[j] = row[f0 + j];
        s[j] = row[half + f0 + j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.c[2 * j] = r.c[2 * j + 1] = c[j];
      r.s[2 * j] = -sign * s[j];
      r.s[2 * j + 1] = sign * s[j];
    }
  } else {
    const bool hi = e0 >= half;
    const int f0 = hi ? e0 - half : e0;
    if (p.axes == nullptr) {
      const float* row = p.table + position(p, 0, t) * p.rot;
      load8(row + f0, r.c);
      load8(row + half + f0, r.s);
    } else {
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        const float* row = p.table + position(p, p.axes[f0 + j], t) * p.rot;
        r.c[j] = row[f0 + j];
        r.s[j] = row[half + f0 + j];
      }
    }
    const float sg = hi ? sign : -sign;
#pragma unroll
    for (int j = 0; j < kE; ++j) r.s[j] *= sg;
  }
}

// y = c * n + s * partner(n).  Every lane of the warp takes part in the shuffles.
__device__ __forceinline__ void rotate(const Params& p, const Turn& r, int partner_lane, float (&n)[kE]) {
  if (p.table == nullptr) return;
  if (p.interleaved) {
    if (r.on) {
#pragma unroll
      for (int j = 0; j < kE; j += 2) {
        const float a = n[j], b = n[j + 1];
        n[j] = r.c[j] * a + r.s[j] * b;
        n[j + 1] = r.c[j + 1] * b + r.s[j + 1] * a;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const float o = __shfl_sync(0xffffffffu, n[j], partner_lane);
      if (r.on) n[j] = r.c[j] * n[j] + r.s[j] * o;
    }
  }
}

__device__ __forceinline__ int partner_of(const Params& p, int lane, int e0) {
  const int half = p.rot / 2;
  if (p.table == nullptr || p.interleaved || e0 >= p.rot) return lane;
  return e0 < half ? lane + half / kE : lane - half / kE;
}

template <int kGroup>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = kGroup / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ void load_gain(const void* w, float gain, float scale, int e0, bool live, float (&g)[kE]) {
  if (w != nullptr && live) {
    load8(reinterpret_cast<const T*>(w) + e0, g);
#pragma unroll
    for (int j = 0; j < kE; ++j) g[j] = (g[j] + gain) * scale;
  } else {
#pragma unroll
    for (int j = 0; j < kE; ++j) g[j] = scale;
  }
}

template <typename T, int kGroup, int kHeads>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Params p) {
  constexpr int kPar = 32 / kGroup;            // heads side by side in a warp
  constexpr int kChunk = kPar * kHeads;
  const int lane = threadIdx.x & 31;
  const int sub = lane / kGroup, e0 = (lane % kGroup) * kE;
  const bool live = e0 < p.D;
  const int partner = partner_of(p, lane, e0);
  const int cq = (p.Hq + kChunk - 1) / kChunk, ck = (p.Hkv + kChunk - 1) / kChunk;
  const int64_t total = p.T * (cq + ck);
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); it < total; it += stride) {
    const int64_t t = it / (cq + ck);
    const int c = (int)(it % (cq + ck));
    const bool is_q = c < cq;
    const int H = is_q ? p.Hq : p.Hkv;
    const int h0 = (is_q ? c : c - cq) * kChunk + sub;
    const T* xr = reinterpret_cast<const T*>(p.x) + t * p.xs + (is_q ? 0 : (int64_t)p.Hq * p.D) + e0;
    T* yr = reinterpret_cast<T*>(is_q ? p.q : p.k) + t * H * p.D + e0;
    float x[kHeads][kE];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i * kPar;
      if (live && h < H) {
        load8(xr + (int64_t)h * p.D, x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < kE; ++j) x[i][j] = 0.f;
      }
    }
    Turn turn;
    load_turn(p, t, e0, 1.f, turn);
    float g[kE];
    load_gain<T>(is_q ? p.qw : p.kw, p.gain, is_q ? p.q_scale : 1.f, e0, live, g);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < kE; ++j) ss += x[i][j] * x[i][j];
      const float r = rsqrtf(group_sum<kGroup>(ss) / (float)p.D + p.eps);
#pragma unroll
      for (int j = 0; j < kE; ++j) x[i][j] *= r * g[j];
      rotate(p, turn, partner, x[i]);
      const int h = h0 + i * kPar;
      if (live && h < H) store8(yr + (int64_t)h * p.D, x[i]);
    }
  }
}

template <typename T, int kGroup, int kHeads>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const Params p) {
  constexpr int kPar = 32 / kGroup;
  constexpr int kChunk = kPar * kHeads;
  __shared__ float red[kThreads / 32][2][kGroup * kE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / kGroup, e0 = (lane % kGroup) * kE;
  const bool live = e0 < p.D;
  const int partner = partner_of(p, lane, e0);
  const int cq = (p.Hq + kChunk - 1) / kChunk, ck = (p.Hkv + kChunk - 1) / kChunk;
  const int per = cq + 2 * ck;
  const int64_t total = p.T * per;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32);
  float dwq[kE], dwk[kE];
#pragma unroll
  for (int j = 0; j < kE; ++j) dwq[j] = dwk[j] = 0.f;
  const int64_t dxs = (int64_t)(p.Hq + 2 * p.Hkv) * p.D;
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / 32) + warp; it < total; it += stride) {
    const int64_t t = it / per;
    const int c = (int)(it % per);
    if (c >= cq + ck) {                        // values pass through
      const int h0 = (c - cq - ck) * kChunk + sub;
      T* out = reinterpret_cast<T*>(p.dx) + t * dxs + (int64_t)(p.Hq + p.Hkv) * p.D + e0;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i * kPar;
        if (live && h < p.Hkv) {
          float f[kE];
          if (p.dv != nullptr) {
            load8(reinterpret_cast<const T*>(p.dv) + t * p.dvs + (int64_t)h * p.D + e0, f);
          } else {
#pragma unroll
            for (int j = 0; j < kE; ++j) f[j] = 0.f;
          }
          store8(out + (int64_t)h * p.D, f);
        }
      }
      continue;
    }
    const bool is_q = c < cq;
    const int H = is_q ? p.Hq : p.Hkv;
    const int h0 = (is_q ? c : c - cq) * kChunk + sub;
    const int64_t part = is_q ? 0 : (int64_t)p.Hq * p.D;
    const T* xr = reinterpret_cast<const T*>(p.x) + t * p.xs + part + e0;
    const T* dr = reinterpret_cast<const T*>(is_q ? p.dq : p.dk) + t * (is_q ? p.dqs : p.dks) + e0;
    T* out = reinterpret_cast<T*>(p.dx) + t * dxs + part + e0;
    float x[kHeads][kE], d[kHeads][kE];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i * kPar;
      if (live && h < H) {
        load8(xr + (int64_t)h * p.D, x[i]);
        load8(dr + (int64_t)h * p.D, d[i]);
      } else {
#pragma unroll
        for (int j = 0; j < kE; ++j) x[i][j] = d[i][j] = 0.f;
      }
    }
    Turn turn;
    load_turn(p, t, e0, -1.f, turn);           // the transposed rotation
    const float scale = is_q ? p.q_scale : 1.f;
    float g[kE];
    load_gain<T>(is_q ? p.qw : p.kw, p.gain, scale, e0, live, g);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < kE; ++j) ss += x[i][j] * x[i][j];
      const float r = rsqrtf(group_sum<kGroup>(ss) / (float)p.D + p.eps);
      rotate(p, turn, partner, d[i]);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < kE; ++j) {
        x[i][j] *= r;
        const float w = d[i][j] * x[i][j] * scale;
        if (is_q) dwq[j] += w; else dwk[j] += w;
        d[i][j] *= g[j];
        dot += d[i][j] * x[i][j];
      }
      const float m = group_sum<kGroup>(dot) / (float)p.D;
#pragma unroll
      for (int j = 0; j < kE; ++j) d[i][j] = r * (d[i][j] - x[i][j] * m);
      const int h = h0 + i * kPar;
      if (live && h < H) store8(out + (int64_t)h * p.D, d[i]);
    }
  }
  if (p.dw_partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < kE; ++j) {
#pragma unroll
    for (int o = 16; o >= kGroup; o >>= 1) {
      dwq[j] += __shfl_xor_sync(0xffffffffu, dwq[j], o);
      dwk[j] += __shfl_xor_sync(0xffffffffu, dwk[j], o);
    }
    if (sub == 0) {
      red[warp][0][e0 + j] = dwq[j];
      red[warp][1][e0 + j] = dwk[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.D; i += kThreads) {
    const int which = i / p.D, e = i % p.D;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) s += red[w][which][e];
    p.dw_partial[((int64_t)blockIdx.x * 2 + which) * p.D + e] = s;
  }
}

// Column sums of the per-block partial weight gradients [parts, cols] in a fixed order: the result does not depend on
// the schedule.  One block of 8 x 32 threads per 32 columns.
__global__ void __launch_bounds__(256) sum_partials_kernel(const float* __restrict__ partial, float* __restrict__ out, int parts,
                                                           int cols) {
  __shared__ float tile[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (col < cols)
    for (int i = ty; i < parts; i += 8) s += partial[(int64_t)i * cols + col];
  tile[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && col < cols) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a += tile[i][tx];
    out[col] = a;
  }
}

}  // namespace qkn

// Lanes per head: the power of two that holds D / 8 vectors.
#define TB_QKN_GROUP(D, ...)                                 \
  if ((D) <= 32) { constexpr int kGroup = 4; __VA_ARGS__(); }        \
  else if ((D) <= 64) { constexpr int kGroup = 8; __VA_ARGS__(); }   \
  else if ((D) <= 128) { constexpr int kGroup = 16; __VA_ARGS__(); } \
  else { constexpr int kGroup = 32; __VA_ARGS__(); }

static void qkn_fill(qkn::Params& p, const at::Tensor& x, int64_t hq, int64_t hkv, const c10::optional<at::Tensor>& qw,
                     const c10::optional<at::Tensor>& kw, const c10::optional<at::Tensor>& table,
                     const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& axes, bool interleaved,
                     double eps, double gain, double q_scale) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && hq > 0 && hkv > 0 && x.size(1) == hq + 2 * hkv,
              "qk_norm_rope: x must be a CUDA tensor [T, Hq + 2 Hkv, D]");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, "qk_norm_rope: unsupported dtype ", x.scalar_type());
  const int64_t D = x.size(2);
  TORCH_CHECK(D % 8 == 0 && D >= 8 && D <= 256, "qk_norm_rope: the head dimension must be a multiple of 8 up to 256, got ", D);
  TORCH_CHECK(x.stride(2) == 1 && x.stride(1) == D && x.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "qk_norm_rope: heads must be adjacent and rows 16-byte aligned");
  auto weight = [&](const c10::optional<at::Tensor>& w) -> const void* {
    if (!w.has_value()) return nullptr;
    TORCH_CHECK(w->device() == x.device() && w->is_contiguous() && w->numel() == D && w->scalar_type() == x.scalar_type() &&
                    reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 == 0,
                "qk_norm_rope: weights must be contiguous, 16-byte aligned [D] tensors of x's dtype and device");
    return w->data_ptr();
  };
  p.x = x.data_ptr();
  p.xs = x.stride(0);
  p.qw = weight(qw);
  p.kw = weight(kw);
  p.T = x.size(0);
  p.Hq = (int)hq; p.Hkv = (int)hkv; p.D = (int)D;
  p.table = nullptr; p.pos = nullptr; p.axes = nullptr; p.n_axes = 1; p.rot = 0; p.P = 0;
  if (table.has_value()) {
    TORCH_CHECK(table->device() == x.device() && table->scalar_type() == at::kFloat && table->is_contiguous() && table->dim() == 2 &&
                    table->size(0) > 0 && table->size(0) <= INT32_MAX && reinterpret_cast<uintptr_t>(table->data_ptr()) % 16 == 0,
                "qk_norm_rope: table must be a contiguous fp32 matrix [positions, rot] on x's device");
    const int64_t rot = table->size(1);
    TORCH_CHECK(rot > 0 && rot <= D && (interleaved ? rot % 8 == 0 : rot % 16 == 0),
                "qk_norm_rope: the rotary width must be a multiple of ", interleaved ? 8 : 16, " up to the head dimension, got ", rot);
    TORCH_CHECK(positions.has_value() && positions->device() == x.device() && positions->scalar_type() == at::kLong &&
                    positions->is_contiguous(),
                "qk_norm_rope: positions must be contiguous int64 on x's device");
    if (axes.has_value()) {
      TORCH_CHECK(axes->device() == x.device() && axes->scalar_type() == at::kInt && axes->is_contiguous() && axes->numel() == rot / 2,
                  "qk_norm_rope: axes must be a contiguous int32 tensor [rot / 2] on x's device");
      TORCH_CHECK(positions->dim() == 2 && positions->size(1) == x.size(0) && positions->size(0) > 0, "qk_norm_rope: with axes, positions must be [axes, T]");
      p.axes = axes->data_ptr<int>();
      p.n_axes = (int)positions->size(0);
    } else {
      TORCH_CHECK(positions->dim() == 1 && positions->size(0) == x.size(0), "qk_norm_rope: positions must be [T]");
    }
    p.table = table->data_ptr<float>();
    p.pos = positions->data_ptr<int64_t>();
    p.rot = (int)rot;
    p.P = (int)table->size(0);
  }
  p.interleaved = interleaved;
  p.eps = (float)eps; p.gain = (float)gain; p.q_scale = (float)q_scale;
  p.status = status_word_ptr();
}

// Heads per lane group: four when that still leaves every SM its 64 warps' worth of items, else one, so that a decode
// step of a few tokens spreads over the SMs.
static bool qkn_wide(const qkn::Params& p, int group) {
  const int64_t chunk = 4 * (32 / group);
  return p.T * ((p.Hq + chunk - 1) / chunk + (p.Hkv + chunk - 1) / chunk) >= (int64_t)num_sms() * 16;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& x, int64_t hq, int64_t hkv, const c10::optional<at::Tensor>& qw,
                                                    const c10::optional<at::Tensor>& kw, const c10::optional<at::Tensor>& table,
                                                    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& axes,
                                                    bool interleaved, double eps, double gain, double q_scale) {
  TORCH_CHECK(x.is_cuda(), "qk_norm_rope: x must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x.device());
  qkn::Params p{};
  qkn_fill(p, x, hq, hkv, qw, kw, table, positions, axes, interleaved, eps, gain, q_scale);
  auto q = at::empty({p.T, hq, p.D}, x.options());
  auto k = at::empty({p.T, hkv, p.D}, x.options());
  if (p.T == 0) return {q, k};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  auto stream = at::cuda::getCurrentCUDAStream();
  TB_QKN_GROUP(p.D, [&] {
    auto launch = [&](auto heads) {
      constexpr int kHeads = decltype(heads)::value;
      const int64_t chunk = kHeads * (32 / kGroup);
      const int64_t items = p.T * ((p.Hq + chunk - 1) / chunk + (p.Hkv + chunk - 1) / chunk);
      const int grid = (int)std::min<int64_t>((items + 7) / 8, (int64_t)num_sms() * 32);
      if (x.scalar_type() == at::kBFloat16) qkn::fwd_kernel<__nv_bfloat16, kGroup, kHeads><<<grid, qkn::kThreads, 0, stream>>>(p);
      else qkn::fwd_kernel<float, kGroup, kHeads><<<grid, qkn::kThreads, 0, stream>>>(p);
    };
    if (qkn_wide(p, kGroup)) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 1>{});
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, k};
}

// Returns dx of x's shape (contiguous) and the fp32 weight gradients [2, D] (empty without weights).
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_bwd(const at::Tensor& dq, const at::Tensor& dk, const c10::optional<at::Tensor>& dv,
                                                    const at::Tensor& x, int64_t hq, int64_t hkv, const c10::optional<at::Tensor>& qw,
                                                    const c10::optional<at::Tensor>& kw, const c10::optional<at::Tensor>& table,
                                                    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& axes,
                                                    bool interleaved, double eps, double gain, double q_scale) {
  TORCH_CHECK(x.is_cuda(), "qk_norm_rope: x must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x.device());
  qkn::Params p{};
  qkn_fill(p, x, hq, hkv, qw, kw, table, positions, axes, interleaved, eps, gain, q_scale);
  auto grad = [&](const at::Tensor& g, int64_t heads, int64_t& stride) -> const void* {
    TORCH_CHECK(g.device() == x.device() && g.scalar_type() == x.scalar_type() && g.dim() == 3 && g.size(0) == p.T && g.size(1) == heads &&
                    g.size(2) == p.D && g.stride(2) == 1 && g.stride(1) == p.D && g.stride(0) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0,
                "qk_norm_rope: gradients must be [T, heads, D] of x's dtype with adjacent heads and 16-byte aligned rows");
    stride = g.stride(0);
    return g.data_ptr();
  };
  const bool has_w = qw.has_value() || kw.has_value();
  auto dx = at::empty({p.T, hq + 2 * hkv, p.D}, x.options());
  auto dw = at::empty({has_w ? 2 : 0, p.D}, x.options().dtype(at::kFloat));
  if (p.T == 0) return {dx, dw.zero_()};
  p.dq = grad(dq, hq, p.dqs);
  p.dk = grad(dk, hkv, p.dks);
  if (dv.has_value()) p.dv = grad(*dv, hkv, p.dvs);
  p.dx = dx.data_ptr();
  auto stream = at::cuda::getCurrentCUDAStream();
  at::Tensor partial;
  int grid = 0;
  TB_QKN_GROUP(p.D, [&] {
    auto launch = [&](auto heads) {
      constexpr int kHeads = decltype(heads)::value;
      const int64_t chunk = kHeads * (32 / kGroup);
      const int64_t items = p.T * ((p.Hq + chunk - 1) / chunk + 2 * ((p.Hkv + chunk - 1) / chunk));
      grid = (int)std::min<int64_t>((items + 7) / 8, (int64_t)num_sms() * 4);
      if (has_w) {
        partial = at::empty({grid, 2, p.D}, x.options().dtype(at::kFloat));
        p.dw_partial = partial.data_ptr<float>();
      }
      if (x.scalar_type() == at::kBFloat16) qkn::bwd_kernel<__nv_bfloat16, kGroup, kHeads><<<grid, qkn::kThreads, 0, stream>>>(p);
      else qkn::bwd_kernel<float, kGroup, kHeads><<<grid, qkn::kThreads, 0, stream>>>(p);
    };
    if (qkn_wide(p, kGroup)) launch(std::integral_constant<int, 2>{});
    else launch(std::integral_constant<int, 1>{});
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (has_w) {
    qkn::sum_partials_kernel<<<(2 * p.D + 31) / 32, 256, 0, stream>>>(partial.data_ptr<float>(), dw.data_ptr<float>(), grid, 2 * p.D);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {dx, dw};
}

}  // namespace tb200
