// Per-head RMSNorm of queries and keys and the rotary embedding in one pass, forward and backward.
//
//   n = x * rsqrt(mean(x^2) + eps) * (w + gain) * scale        y = R(position) n on the first `rot` elements
//   backward: dn = R^T dy, xh = x * r, g = dn (w + gain) scale, dx = r (g - xh mean(g xh)), dw = sum scale dn xh
//
// Bound by HBM: a few flops per byte, every q / k element is read once and written once (the backward recomputes
// the row's rsqrt from x, which it has to read anyway, so the forward stores nothing for it).  A head vector lies
// on kGroup lanes with 8 elements each (16-byte loads), so the sum of squares is log2(kGroup) shuffles and the
// rotate-half partner is one shuffle of the packed values away.  A warp owns kHeads * (32 / kGroup) heads of one kind and
// walks over tokens: the gains and the weight gradient's sums stay in registers and a token's cos / sin are read once for
// all its heads.  The next token's vectors are on their way into shared memory meanwhile (cp.async, kStages tokens deep):
// with loads into registers alone a warp waited out the latency of every token, and the registers that more warps or more
// loads in flight would have needed were not there.  A lane reads back what it copied itself, so nothing is synchronised.
// 8192 tokens, 32 + 4 heads of 128, bf16: forward 33 us for 155 MB (4.7 TB/s), backward 59 us for 247 MB (4.2 TB/s).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace tb200 {
int* status_word_ptr();

namespace qkn {

constexpr int kE = 8;          // elements per lane
constexpr int kThreads = 128;
// Resident blocks per SM: what the registers allow without spilling.
template <typename T>
constexpr int kFwdBlocks = sizeof(T) == 2 ? 6 : 4;
template <typename T>
constexpr int kBwdBlocks = 4;

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

// Two fp32 values in one register pair: the packed instructions halve the arithmetic, which would else bound the kernels.
using F2 = uint64_t;
constexpr int kP = kE / 2;
constexpr int kStages = 2;     // tokens in flight per warp: the one at hand and the next (three and four gained nothing)
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(F2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 swap2(F2 v) {
  float lo, hi;
  split(v, lo, hi);
  return f2(hi, lo);
}
__device__ __forceinline__ float sum2(F2 v) {
  float lo, hi;
  split(v, lo, hi);
  return lo + hi;
}

// 8 consecutive elements as they are stored, and as four fp32 pairs.
template <typename T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint32_t v[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = v[2] = v[3] = 0u; }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]); }
  __device__ __forceinline__ void get(F2 (&f)[kP]) const {
#pragma unroll
    for (int j = 0; j < kP; ++j) f[j] = f2(__uint_as_float(v[j] << 16), __uint_as_float(v[j] & 0xffff0000u));
  }
  __device__ __forceinline__ void set(const F2 (&f)[kP]) {
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      float lo, hi;
      split(f[j], lo, hi);
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      v[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  __device__ __forceinline__ Raw from_lane(int lane) const {
    Raw r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = __shfl_sync(0xffffffffu, v[j], lane);
    return r;
  }
};
template <>
struct Raw<float> {
  F2 v[kP];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = f2(a.x, a.y); v[1] = f2(a.z, a.w); v[2] = f2(b.x, b.y); v[3] = f2(b.z, b.w);
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = v[2] = v[3] = 0ull; }
  __device__ __forceinline__ void store(float* p) const {
    float4 a, b;
    split(v[0], a.x, a.y); split(v[1], a.z, a.w); split(v[2], b.x, b.y); split(v[3], b.z, b.w);
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void get(F2 (&f)[kP]) const {
#pragma unroll
    for (int j = 0; j < kP; ++j) f[j] = v[j];
  }
  __device__ __forceinline__ void set(const F2 (&f)[kP]) {
#pragma unroll
    for (int j = 0; j < kP; ++j) v[j] = f[j];
  }
  __device__ __forceinline__ Raw from_lane(int lane) const {
    Raw r;
#pragma unroll
    for (int j = 0; j < kP; ++j) r.v[j] = __shfl_sync(0xffffffffu, v[j], lane);
    return r;
  }
};

// A lane's kE elements -> its own place in shared memory; zeros when `live` is false.
template <typename T>
__device__ __forceinline__ void copy_async(uint32_t dst, const T* src, bool live) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * 512), "l"(reinterpret_cast<const char*>(src) + i * 16),
                 "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }
template <typename T>
__device__ __forceinline__ Raw<T> copied(const uint8_t* at) {
  Raw<T> r;
  if constexpr (sizeof(T) == 2) {
    r.load(reinterpret_cast<const T*>(at));
  } else {
    const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 512);
    r.v[0] = f2(a.x, a.y); r.v[1] = f2(a.z, a.w); r.v[2] = f2(b.x, b.y); r.v[3] = f2(b.z, b.w);
  }
  return r;
}
template <typename T>
constexpr int kVector = 32 * kE * sizeof(T);     // a warp's vectors of one load

__device__ __forceinline__ int64_t position(const Params& p, int axis, int64_t t) {
  const bool bad_axis = axis < 0 || axis >= p.n_axes;
  int64_t at = bad_axis ? -1 : p.pos[(int64_t)axis * p.T + t];
  if (at < 0 || at >= p.P) {
    atomicOr(p.status, kStatusRopePositionOutOfRange);
    at = at < 0 ? 0 : p.P - 1;
  }
  return at;
}

// What a lane knows of its place: its elements, whether they rotate and where its rotate-half partner sits.
struct Place {
  int sub, e0, partner;
  bool live, turns, upper;
  template <int kGroup>
  static __device__ __forceinline__ Place make(const Params& p) {
    const int lane = threadIdx.x & 31, half = p.rot / 2;
    Place q;
    q.sub = lane / kGroup;
    q.e0 = (lane % kGroup) * kE;
    q.live = q.e0 < p.D;
    q.turns = q.e0 < p.rot;                      // rot is 0 without a table
    q.upper = !p.interleaved && q.e0 >= half;
    q.partner = q.turns && !p.interleaved ? (q.upper ? lane - half / kE : lane + half / kE) : lane;
    return q;
  }
};

// cos and signed sin of a lane's 8 elements for one token, such that y = c * n + s * partner(n): the partner of element e
// is e +- rot / 2 on another lane (rotate-half) or e ^ 1 (interleaved).  `sign` = -1 gives the transposed rotation.
// `row0` is the token's row of the table when there is one axis (fetched a token ahead).
__device__ __forceinline__ void load_turn(const Params& p, const Place& at, int64_t t, int64_t row0, float sign, F2 (&c)[kP], F2 (&s)[kP]) {
  if (!at.turns) {
#pragma unroll
    for (int j = 0; j < kP; ++j) { c[j] = f2(1.f, 1.f); s[j] = 0ull; }
    return;
  }
  const int half = p.rot / 2;
  if (p.interleaved) {
    const int f0 = at.e0 / 2;
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      const float* row = p.table + (p.axes == nullptr ? row0 : position(p, p.axes[f0 + j], t)) * p.rot;
      const float cc = row[f0 + j], ss = sign * row[half + f0 + j];
      c[j] = f2(cc, cc);
      s[j] = f2(-ss, ss);
    }
    return;
  }
  const int f0 = at.upper ? at.e0 - half : at.e0;
  Raw<float> a, b;
  if (p.axes == nullptr) {
    const float* row = p.table + row0 * p.rot;
    a.load(row + f0);
    b.load(row + half + f0);
  } else {
    float cc[kE], ss[kE];
#pragma unroll
    for (int j = 0; j < kE; ++j) {
      const float* row = p.table + position(p, p.axes[f0 + j], t) * p.rot;
      cc[j] = row[f0 + j];
      ss[j] = row[half + f0 + j];
    }
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      a.v[j] = f2(cc[2 * j], cc[2 * j + 1]);
      b.v[j] = f2(ss[2 * j], ss[2 * j + 1]);
    }
  }
  const float sg = at.upper ? sign : -sign;
#pragma unroll
  for (int j = 0; j < kP; ++j) {
    c[j] = a.v[j];
    s[j] = mul2(b.v[j], f2(sg, sg));
  }
}

__device__ __forceinline__ int64_t table_row(const Params& p, int64_t t) {
  return p.table != nullptr && p.axes == nullptr && t < p.T ? position(p, 0, t) : 0;
}

template <int kGroup>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = kGroup / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ void load_gain(const void* w, float gain, float scale, int e0, bool live, F2 (&g)[kP]) {
#pragma unroll
  for (int j = 0; j < kP; ++j) g[j] = f2(scale, scale);
  if (w != nullptr && live) {
    Raw<T> r;
    r.load(reinterpret_cast<const T*>(w) + e0);
    F2 f[kP];
    r.get(f);
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      float lo, hi;
      split(f[j], lo, hi);
      g[j] = f2((lo + gain) * scale, (hi + gain) * scale);
    }
  }
}

// The partner's values of a lane's elements.
template <typename T>
__device__ __forceinline__ void partner_of(const Params& p, const Place& at, const Raw<T>& x, F2 (&o)[kP]) {
  if (p.interleaved) {
    x.get(o);
#pragma unroll
    for (int j = 0; j < kP; ++j) o[j] = swap2(o[j]);
  } else {
    x.from_lane(at.partner).get(o);
  }
}

template <typename T, int kGroup, int kHeads>
__global__ void __launch_bounds__(kThreads, kFwdBlocks<T>) fwd_kernel(const Params p) {
  constexpr int kPar = 32 / kGroup;              // heads side by side in a warp
  constexpr int kChunk = kPar * kHeads;
  const Place at = Place::make<kGroup>(p);
  const int cq = (p.Hq + kChunk - 1) / kChunk, per = cq + (p.Hkv + kChunk - 1) / kChunk;
  const int warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int step = gridDim.x * (kThreads / 32) / per;
  const int chunk = warp % per;
  const bool is_q = chunk < cq;
  const int H = is_q ? p.Hq : p.Hkv;
  const int h0 = (is_q ? chunk : chunk - cq) * kChunk + at.sub;
  if (warp / per >= step) return;
  // y = r (c g x + s g' x') with the gains of the element and of its partner
  F2 g[kP], gp[kP];
  load_gain<T>(is_q ? p.qw : p.kw, p.gain, is_q ? p.q_scale : 1.f, at.e0, at.live, g);
  {
    Raw<float> mine;
    mine.set(g);
    partner_of<float>(p, at, mine, gp);
  }
  const T* xb = reinterpret_cast<const T*>(p.x) + (is_q ? 0 : (int64_t)p.Hq * p.D) + (int64_t)h0 * p.D + at.e0;
  T* yb = reinterpret_cast<T*>(is_q ? p.q : p.k) + (int64_t)h0 * p.D + at.e0;
  const float inv_d = 1.f / (float)p.D;
  extern __shared__ __align__(16) uint8_t ring[];
  uint8_t* mine = ring + (threadIdx.x >> 5) * (kStages * kHeads * kVector<T>) + (threadIdx.x & 31) * 16;
  const uint32_t mine_s = (uint32_t)__cvta_generic_to_shared(mine);
  auto fetch = [&](int64_t t, int stage) {
    if (t < p.T) {
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const bool on = at.live && h0 + i * kPar < H;
        copy_async<T>(mine_s + (stage * kHeads + i) * kVector<T>, on ? xb + t * p.xs + i * kPar * p.D : xb, on);
      }
    }
    copies_commit();
  };
  const int64_t first = warp / per;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(first + (int64_t)i * step, i);
  int64_t row = table_row(p, first);
  int stage = 0;
  for (int64_t t = first; t < p.T; t += step) {
    T* yr = yb + t * H * p.D;
    fetch(t + (int64_t)(kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
    F2 c[kP], s[kP];
    load_turn(p, at, t, row, 1.f, c, s);
    row = table_row(p, t + step);
    copies_wait<kStages - 1>();
    const uint8_t* here = mine + stage * kHeads * kVector<T>;
    stage = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
    for (int j = 0; j < kP; ++j) {
      c[j] = mul2(c[j], g[j]);
      s[j] = mul2(s[j], gp[j]);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const Raw<T> x = copied<T>(here + i * kVector<T>);
      F2 f[kP], o[kP];
      x.get(f);
      partner_of<T>(p, at, x, o);
      F2 ss = mul2(f[0], f[0]);
#pragma unroll
      for (int j = 1; j < kP; ++j) ss = fma2(f[j], f[j], ss);
      const float r = rsqrtf(group_sum<kGroup>(sum2(ss)) * inv_d + p.eps);
#pragma unroll
      for (int j = 0; j < kP; ++j) f[j] = mul2(f2(r, r), fma2(c[j], f[j], mul2(s[j], o[j])));
      Raw<T> y;
      y.set(f);
      if (at.live && h0 + i * kPar < H) y.store(yr + i * kPar * p.D);
    }
  }
}

template <typename T, int kGroup, int kHeads>
__global__ void __launch_bounds__(kThreads, kBwdBlocks<T>) bwd_kernel(const Params p) {
  constexpr int kPar = 32 / kGroup;
  constexpr int kChunk = kPar * kHeads;
  __shared__ float red[kThreads / 32][kGroup * kE];
  __shared__ int kind[kThreads / 32];            // 0 = queries, 1 = keys, 2 = nothing to sum
  const Place at = Place::make<kGroup>(p);
  const int cq = (p.Hq + kChunk - 1) / kChunk, ck = (p.Hkv + kChunk - 1) / kChunk, per = cq + 2 * ck;
  const int warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int step = gridDim.x * (kThreads / 32) / per;
  const int chunk = warp % per;
  const bool is_q = chunk < cq, is_v = chunk >= cq + ck;
  const int H = is_q ? p.Hq : p.Hkv;
  const int h0 = (is_q ? chunk : is_v ? chunk - cq - ck : chunk - cq) * kChunk + at.sub;
  const int64_t t_end = warp / per < step ? p.T : 0;
  const int64_t dxs = (int64_t)(p.Hq + 2 * p.Hkv) * p.D;
  T* ob = reinterpret_cast<T*>(p.dx) + (int64_t)(is_q ? 0 : is_v ? p.Hq + p.Hkv : p.Hq) * p.D + (int64_t)h0 * p.D + at.e0;
  F2 dw[kP];
#pragma unroll
  for (int j = 0; j < kP; ++j) dw[j] = 0ull;
  if (is_v) {                                    // values pass through
    for (int64_t t = warp / per; t < t_end; t += step) {
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (!at.live || h0 + i * kPar >= H) continue;
        Raw<T> v;
        v.zero();
        if (p.dv != nullptr) v.load(reinterpret_cast<const T*>(p.dv) + t * p.dvs + (int64_t)(h0 + i * kPar) * p.D + at.e0);
        v.store(ob + t * dxs + i * kPar * p.D);
      }
    }
  } else {
    const T* xb = reinterpret_cast<const T*>(p.x) + (is_q ? 0 : (int64_t)p.Hq * p.D) + (int64_t)h0 * p.D + at.e0;
    const T* db = reinterpret_cast<const T*>(is_q ? p.dq : p.dk) + (int64_t)h0 * p.D + at.e0;
    const int64_t ds = is_q ? p.dqs : p.dks;
    const float scale = is_q ? p.q_scale : 1.f, inv_d = 1.f / (float)p.D;
    F2 g[kP];
    load_gain<T>(is_q ? p.qw : p.kw, p.gain, scale, at.e0, at.live, g);
    extern __shared__ __align__(16) uint8_t ring[];
    uint8_t* mine = ring + (threadIdx.x >> 5) * (kStages * 2 * kHeads * kVector<T>) + (threadIdx.x & 31) * 16;
    const uint32_t mine_s = (uint32_t)__cvta_generic_to_shared(mine);
    auto fetch = [&](int64_t t, int stage) {
      if (t < t_end) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const bool on = at.live && h0 + i * kPar < H;
          copy_async<T>(mine_s + (stage * 2 * kHeads + 2 * i) * kVector<T>, on ? xb + t * p.xs + i * kPar * p.D : xb, on);
          copy_async<T>(mine_s + (stage * 2 * kHeads + 2 * i + 1) * kVector<T>, on ? db + t * ds + i * kPar * p.D : db, on);
        }
      }
      copies_commit();
    };
    const int64_t first = warp / per;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(first + (int64_t)i * step, i);
    int64_t row = t_end > 0 ? table_row(p, first) : 0;
    int stage = 0;
    for (int64_t t = first; t < t_end; t += step) {
      fetch(t + (int64_t)(kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
      F2 c[kP], s[kP];
      load_turn(p, at, t, row, -1.f, c, s);
      row = table_row(p, t + step);
      copies_wait<kStages - 1>();
      const uint8_t* here = mine + stage * 2 * kHeads * kVector<T>;
      stage = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        const Raw<T> d = copied<T>(here + (2 * i + 1) * kVector<T>);
        F2 f[kP], dn[kP], o[kP], gd[kP];
        d.get(dn);
        partner_of<T>(p, at, d, o);
        copied<T>(here + 2 * i * kVector<T>).get(f);
        F2 ss = 0ull, dot = 0ull;
#pragma unroll
        for (int j = 0; j < kP; ++j) {
          dn[j] = fma2(c[j], dn[j], mul2(s[j], o[j]));
          gd[j] = mul2(g[j], dn[j]);
          ss = fma2(f[j], f[j], ss);
          dot = fma2(gd[j], f[j], dot);
        }
        const float r = rsqrtf(group_sum<kGroup>(sum2(ss)) * inv_d + p.eps);
        const float m = -group_sum<kGroup>(sum2(dot)) * inv_d * r * r * r;      // dx = r g + m x
        // a head that does not exist adds nothing: its zeros would meet an infinite r without eps
        const float rs = h0 + i * kPar < H ? r * scale : 0.f;
#pragma unroll
        for (int j = 0; j < kP; ++j) {
          dw[j] = fma2(f2(rs, rs), mul2(dn[j], f[j]), dw[j]);
          f[j] = fma2(f2(m, m), f[j], mul2(f2(r, r), gd[j]));
        }
        Raw<T> y;
        y.set(f);
        if (at.live && h0 + i * kPar < H) y.store(ob + t * dxs + i * kPar * p.D);
      }
    }
  }
  if (p.dw_partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < kP; ++j) {
    float w[2];
    split(dw[j], w[0], w[1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = 16; o >= kGroup; o >>= 1) w[e] += __shfl_xor_sync(0xffffffffu, w[e], o);
      if (at.sub == 0) red[threadIdx.x >> 5][at.e0 + 2 * j + e] = w[e];
    }
  }
  if ((threadIdx.x & 31) == 0) kind[threadIdx.x >> 5] = is_v ? 2 : is_q ? 0 : 1;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.D; i += kThreads) {
    const int which = i / p.D, e = i % p.D;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w)
      if (kind[w] == which) s += red[w][e];
    p.dw_partial[((int64_t)blockIdx.x * 2 + which) * p.D + e] = s;
  }
}

// Column sums of the per-block partial weight gradients [parts, cols] in a fixed order: the result does not depend on
// the schedule.  One block of 32 x 32 threads per 32 columns; rounded once to the output's type.
template <typename O>
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* __restrict__ partial, O* __restrict__ out, int parts, int cols) {
  __shared__ float tile[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int i = ty; i < parts; i += 32) s += partial[(int64_t)i * cols + col];
  }
  tile[ty][tx] = s;
  __syncthreads();
  const float a = warp_sum(tile[tx][ty]);        // warp ty sums column ty of the tile
  if (tx == 0 && blockIdx.x * 32 + ty < cols) out[blockIdx.x * 32 + ty] = from_float<O>(a);
}

}  // namespace qkn

// Lanes per head: the power of two that holds D / 8 vectors.
#define TB_QKN_GROUP(D, ...)                                 \
  if ((D) <= 32) { constexpr int kGroup = 4; __VA_ARGS__(); }        \
  else if ((D) <= 64) { constexpr int kGroup = 8; __VA_ARGS__(); }   \
  else if ((D) <= 128) { constexpr int kGroup = 16; __VA_ARGS__(); } \
  else { constexpr int kGroup = 32; __VA_ARGS__(); }

// The tensor itself when its heads are adjacent and its rows start on 16 bytes, else a copy that is so.
static at::Tensor qkn_rows(const at::Tensor& t) {
  if (t.dim() == 3 && t.stride(2) == 1 && t.stride(1) == t.size(2) && t.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

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

// Blocks of a launch: as many as are resident (kPerSm) or as the work needs, and never fewer warps than one token's chunks.
static int qkn_grid(int64_t T, int64_t per, int per_sm) {
  TORCH_CHECK(T <= (1 << 30) && per <= (1 << 20), "qk_norm_rope: too many tokens or heads");
  constexpr int kWarps = qkn::kThreads / 32;
  const int64_t want = (T * per + kWarps - 1) / kWarps, full = std::max<int64_t>((int64_t)num_sms() * per_sm, (per + kWarps - 1) / kWarps);
  return (int)std::min<int64_t>(want, full);
}

// Wide warps (several heads a lane) once every resident warp still has a token to itself; a decode step of a few tokens
// spreads over the SMs instead.  Forward of 32 + 8 heads of 128, wide / narrow: 256 tokens 12.2 / 8.8 us, 512 tokens
// 8.8 / 10.6 us, 1024 tokens 10.8 / 13.6 us.
static bool qkn_wide(const qkn::Params& p, int group) {
  const int64_t chunk = 4 * (32 / group);        // of the widest warps
  return p.T * ((p.Hq + chunk - 1) / chunk + (p.Hkv + chunk - 1) / chunk) >= (int64_t)num_sms() * 16;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& x_in, int64_t hq, int64_t hkv, const c10::optional<at::Tensor>& qw,
                                                    const c10::optional<at::Tensor>& kw, const c10::optional<at::Tensor>& table,
                                                    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& axes,
                                                    bool interleaved, double eps, double gain, double q_scale) {
  TORCH_CHECK(x_in.is_cuda(), "qk_norm_rope: x must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x_in.device());
  const at::Tensor x = qkn_rows(x_in);
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
      const int grid = qkn_grid(p.T, (p.Hq + chunk - 1) / chunk + (p.Hkv + chunk - 1) / chunk, x.element_size() == 2 ? qkn::kFwdBlocks<__nv_bfloat16> : qkn::kFwdBlocks<float>);
      const int smem = qkn::kThreads / 32 * qkn::kStages * kHeads * 32 * qkn::kE * (int)x.element_size();      // at most 48 KB
      if (x.scalar_type() == at::kBFloat16) qkn::fwd_kernel<__nv_bfloat16, kGroup, kHeads><<<grid, qkn::kThreads, smem, stream>>>(p);
      else qkn::fwd_kernel<float, kGroup, kHeads><<<grid, qkn::kThreads, smem, stream>>>(p);
    };
    if (qkn_wide(p, kGroup)) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 1>{});
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, k};
}

// Returns dx of x's shape (contiguous) and the weight gradients [2, D] (empty without weights), fp32 or x's type.
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_bwd(const at::Tensor& dq, const at::Tensor& dk, const c10::optional<at::Tensor>& dv,
                                                    const at::Tensor& x_in, int64_t hq, int64_t hkv, const c10::optional<at::Tensor>& qw,
                                                    const c10::optional<at::Tensor>& kw, const c10::optional<at::Tensor>& table,
                                                    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& axes,
                                                    bool interleaved, double eps, double gain, double q_scale, bool fp32_dw) {
  TORCH_CHECK(x_in.is_cuda(), "qk_norm_rope: x must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(x_in.device());
  const at::Tensor x = qkn_rows(x_in);
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
  auto dw = at::empty({has_w ? 2 : 0, p.D}, fp32_dw ? x.options().dtype(at::kFloat) : x.options());
  if (p.T == 0) return {dx, dw.zero_()};
  const at::Tensor dq_ = qkn_rows(dq), dk_ = qkn_rows(dk), dv_ = dv.has_value() ? qkn_rows(*dv) : at::Tensor();
  p.dq = grad(dq_, hq, p.dqs);
  p.dk = grad(dk_, hkv, p.dks);
  if (dv_.defined()) p.dv = grad(dv_, hkv, p.dvs);
  p.dx = dx.data_ptr();
  auto stream = at::cuda::getCurrentCUDAStream();
  at::Tensor partial;
  int grid = 0;
  TB_QKN_GROUP(p.D, [&] {
    auto launch = [&](auto heads) {
      constexpr int kHeads = decltype(heads)::value;
      const int64_t chunk = kHeads * (32 / kGroup);
      grid = qkn_grid(p.T, (p.Hq + chunk - 1) / chunk + 2 * ((p.Hkv + chunk - 1) / chunk), x.element_size() == 2 ? qkn::kBwdBlocks<__nv_bfloat16> : qkn::kBwdBlocks<float>);
      if (has_w) {
        partial = at::empty({grid, 2, p.D}, x.options().dtype(at::kFloat));
        p.dw_partial = partial.data_ptr<float>();
      }
      const int smem = qkn::kThreads / 32 * qkn::kStages * 2 * kHeads * 32 * qkn::kE * (int)x.element_size();
      if (x.scalar_type() == at::kBFloat16) qkn::bwd_kernel<__nv_bfloat16, kGroup, kHeads><<<grid, qkn::kThreads, smem, stream>>>(p);
      else if constexpr (kHeads <= 2) qkn::bwd_kernel<float, kGroup, kHeads><<<grid, qkn::kThreads, smem, stream>>>(p);
    };
    // four heads a lane read a token's cos / sin half as often as two: 65 -> 61 us (8192 tokens, 32 + 4 heads of 128), 54 -> 43 us
    // (4097 tokens, 16 + 4 heads of 256, three axes); fp32 vectors are twice as long and keep to two
    if (!qkn_wide(p, kGroup)) launch(std::integral_constant<int, 1>{});
    else if (x.scalar_type() == at::kBFloat16) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 2>{});
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (has_w) {
    const int blocks = (2 * p.D + 31) / 32;
    if (dw.scalar_type() == at::kFloat) qkn::sum_partials_kernel<<<blocks, 1024, 0, stream>>>(partial.data_ptr<float>(), dw.data_ptr<float>(), grid, 2 * p.D);
    else qkn::sum_partials_kernel<<<blocks, 1024, 0, stream>>>(partial.data_ptr<float>(), reinterpret_cast<__nv_bfloat16*>(dw.data_ptr()), grid, 2 * p.D);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {dx, dw};
}

}  // namespace tb200
