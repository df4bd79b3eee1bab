// Layer norm over the last dimension with an optional affine (weight, bias)
// and an optional modulation (scale, shift, one row per sample), forward and
// backward.
//
//   z = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   y = (z * w + b) * (1 + s) + t
// With g = w (1 + s), i = dy * g and A = sum(i) / D, B = sum(i z) / D per row:
//   dx = rstd * (i - A - z B)
// and with the per-sample column sums S1 = sum dy, S2 = sum dy z:
//   dt = S1,  ds = w S2 + b S1,  dw = sum_samples (1 + s) S2,
//   db = sum_samples (1 + s) S1
// so one pass over x and dy feeds every gradient. Statistics and sums are f32
// throughout (mean first, then the centred squares, both from registers);
// each output is rounded once. The row sum is divided by D: the product with a
// rounded 1 / D can miss the mean of a row of one value by an ulp, which a
// small eps turns into a z far from zero.
//
// HBM bounds both directions: x in and y out forward, x and dy in and dx out
// backward. Column sums go through per-CTA partials and a second kernel in a
// fixed order, without atomics, so gradients are the same on every run.
#include <cuda_runtime.h>
#include <algorithm>
#include <initializer_list>
#include "gwb.h"
#include "ptx.cuh"
#include "elem.cuh"

namespace gwb {
namespace norm {

struct Param {              // a weight / bias / scale / shift vector
  const void* p;            // null when absent
  int f32;                  // 1: f32, 0: x's type
  int64_t stride;           // elements between samples (0: shared)
};

// VEC values of a parameter at column c of sample b
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const Param& a, int64_t b, int c, float (&o)[VEC]) {
  if (a.f32) {
    const float* p = static_cast<const float*>(a.p) + b * a.stride + c;
    if constexpr (VEC == 1) {
      o[0] = __ldg(p);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p + j));
        o[j] = f.x; o[j + 1] = f.y; o[j + 2] = f.z; o[j + 3] = f.w;
      }
    }
  } else {
    Pack<T, VEC> v;
    v.load(static_cast<const T*>(a.p) + b * a.stride + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = v.get(j);
  }
}

struct FwdArgs {
  const void* x; int64_t xs;     // row stride in elements
  Param w, b, s, t;
  void* y; float* mean; float* rstd;
  int64_t M; int D; int64_t rows_per_mod; float eps;
};

struct BwdArgs {
  const void* dy; int64_t dys;
  const void* x; int64_t xs;
  const float* mean; const float* rstd;
  Param w, b, s;
  void* dx;                      // may be null
  float* partial;                // [samples * chunks][2][D] or null
  int64_t rows_per_mod; int D; int chunks; int64_t chunk_rows;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the whole CTA, the same bits in every thread (fixed order).
// `slot` alternates between calls so that one barrier per sum is enough.
__device__ __forceinline__ float block_sum(float v, float* slot) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  return warp_sum(lane < nw ? slot[lane] : 0.0f);
}

// ------------------------------------------------ rows through shared memory
// Bulk copies bring rows as the 16-byte granules that cover them, so a row may
// start anywhere: `lead` bytes into its first granule. Nothing before the
// granule of a row's first element or past the granule of its last is read,
// and of the matrix's last granule only its elements.
struct Span { const uint8_t* from; uint32_t lead, bytes; };

template <typename T>
__device__ __forceinline__ Span span_of(const T* first, int64_t n) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(first);
  Span s;
  s.lead = (uint32_t)(a & 15u);
  s.from = reinterpret_cast<const uint8_t*>(a - s.lead);
  s.bytes = (s.lead + (uint32_t)(n * sizeof(T)) + 15u) & ~15u;
  return s;
}

// One thread: the copy of n elements at `first` to dst, to complete on `bar`
// (whose expected bytes the caller has not announced yet); returns them.
// `last` (the last row, or rows that lie on top of each other): nothing may be
// read behind the elements, so a part granule at the end is stored by hand, ordered before the copy's completion by this
// thread's own arrival.
template <typename T>
__device__ __forceinline__ uint32_t span_bytes(const T* first, int64_t n, bool last, uint8_t* dst) {
  const Span s = span_of(first, n);
  const uint32_t end = s.lead + (uint32_t)(n * sizeof(T));
  if (!last || end == s.bytes) return s.bytes;
  const uint32_t whole = end & ~15u;
  for (uint32_t b = whole > s.lead ? whole : s.lead; b < end; b += sizeof(T))
    *reinterpret_cast<T*>(dst + b) = *reinterpret_cast<const T*>(s.from + b);
  return whole;
}

// After a wait that ran out: the copies in flight land (again with a limit)
// before the shared memory goes to another CTA.
__device__ __forceinline__ void drain(uint64_t* full, int stages, int from, int to) {
  for (int k = from; k < to; ++k)
    (void)mbar_wait(&full[k % stages], (k / stages) & 1, GWB_ERR_TIMEOUT_ACT);
}

// g = w (1 + s) and h = b (1 + s) + t of one sample's columns, f32, so that
// y = z g + h
template <typename T>
__device__ __forceinline__ void combine(const Param& w, const Param& b, const Param& s,
                                        const Param& t, int64_t smp, int c, float& g, float& h) {
  float p[1], up = 1.0f;
  if (s.p) { load_param<T, 1>(s, smp, c, p); up += p[0]; }
  g = up;
  h = 0.0f;
  if (w.p) { load_param<T, 1>(w, 0, c, p); g *= p[0]; }
  if (b.p) { load_param<T, 1>(b, 0, c, p); h = p[0] * up; }
  if (t.p) { load_param<T, 1>(t, smp, c, p); h += p[0]; }
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// f(i, column, column exists) for a lane's elements l, l + L, ...: eight at a
// time without a test where all lanes have them (a test an element costs a
// predicate that outlives the row's registers).
template <int E, int LO, int L, typename F>
__device__ __forceinline__ void each(int D, int l, const F& f) {
#pragma unroll
  for (int h = 0; h < E; h += 8) {
    if (h + 8 <= LO || (h + 8) * L <= D) {
#pragma unroll
      for (int i = h; i < h + 8; ++i) f(i, l + i * L, true);
    } else if (h * L < D) {
#pragma unroll
      for (int i = h; i < h + 8; ++i) f(i, l + i * L, l + i * L < D);
    }
  }
}

struct FwdPlan {
  int chunks;                    // CTAs a sample
  int64_t chunk_rows;            // rows of one, a multiple of slot_rows
  int slot_rows, stages;         // rows a copy brings, slots a warp
  int warps;                     // warps that take rows; any others help with g and h
  uint32_t slot_bytes;
};

// A warp takes whole rows (32 / L at a time, L lanes each), E elements a
// lane, from its own ring of bulk copies: no barrier but the one that shares
// g and h, and few instructions a row besides the arithmetic (18432 x 3072
// bf16 with scale and shift: 46 us, 4.9 TB/s; without parameters 33, 6.8 TB/s:
// the rest is g and h coming out of shared memory for every row). VECTOR: rows and parameters lie on 16 bytes, a lane has vectors
// lane, lane + L, ...; else elements lane, lane + L, ..., so that any
// alignment reads shared memory without conflicts.
template <typename T, int E, int LO, int L, bool VECTOR>
__global__ void __launch_bounds__(E <= 32 ? 384 : E <= 64 ? 512 : E <= 96 ? 384 : 256, E <= 32 ? 2 : 1)
forward_kernel(const FwdArgs a, const FwdPlan p) {
  constexpr int VEC = 16 / (int)sizeof(T), P = Pairs<T>::N, C = E / VEC, G = 32 / L;
  constexpr int SURE = LO / VEC;                         // vectors that every lane has
  extern __shared__ __align__(16) uint8_t smem[];
  const int warps = p.warps, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l = lane % L, sub = lane / L;
  const int pd = (a.D + 3) & ~3;
  float* gs = reinterpret_cast<float*>(smem);            // [pd] g, [pd] h
  float* hs = gs + pd;
  uint64_t* full = reinterpret_cast<uint64_t*>(hs + pd) + warp * p.stages;
  uint8_t* ring = smem + ((2 * pd * 4 + warps * p.stages * 8 + 15) & ~15) +
                  (size_t)warp * p.stages * p.slot_bytes;
  const int64_t smp = blockIdx.x / p.chunks;
  const int64_t c0 = (int64_t)(blockIdx.x % p.chunks) * p.chunk_rows;
  const int64_t c1 = c0 + p.chunk_rows < a.rows_per_mod ? c0 + p.chunk_rows : a.rows_per_mod;
  const int64_t base = smp * a.rows_per_mod;
  const T* x = static_cast<const T*>(a.x);
  // slot s of this warp: rows first .. first + slot_rows of the chunk
  const auto first_of = [&](int s) { return c0 + ((int64_t)s * warps + warp) * p.slot_rows; };
  const int64_t groups = c1 > c0 ? (c1 - c0 + p.slot_rows - 1) / p.slot_rows : 0;
  const int steps = (int)((groups - warp + warps - 1) / warps);
  const auto fill = [&](int s) {                         // lane 0
    const int64_t r = base + first_of(s);
    const int64_t left = base + c1 - r, rows = left < p.slot_rows ? left : p.slot_rows;
    const int64_t n = (rows - 1) * a.D + a.D;            // one row, or rows that adjoin
    uint8_t* dst = ring + (size_t)(s % p.stages) * p.slot_bytes;
    const T* src = x + r * a.xs;
    const uint32_t bytes = span_bytes(src, n, r + rows == a.M || a.xs < a.D, dst);
    mbar_arrive_expect_tx(&full[s % p.stages], bytes);
    if (bytes) bulk_load(dst, span_of(src, n).from, bytes, &full[s % p.stages]);
  };
  if (lane == 0 && warp < warps) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
    for (int s = 0; s < p.stages && s < steps; ++s) fill(s);
  }
  const bool params = a.w.p || a.b.p || a.s.p || a.t.p;
  if (params)
    for (int c0 = threadIdx.x; c0 < a.D; c0 += 4 * blockDim.x) {
      // four columns' loads in flight together
      float g[4], h[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = c0 + k * (int)blockDim.x;
        if (c < a.D) combine<T>(a.w, a.b, a.s, a.t, smp, c, g[k], h[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // VECTOR: four columns of a vector a plane, so that the lanes' 16-byte
        // reads adjoin (a vector's eight in a row would share banks two by two)
        const int c = c0 + k * (int)blockDim.x;
        const int at = VECTOR ? c % VEC / 4 * (a.D / (VEC / 4)) + c / VEC * 4 + c % 4 : c;
        if (c < a.D) { gs[at] = g[k]; hs[at] = h[k]; }
      }
    }
  __syncthreads();
  if (warp >= warps) return;
  const float inv_d = 1.0f / (float)a.D;
  const int nvec = a.D / VEC;
  T* y = static_cast<T*>(a.y);
  int slot = 0, phase = 0;
  for (int s = 0; s < steps; ++s) {
    if (!mbar_wait_warp(&full[slot], phase, GWB_ERR_TIMEOUT_ACT)) {
      if (lane == 0) drain(full, p.stages, s, min(steps, s + p.stages));
      return;
    }
    const int64_t r0 = base + first_of(s);
    const int rows = (int)min((int64_t)p.slot_rows, base + c1 - r0);
    const uint8_t* src = ring + (size_t)slot * p.slot_bytes;
    if (!VECTOR) src += reinterpret_cast<uintptr_t>(x + r0 * a.xs) & 15u;
    for (int k0 = 0; k0 < rows; k0 += G) {
      const int k = k0 + sub;
      const bool live = k < rows;
      F2 v[VECTOR ? E / 2 : 1];
      float e[VECTOR ? 1 : E];
      F2 acc = f2(0.0f, 0.0f);
      const T* row = reinterpret_cast<const T*>(src) + (size_t)(live ? k : 0) * a.D;
      if constexpr (VECTOR) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          F2 u[P];
          if (c < SURE || l + c * L < nvec) {
            unpack<T>(*reinterpret_cast<const uint4*>(row + (l + c * L) * VEC), u);
          } else {
#pragma unroll
            for (int j = 0; j < P; ++j) u[j] = f2(0.0f, 0.0f);
          }
#pragma unroll
          for (int j = 0; j < P; ++j) { v[c * P + j] = u[j]; acc = add2(acc, u[j]); }
        }
      } else {
        float part = 0.0f;
        each<E, LO, L>(a.D, l, [&](int i, int c, bool in) {
          e[i] = in ? to_f32<T>(row[c]) : 0.0f;
          part += e[i];
        });
        acc = f2(part, 0.0f);
      }
      if (k0 + G >= rows) {
        // the slot is in registers: bring the rows after next
        __syncwarp();
        if (lane == 0 && s + p.stages < steps) fill(s + p.stages);
      }
      const float mean = lanes_sum<L>(sum2(acc)) / (float)a.D;
      const F2 neg = f2(-mean, -mean);
      acc = f2(0.0f, 0.0f);
      if constexpr (VECTOR) {
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (c < SURE || l + c * L < nvec)
#pragma unroll
            for (int j = c * P; j < c * P + P; ++j) {
              v[j] = add2(v[j], neg);
              acc = fma2(v[j], v[j], acc);
            }
      } else {
        float part = 0.0f;
        each<E, LO, L>(a.D, l, [&](int i, int, bool in) {
          e[i] -= mean;
          if (in) part += e[i] * e[i];
        });
        acc = f2(part, 0.0f);
      }
      // rsqrtf: 2 ulp, far inside the statistics' own rounding
      const float rstd = rsqrtf(lanes_sum<L>(sum2(acc)) * inv_d + a.eps);
      if (!live) continue;
      const int64_t r = r0 + k;
      if (l == 0 && a.mean != nullptr) {
        a.mean[r] = mean;
        a.rstd[r] = rstd;
      }
      const F2 r2 = f2(rstd, rstd);
      T* out = y + r * a.D;
      if constexpr (VECTOR) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int i = l + c * L;
          if (c >= SURE && i >= nvec) continue;
          F2 u[P];
#pragma unroll
          for (int j = 0; j < P; ++j) u[j] = mul2(v[c * P + j], r2);
          if (params) {
#pragma unroll
            for (int j = 0; j < P; j += 2) {
              const int at = (j / 2) * (a.D / (VEC / 4)) + i * 4;
              const float4 g4 = *reinterpret_cast<const float4*>(gs + at);
              const float4 h4 = *reinterpret_cast<const float4*>(hs + at);
              u[j] = fma2(u[j], f2(g4.x, g4.y), f2(h4.x, h4.y));
              u[j + 1] = fma2(u[j + 1], f2(g4.z, g4.w), f2(h4.z, h4.w));
            }
          }
          *reinterpret_cast<uint4*>(out + i * VEC) = repack<T>(u);
        }
      } else {
        each<E, LO, L>(a.D, l, [&](int i, int c, bool in) {
          if (!in) return;
          const float z = e[i] * rstd;
          out[c] = from_f32<T>(params ? z * gs[c] + hs[c] : z);
        });
      }
    }
    if (++slot == p.stages) { slot = 0; phase ^= 1; }
  }
}

// Rows of over 4096 elements, one a CTA of 512 threads; the row stays in
// registers, C vectors a thread, between the statistics and the output.
template <typename T, int VEC, int C>
__global__ void __launch_bounds__(512) forward_block_kernel(const FwdArgs a) {
  __shared__ float red[2][32];
  const int lanes = blockDim.x, t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int nvec = a.D / VEC;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  Pack<T, VEC> raw[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (t + c * lanes < nvec) raw[c].load(x + (t + c * lanes) * VEC);
  float v[C][VEC], sum = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[c][j] = t + c * lanes < nvec ? raw[c].get(j) : 0.0f;
      sum += v[c][j];
    }
  const float inv_d = 1.0f / (float)a.D;
  const float mean = block_sum(sum, red[0]) / (float)a.D;
  float sq = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (t + c * lanes < nvec)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[c][j] -= mean;
        sq += v[c][j] * v[c][j];
      }
  const float var = block_sum(sq, red[1]) * inv_d;
  const float rstd = rsqrtf(var + a.eps);
  if (t == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const int64_t smp = a.s.p || a.t.p ? row / a.rows_per_mod : 0;
  T* y = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = t + c * lanes;
    if (i >= nvec) continue;
    float p[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[c][j] *= rstd;
    if (a.w.p) {
      load_param<T, VEC>(a.w, 0, i * VEC, p);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[c][j] *= p[j];
    }
    if (a.b.p) {
      load_param<T, VEC>(a.b, 0, i * VEC, p);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[c][j] += p[j];
    }
    if (a.s.p) {
      load_param<T, VEC>(a.s, smp, i * VEC, p);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[c][j] *= 1.0f + p[j];
    }
    if (a.t.p) {
      load_param<T, VEC>(a.t, smp, i * VEC, p);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[c][j] += p[j];
    }
    Pack<T, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.set(j, v[c][j]);
    o.store(y + i * VEC);
  }
}

// The same for rows and parameters on 16 bytes, in packed f32: C vectors a
// thread, its parameters read as vectors where they are used. Two barriers a
// row, but thousands of CTAs to hide them behind: it beats the warp a row, with
// its g and h to prepare and rows to take in turn, up to a few rows a warp (1024
// and 4608 rows of 3072 bf16: 9.8 and 16.5 us a call against 13.4 and 18.5).
template <typename T>
__device__ __forceinline__ void load_pairs(const Param& a, int64_t b, int c,
                                           F2 (&o)[Pairs<T>::N]) {
  if (a.f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.p) + b * a.stride + c);
#pragma unroll
    for (int j = 0; j < Pairs<T>::N; j += 2) {
      const float4 f = __ldg(p + j / 2);
      o[j] = f2(f.x, f.y);
      o[j + 1] = f2(f.z, f.w);
    }
  } else {
    unpack<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.p) + b * a.stride + c)), o);
  }
}

template <typename T, int C>
__global__ void __launch_bounds__(512) forward_pairs_kernel(const FwdArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T), P = Pairs<T>::N;
  __shared__ float red[2][16];
  const int lanes = blockDim.x, t = threadIdx.x, nw = lanes >> 5, nvec = a.D / VEC;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const float inv_d = 1.0f / (float)a.D;
  const auto total = [&](F2 v, int k) {
    const float w = warp_sum(sum2(v));
    if (nw == 1) return w;
    if ((t & 31) == 0) red[k][t >> 5] = w;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < nw; ++i) s += red[k][i];
    return s;
  };
  uint4 raw[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
    raw[c] = t + c * lanes < nvec ? *reinterpret_cast<const uint4*>(x + (t + c * lanes) * VEC)
                                  : make_uint4(0, 0, 0, 0);
  F2 v[C][P], acc = f2(0.0f, 0.0f);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    unpack<T>(raw[c], v[c]);
#pragma unroll
    for (int j = 0; j < P; ++j) acc = add2(acc, v[c][j]);
  }
  const float mean = total(acc, 0) / (float)a.D;
  const F2 neg = f2(-mean, -mean);
  acc = f2(0.0f, 0.0f);
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (t + c * lanes < nvec)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        v[c][j] = add2(v[c][j], neg);
        acc = fma2(v[c][j], v[c][j], acc);
      }
  const float rstd = rsqrtf(total(acc, 1) * inv_d + a.eps);
  if (t == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const int64_t smp = a.s.p || a.t.p ? row / a.rows_per_mod : 0;
  const F2 r2 = f2(rstd, rstd), one = f2(1.0f, 1.0f);
  T* y = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = t + c * lanes;
    if (i >= nvec) continue;
    F2 p[P];
#pragma unroll
    for (int j = 0; j < P; ++j) v[c][j] = mul2(v[c][j], r2);
    if (a.w.p) {
      load_pairs<T>(a.w, 0, i * VEC, p);
#pragma unroll
      for (int j = 0; j < P; ++j) v[c][j] = mul2(v[c][j], p[j]);
    }
    if (a.b.p) {
      load_pairs<T>(a.b, 0, i * VEC, p);
#pragma unroll
      for (int j = 0; j < P; ++j) v[c][j] = add2(v[c][j], p[j]);
    }
    if (a.s.p) {
      load_pairs<T>(a.s, smp, i * VEC, p);
#pragma unroll
      for (int j = 0; j < P; ++j) v[c][j] = mul2(v[c][j], add2(one, p[j]));
    }
    if (a.t.p) {
      load_pairs<T>(a.t, smp, i * VEC, p);
#pragma unroll
      for (int j = 0; j < P; ++j) v[c][j] = add2(v[c][j], p[j]);
    }
    *reinterpret_cast<uint4*>(y + i * VEC) = repack<T>(v[c]);
  }
}

// Rows too wide for the registers of one CTA: three passes, the second and
// third from L2.
template <typename T>
__global__ void __launch_bounds__(1024) forward_wide_kernel(const FwdArgs a) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  float sum = 0.0f;
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) sum += to_f32<T>(x[c]);
  const float inv_d = 1.0f / (float)a.D;
  const float mean = block_sum(sum, red[0]) / (float)a.D;
  float sq = 0.0f;
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
    const float d = to_f32<T>(x[c]) - mean;
    sq += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum(sq, red[1]) * inv_d + a.eps);
  if (threadIdx.x == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const int64_t smp = a.s.p || a.t.p ? row / a.rows_per_mod : 0;
  T* y = static_cast<T*>(a.y) + row * a.D;
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
    float v = (to_f32<T>(x[c]) - mean) * rstd, p[1];
    if (a.w.p) { load_param<T, 1>(a.w, 0, c, p); v *= p[0]; }
    if (a.b.p) { load_param<T, 1>(a.b, 0, c, p); v += p[0]; }
    if (a.s.p) { load_param<T, 1>(a.s, smp, c, p); v *= 1.0f + p[0]; }
    if (a.t.p) { load_param<T, 1>(a.t, smp, c, p); v += p[0]; }
    y[c] = from_f32<T>(v);
  }
}

// g = w (1 + s) of one sample's columns
template <typename T, int VEC>
__device__ __forceinline__ void gain(const Param& w, const Param& s, int64_t smp, int c,
                                     float (&g)[VEC]) {
  float p[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) g[j] = 1.0f;
  if (w.p) {
    load_param<T, VEC>(w, 0, c, p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] = p[j];
  }
  if (s.p) {
    load_param<T, VEC>(s, smp, c, p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[j] *= 1.0f + p[j];
  }
}

// Narrow rows (up to 64 vectors): CTA blockIdx.x takes one chunk of one
// sample's rows, its eight warps rows in turn, one a warp; a thread keeps its
// C vectors of columns, joined over the warps at the end.
template <typename T, int VEC, int C>
__global__ void __launch_bounds__(256, C == 1 ? 4 : 2) backward_kernel(const BwdArgs a) {
  extern __shared__ float part_sm[];             // [8][2][D]
  const int warp = threadIdx.x >> 5, t = threadIdx.x & 31;
  const int nvec = a.D / VEC;
  const int64_t smp = blockIdx.x / a.chunks;
  const int64_t r0 = (int64_t)(blockIdx.x % a.chunks) * a.chunk_rows;
  const int64_t r1 = r0 + a.chunk_rows < a.rows_per_mod ? r0 + a.chunk_rows : a.rows_per_mod;
  const int64_t base = smp * a.rows_per_mod;
  const float inv_d = 1.0f / (float)a.D;
  float g[C][VEC], s1[C][VEC], s2[C][VEC];
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) g[c][j] = s1[c][j] = s2[c][j] = 0.0f;
    if (t + c * 32 < nvec) gain<T, VEC>(a.w, a.s, smp, (t + c * 32) * VEC, g[c]);
  }
  Pack<T, VEC> xn[C], dn[C];                     // the next row's
  float meann = 0.0f, rstdn = 0.0f;
  const auto fetch = [&](int64_t r) {
    const int64_t row = base + r;
    meann = __ldg(a.mean + row);
    rstdn = __ldg(a.rstd + row);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (t + c * 32 < nvec) {
        xn[c].load(static_cast<const T*>(a.x) + row * a.xs + (t + c * 32) * VEC);
        dn[c].load(static_cast<const T*>(a.dy) + row * a.dys + (t + c * 32) * VEC);
      }
  };
  if (r0 + warp < r1) fetch(r0 + warp);
  for (int64_t r = r0 + warp; r < r1; r += 8) {
    Pack<T, VEC> xv[C], dv[C];
    const float mean = meann, rstd = rstdn;
#pragma unroll
    for (int c = 0; c < C; ++c) { xv[c] = xn[c]; dv[c] = dn[c]; }
    if (r + 8 < r1) fetch(r + 8);
    float sa = 0.0f, sb = 0.0f;
    if constexpr (VEC > 1) {
      constexpr int P = VEC / 2;
      const F2 neg = f2(-mean, -mean), r2 = f2(rstd, rstd);
      F2 ta = f2(0.0f, 0.0f), tb = ta;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (t + c * 32 < nvec) {
          F2 x2[P], d2[P];
          unpack<T>(xv[c].bits(), x2);
          unpack<T>(dv[c].bits(), d2);
#pragma unroll
          for (int j = 0; j < P; ++j) {
            const F2 g2 = f2(g[c][2 * j], g[c][2 * j + 1]), q = mul2(d2[j], add2(x2[j], neg));
            const float2 u = split(add2(f2(s1[c][2 * j], s1[c][2 * j + 1]), d2[j]));
            const float2 w = split(fma2(q, r2, f2(s2[c][2 * j], s2[c][2 * j + 1])));
            s1[c][2 * j] = u.x; s1[c][2 * j + 1] = u.y;
            s2[c][2 * j] = w.x; s2[c][2 * j + 1] = w.y;
            ta = fma2(d2[j], g2, ta);
            tb = fma2(q, g2, tb);
          }
        }
      sa = sum2(ta);
      sb = sum2(tb) * rstd;
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (t + c * 32 < nvec) {
          const float z = (xv[c].get(0) - mean) * rstd, d = dv[c].get(0), e = d * z;
          s1[c][0] += d;
          s2[c][0] += e;
          sa += d * g[c][0];
          sb += e * g[c][0];
        }
    }
    if (a.dx == nullptr) continue;
    const float ma = warp_sum(sa) * inv_d, mb = warp_sum(sb) * inv_d;
    // dx = rstd (d g - A - z B) = (d g) rstd + (x c1 + c0)
    const float c1 = -rstd * rstd * mb, c0 = -mean * c1 - rstd * ma;
    T* dx = static_cast<T*>(a.dx) + (base + r) * a.D;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (t + c * 32 < nvec) {
        if constexpr (VEC > 1) {
          constexpr int P = VEC / 2;
          F2 x2[P], d2[P];
          unpack<T>(xv[c].bits(), x2);
          unpack<T>(dv[c].bits(), d2);
#pragma unroll
          for (int j = 0; j < P; ++j)
            d2[j] = fma2(mul2(d2[j], f2(g[c][2 * j], g[c][2 * j + 1])), f2(rstd, rstd),
                         fma2(x2[j], f2(c1, c1), f2(c0, c0)));
          xv[c].put(repack<T>(d2));
          xv[c].store(dx + (t + c * 32) * VEC);
        } else {
          dx[t + c * 32] = from_f32<T>(dv[c].get(0) * g[c][0] * rstd + (xv[c].get(0) * c1 + c0));
        }
      }
  }
  if (a.partial == nullptr) return;
  float* mine = part_sm + warp * 2 * a.D;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (t + c * 32 < nvec)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        mine[(t + c * 32) * VEC + j] = s1[c][j];
        mine[a.D + (t + c * 32) * VEC + j] = s2[c][j];
      }
  __syncthreads();
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.D;
  for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
    float v = 0.0f;
    for (int w = 0; w < 8; ++w) v += part_sm[w * 2 * a.D + i];
    out[i] = v;
  }
}

// Sums N values (a power of two, at most 8) over the warp's lanes in N - 1 +
// 5 - log2 N shuffles rather than 5 N: each step halves the values a lane
// carries. Returns the sum of value (lane >> (5 - log2 N)); fixed order.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int half = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, half /= 2) {
    const bool up = lane & half;
#pragma unroll
    for (int k = 0; k < n / 2; ++k) {
      const float keep = up ? v[k + n / 2] : v[k], give = up ? v[k] : v[k + n / 2];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, give, half);
    }
  }
#pragma unroll
  for (; half; half /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], half);
  return v[0];
}

struct BwdPlan { int stages; uint32_t x_slot; int64_t last; };

// One CTA per chunk of one sample's rows. Bulk copies bring two rows of x and
// dy at a time into a ring of slots, far enough ahead that reading never
// waits for the row sums' barrier. A thread keeps its E columns of the gain
// and of both column sums in registers for the whole chunk; the second pass
// over a slot (dx) reads it from shared memory again, because holding it would
// halve the warps a multiprocessor runs, and their number is what hides the
// latencies here (16 columns a thread and half the warps took 90 us against 79
// at 18432 x 3072 bf16, 4.3 TB/s; issue slots are 59 % busy). A slot is filled again after the next
// step's barrier. Every wait is bounded, and all threads leave together.
template <typename T, int E, bool VECTOR>
__global__ void __launch_bounds__(E <= 8 ? 416 : E <= 16 ? 512 : 384, E <= 8 ? 2 : 1)
backward_staged_kernel(const BwdArgs a, const BwdPlan p) {
  constexpr int R = 2, VEC = 16 / (int)sizeof(T), P = Pairs<T>::N, C = E / VEC;
  extern __shared__ __align__(16) uint8_t ring[];        // [stages][R][x, dy]
  __shared__ float red[2][16][2 * R];
  __shared__ __align__(8) uint64_t full[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = threadIdx.x;
  const int lanes = blockDim.x - 32, nw = lanes >> 5, nvec = a.D / VEC;   // the last warp copies
  const int64_t smp = blockIdx.x / a.chunks;
  const int64_t r0 = (int64_t)(blockIdx.x % a.chunks) * a.chunk_rows;
  const int count = (int)max((int64_t)0, min(a.chunk_rows, a.rows_per_mod - r0));
  const int64_t base = smp * a.rows_per_mod + r0;
  const int steps = (count + R - 1) / R;
  const uint32_t slot_bytes = 2 * R * p.x_slot;
  const float inv_d = 1.0f / (float)a.D;
  const T* x = static_cast<const T*>(a.x) + base * a.xs;
  const T* dy = static_cast<const T*>(a.dy) + base * a.dys;
  // lanes 0 .. 2 R - 1 of the copying warp: row lane / 2 of x or dy each
  const auto fill = [&](int s, int slot) {
    const int r = s * R + (lane >> 1);
    const T* src = lane & 1 ? dy + r * a.dys : x + r * a.xs;
    uint8_t* dst = ring + slot * slot_bytes + lane * p.x_slot;
    const bool last = base + r == p.last || (lane & 1 ? a.dys : a.xs) < a.D;
    const uint32_t bytes = r < count ? span_bytes(src, a.D, last, dst) : 0u;
    mbar_arrive_expect_tx(&full[slot], bytes);
    if (bytes) bulk_load(dst, span_of(src, a.D).from, bytes, &full[slot]);
  };
  if (t == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 2 * R);
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == nw) {
    // a warp of its own, or the others would wait for it while it works out
    // addresses
    int filled = min(steps, p.stages), freed = 0, s = 0;
    if (lane < 2 * R)
      for (int k = 0; k < filled; ++k) fill(k, k);
    for (; s < steps; ++s) {
      if (!__syncthreads_and(1)) break;
      // every thread is past the second pass of step s - 1
      if (s > 0 && filled < steps) {
        if (lane < 2 * R) fill(filled, freed);
        if (++freed == p.stages) freed = 0;
        ++filled;
      }
    }
    // a wait ran out: let the copies in flight land before this CTA ends
    if (s < steps && lane == 0) drain(full, p.stages, s, filled);
    return;
  }
  // columns: vectors t, t + lanes, ..., or 32 E to a warp with its lanes side
  // by side (the offsets between a lane's elements are then constants, and
  // only the last warp has any missing)
  const int col0 = warp * (32 * E) + lane;
  const bool whole = warp * (32 * E) + 32 * E <= a.D;
  const F2 zero = f2(0.0f, 0.0f);
  F2 g[E / 2], s1[E / 2], s2[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) {
    float gv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * j + e;
      const int col = VECTOR ? (t + i / VEC * lanes) * VEC + i % VEC : col0 + 32 * i;
      float h;
      gv[e] = 0.0f;
      if (col < a.D) combine<T>(a.w, {}, a.s, {}, smp, col, gv[e], h);
    }
    g[j] = f2(gv[0], gv[1]);
    s1[j] = s2[j] = zero;
  }
  // one vector's worth of columns of a row in a slot; absent ones give `none`
  const auto read = [&](const uint8_t* row, uint32_t lead, int c, float none, F2 (&v)[P]) {
    if constexpr (VECTOR) {
      unpack<T>(*reinterpret_cast<const uint4*>(row + (t + c * lanes) * 16), v);
    } else {
      const T* r = reinterpret_cast<const T*>(row + lead) + col0;
      const int at = 32 * c * VEC;
      if (whole) {
#pragma unroll
        for (int j = 0; j < P; ++j)
          v[j] = f2(to_f32<T>(r[at + 64 * j]), to_f32<T>(r[at + 64 * j + 32]));
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const int k = at + 64 * j;
          v[j] = f2(col0 + k < a.D ? to_f32<T>(r[k]) : none,
                    col0 + k + 32 < a.D ? to_f32<T>(r[k + 32]) : none);
        }
      }
    }
  };
  float mean[R], rstd[R], mean1[R], rstd1[R];            // of this step, of the next
  const auto stats = [&](int s) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int r = min(s * R + k, count - 1);
      mean1[k] = __ldg(a.mean + base + r);
      rstd1[k] = __ldg(a.rstd + base + r);
    }
  };
  if (steps) stats(0);
  for (int s = 0, slot = 0, phase = 0; s < steps; ++s) {
#pragma unroll
    for (int k = 0; k < R; ++k) { mean[k] = mean1[k]; rstd[k] = rstd1[k]; }
    if (s + 1 < steps) stats(s + 1);
    const bool ok = mbar_wait(&full[slot], phase, GWB_ERR_TIMEOUT_ACT);
    const uint8_t* src = ring + slot * slot_bytes;
    const int rows = min(R, count - s * R);
    uint32_t xl[R], dl[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      xl[k] = VECTOR ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(x + (int64_t)(s * R + k) * a.xs) & 15u);
      dl[k] = VECTOR ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(dy + (int64_t)(s * R + k) * a.dys) & 15u);
    }
    // With p = d (x - mean): S1 += d, S2 += p rstd; sum(i) = sum(d g) and
    // sum(i z) = rstd sum(p g).
    F2 dd[R][VECTOR ? E / 2 : 1];      // d, kept for the second pass where registers allow
    float sums[2 * R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      F2 sa = zero, sb = zero;
      const F2 neg = f2(-mean[k], -mean[k]), r2 = f2(rstd[k], rstd[k]);
      if (k < rows)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (VECTOR && t + c * lanes >= nvec) continue;
          F2 xv[P], dv[P];
          read(src + 2 * k * p.x_slot, xl[k], c, mean[k], xv);
          read(src + (2 * k + 1) * p.x_slot, dl[k], c, 0.0f, dv);
#pragma unroll
          for (int j = 0; j < P; ++j) {
            const int i = c * P + j;
            if (VECTOR) dd[k][i] = dv[j];
            const F2 q = mul2(dv[j], add2(xv[j], neg));
            s1[i] = add2(s1[i], dv[j]);
            s2[i] = fma2(q, r2, s2[i]);
            sa = fma2(dv[j], g[i], sa);
            sb = fma2(q, g[i], sb);
          }
        }
      sums[2 * k] = sum2(sa);
      sums[2 * k + 1] = sum2(sb) * rstd[k];
    }
    const float mine = warp_sums<2 * R>(sums);
    if ((lane & 7) == 0) red[s & 1][warp][lane >> 3] = mine;
    if (!__syncthreads_and(ok)) return;
    if (a.dx != nullptr) {
      // lanes 8 v .. 8 v + 7 add value v's warp sums, then hand the total round
      float v = (lane & 7) < nw ? red[s & 1][lane & 7][lane >> 3] : 0.0f;
      if ((lane & 7) + 8 < nw) v += red[s & 1][(lane & 7) + 8][lane >> 3];
#pragma unroll
      for (int o = 4; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        // dx = rstd (d g - A - z B) = (d g) rstd + (x c1 + c0)
        const float ma = __shfl_sync(0xffffffffu, v, 16 * k) * inv_d;
        const float mb = __shfl_sync(0xffffffffu, v, 16 * k + 8) * inv_d;
        if (k >= rows) continue;
        const float c1 = -rstd[k] * rstd[k] * mb, c0 = -mean[k] * c1 - rstd[k] * ma;
        const F2 r2 = f2(rstd[k], rstd[k]), c12 = f2(c1, c1), c02 = f2(c0, c0);
        T* dx = static_cast<T*>(a.dx) + (base + s * R + k) * a.D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (VECTOR && t + c * lanes >= nvec) continue;
          F2 d[P], dv[P];
          read(src + 2 * k * p.x_slot, xl[k], c, 0.0f, d);
          if (!VECTOR) read(src + (2 * k + 1) * p.x_slot, dl[k], c, 0.0f, dv);
#pragma unroll
          for (int j = 0; j < P; ++j)
            d[j] = fma2(mul2(VECTOR ? dd[k][c * P + j] : dv[j], g[c * P + j]), r2,
                        fma2(d[j], c12, c02));
          if constexpr (VECTOR) {
            *reinterpret_cast<uint4*>(dx + (t + c * lanes) * VEC) = repack<T>(d);
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const int col = col0 + 32 * (c * VEC + j);
              const float2 f = split(d[j / 2]);
              if (whole || col < a.D) dx[col] = from_f32<T>(j & 1 ? f.y : f.x);
            }
          }
        }
      }
    }
    if (++slot == p.stages) { slot = 0; phase ^= 1; }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int col = VECTOR ? (t + i / VEC * lanes) * VEC + i % VEC : col0 + 32 * i;
    const float2 u = split(s1[i / 2]), v = split(s2[i / 2]);
    if (col < a.D) {
      out[col] = i & 1 ? u.y : u.x;
      out[a.D + col] = i & 1 ? v.y : v.x;
    }
  }
}

// Rows too wide for registers: the row sums and dx by one CTA per row, ...
template <typename T>
__global__ void __launch_bounds__(1024) backward_wide_kernel(const BwdArgs a) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x, smp = row / a.rows_per_mod;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* dy = static_cast<const T*>(a.dy) + row * a.dys;
  const float mean = a.mean[row], rstd = a.rstd[row], inv_d = 1.0f / (float)a.D;
  float sa = 0.0f, sb = 0.0f, g[1];
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
    gain<T, 1>(a.w, a.s, smp, c, g);
    const float i = to_f32<T>(dy[c]) * g[0];
    sa += i;
    sb += i * (to_f32<T>(x[c]) - mean) * rstd;
  }
  const float ma = block_sum(sa, red[0]) * inv_d, mb = block_sum(sb, red[1]) * inv_d;
  T* dx = static_cast<T*>(a.dx) + row * a.D;
  for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
    gain<T, 1>(a.w, a.s, smp, c, g);
    const float z = (to_f32<T>(x[c]) - mean) * rstd;
    dx[c] = from_f32<T>(rstd * (to_f32<T>(dy[c]) * g[0] - ma - z * mb));
  }
}

// ... the column sums by 32-column tiles of each chunk (blockIdx.y the tile).
template <typename T>
__global__ void __launch_bounds__(256) backward_wide_sums_kernel(const BwdArgs a) {
  __shared__ float acc[2][8][32];
  const int c = blockIdx.y * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  const int64_t smp = blockIdx.x / a.chunks;
  const int64_t r0 = (int64_t)(blockIdx.x % a.chunks) * a.chunk_rows;
  const int64_t r1 = r0 + a.chunk_rows < a.rows_per_mod ? r0 + a.chunk_rows : a.rows_per_mod;
  float s1 = 0.0f, s2 = 0.0f;
  if (c < a.D)
    for (int64_t r = r0 + w; r < r1; r += 8) {
      const int64_t row = smp * a.rows_per_mod + r;
      const float d = to_f32<T>(static_cast<const T*>(a.dy)[row * a.dys + c]);
      s1 += d;
      s2 += d * (to_f32<T>(static_cast<const T*>(a.x)[row * a.xs + c]) - a.mean[row]) * a.rstd[row];
    }
  acc[0][w][threadIdx.x & 31] = s1;
  acc[1][w][threadIdx.x & 31] = s2;
  __syncthreads();
  if (w < 2 && c < a.D) {
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += acc[w][k][threadIdx.x & 31];
    a.partial[((int64_t)blockIdx.x * 2 + w) * a.D + c] = v;
  }
}

struct SumArgs {
  const float* partial; int64_t samples; int chunks; int D;
  Param w, b, s;
  void* dw; void* db; void* ds; void* dt;      // any may be null
};

// Sums the partials, 32 columns a CTA, its 16 warps joined in a fixed order.
// blockIdx.y takes samples in turn for dscale and dshift, its warps a sample's
// chunks; with weight gradients wanted, the last blockIdx.y takes all samples'
// chunks at once for them, each times its sample's 1 + s. Runs of 64 terms are
// added up before they join a thread's total, so many samples lose no more
// bits than few.
template <typename T>
__global__ void __launch_bounds__(512) sums_kernel(const SumArgs a) {
  __shared__ float acc[2][16][33];
  constexpr int WARPS = 16, RUN = 64;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  // the warps' sums, joined, in warp 0
  const auto join = [&](float& u, float& v) {
    acc[0][w][lane] = u;
    acc[1][w][lane] = v;
    __syncthreads();
    if (w == 0) {
      u = v = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) { u += acc[0][k][lane]; v += acc[1][k][lane]; }
    }
  };
  const bool weights = a.dw || a.db;
  if (weights && blockIdx.y == gridDim.y - 1) {
    const uint32_t total = (uint32_t)(a.samples * a.chunks);   // at most 2^31
    float dw = 0.0f, db = 0.0f;
    const auto add = [&](auto scaled) {
      for (uint32_t i0 = w; i0 < total; i0 += WARPS * RUN) {
        const uint32_t end = min(total, i0 + WARPS * RUN);
        float rw = 0.0f, rb = 0.0f;
#pragma unroll 8
        for (uint32_t i = i0; i < end; i += WARPS) {
          const float* p = a.partial + i * 2 * (int64_t)a.D + c;
          if constexpr (decltype(scaled)::value) {
            float s[1];
            load_param<T, 1>(a.s, i / (uint32_t)a.chunks, c, s);
            rb = fmaf(1.0f + s[0], __ldg(p), rb);
            rw = fmaf(1.0f + s[0], __ldg(p + a.D), rw);
          } else {
            rb += __ldg(p);
            rw += __ldg(p + a.D);
          }
        }
        dw += rw;
        db += rb;
      }
    };
    if (c < a.D) {
      if (a.s.p) add(std::true_type{});
      else add(std::false_type{});
    }
    join(dw, db);
    if (w == 0 && c < a.D) {
      const auto put = [&](void* o, float v) {
        if (a.w.f32) static_cast<float*>(o)[c] = v;
        else static_cast<T*>(o)[c] = from_f32<T>(v);
      };
      if (a.dw) put(a.dw, dw);
      if (a.db) put(a.db, db);
    }
    return;
  }
  const int rows = gridDim.y - weights;
  for (int64_t smp = blockIdx.y; smp < a.samples; smp += rows) {
    float s1 = 0.0f, s2 = 0.0f;
    if (c < a.D)
      for (int k = w; k < a.chunks; k += WARPS) {
        const float* p = a.partial + (smp * a.chunks + k) * 2 * (int64_t)a.D + c;
        s1 += __ldg(p);
        s2 += __ldg(p + a.D);
      }
    join(s1, s2);
    if (w == 0 && c < a.D) {
      const auto put = [&](void* o, float v) {
        if (a.s.f32) static_cast<float*>(o)[smp * a.D + c] = v;
        else static_cast<T*>(o)[smp * a.D + c] = from_f32<T>(v);
      };
      if (a.dt) put(a.dt, s1);
      if (a.ds) {
        float p[1], v = s2;
        if (a.w.p) { load_param<T, 1>(a.w, 0, c, p); v *= p[0]; }
        if (a.b.p) { load_param<T, 1>(a.b, 0, c, p); v += p[0] * s1; }
        put(a.ds, v);
      }
    }
    __syncthreads();
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// 16-byte access is possible: every base, row stride and sample stride keeps it
template <typename T>
bool vector_ok(int D, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides,
               std::initializer_list<Param> params) {
  constexpr int V = 16 / (int)sizeof(T);
  if (D % V) return false;
  for (const void* p : ptrs) if (!aligned16(p)) return false;
  for (int64_t s : strides) if (s % V) return false;
  for (const Param& a : params)
    if (a.p && (!aligned16(a.p) || a.stride % V)) return false;
  return true;
}

template <typename T, int E, int LO, int L, bool VECTOR>
int forward_l(FwdArgs a, cudaStream_t st) {
  auto kern = forward_kernel<T, E, LO, L, VECTOR>;
  constexpr int most_warps = E <= 32 ? 12 : E <= 64 ? 16 : E <= 96 ? 12 : 8, per_sm = E <= 32 ? 2 : 1;
  const bool mod = a.s.p || a.t.p;
  if (!mod) a.rows_per_mod = a.M;
  const int64_t samples = a.M / a.rows_per_mod;
  FwdPlan p;
  // a copy brings one row, or several that adjoin up to 4 KB (small copies
  // cost their issue, not their bytes), as long as every warp gets one
  const int row = a.D * (int)sizeof(T), sms = sm_count();
  p.slot_rows = 1;
  if (a.xs == a.D) {
    while (p.slot_rows < 16 && 2 * p.slot_rows * row <= 4096 &&
           a.M / (2 * p.slot_rows) >= (int64_t)sms * per_sm * most_warps)
      p.slot_rows *= 2;
    if (a.M >= 32 / L && p.slot_rows < 32 / L) p.slot_rows = 32 / L;
  }
  p.slot_bytes = (uint32_t)(p.slot_rows * row + 15 + 15) / 16 * 16;
  const int fixed = 2 * ((a.D + 3) & ~3) * 4 + 16 * 8 * 8 + 16;
  const int room = 225 * 1024 / per_sm - 1024 - fixed;
  int warps = most_warps;
  const int64_t groups = (a.rows_per_mod + p.slot_rows - 1) / p.slot_rows;
  // two slots a warp at least: one read, one in flight
  while (warps > 1 && warps * 2 * (int)p.slot_bytes > room) --warps;
  while (warps > 1 && samples * ((groups + warps - 1) / warps) < (int64_t)sms * per_sm) --warps;
  p.stages = std::max(2, std::min(4, room / (warps * (int)p.slot_bytes)));
  const int64_t most = (groups + warps - 1) / warps;
  const int64_t want = ((int64_t)sms * per_sm + samples - 1) / samples;
  const int64_t chunks = std::max<int64_t>(1, std::min(most, want));
  p.chunk_rows = (groups + chunks - 1) / chunks * p.slot_rows;
  p.chunks = (int)((a.rows_per_mod + p.chunk_rows - 1) / p.chunk_rows);
  const int64_t blocks = samples * p.chunks;
  if (blocks > 0x7fffffff) return GWB_E_CAPACITY;
  const size_t smem = ((2 * ((a.D + 3) & ~3) * 4 + warps * p.stages * 8 + 15) & ~15) +
                      (size_t)warps * p.stages * p.slot_bytes;
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(reinterpret_cast<const void*>(kern), ready, 225 * 1024)) return GWB_E_LAUNCH;
  // a CTA of few rows has many columns of g and h for few warps
  const bool params = a.w.p || a.b.p || mod;
  p.warps = warps;
  kern<<<(unsigned)blocks, 32 * (params ? std::max(warps, 8) : warps), smem, st>>>(a, p);
  return launch_status();
}

// Lanes a row: eight up to 64 elements (four rows a warp), else 32, with the
// fewest elements a lane that cover it.
template <typename T, bool VECTOR>
int forward_v(const FwdArgs& a, cudaStream_t st) {
  if (a.D <= 64) return forward_l<T, 8, 0, 8, VECTOR>(a, st);
  const int e = (a.D + 31) / 32;
  if (a.D <= 128) return forward_l<T, 16, 8, 8, VECTOR>(a, st);
  if (e <= 8) return forward_l<T, 8, 4, 32, VECTOR>(a, st);
  if (e <= 16) return forward_l<T, 16, 8, 32, VECTOR>(a, st);
  if (e <= 24) return forward_l<T, 24, 16, 32, VECTOR>(a, st);
  if (e <= 32) return forward_l<T, 32, 24, 32, VECTOR>(a, st);
  if (e <= 48) return forward_l<T, 48, 32, 32, VECTOR>(a, st);
  if (e <= 64) return forward_l<T, 64, 48, 32, VECTOR>(a, st);
  if (e <= 96) return forward_l<T, 96, 64, 32, VECTOR>(a, st);
  if (e <= 128) return forward_l<T, 128, 96, 32, VECTOR>(a, st);
  constexpr int V = VECTOR ? 16 / (int)sizeof(T) : 1;
  const int c = (a.D / V + 511) / 512;
  const bool mod_ok = !VECTOR || vector_ok<T>(a.D, {}, {}, {a.w, a.b, a.s, a.t});
  if (mod_ok && c <= 2) forward_block_kernel<T, V, 2><<<(unsigned)a.M, 512, 0, st>>>(a);
  else if (mod_ok && c <= 4) forward_block_kernel<T, V, 4><<<(unsigned)a.M, 512, 0, st>>>(a);
  else if (!VECTOR && c <= 16) forward_block_kernel<T, 1, 16><<<(unsigned)a.M, 512, 0, st>>>(a);
  else forward_wide_kernel<T><<<(unsigned)a.M, 1024, 0, st>>>(a);
  return launch_status();
}

// A CTA a row rather than a warp a row: up to 56 rows a multiprocessor, and for
// wide f32 rows, whose copies leave the other form too few warps (18432 x 3072
// f32: 86 us a call against 99; bf16: 60 against 50).
inline bool pairs_fit(const FwdArgs& a, int V) {
  if (a.D / V <= 32 || a.D > 4096) return false;
  return (V == 4 && a.D > 2048) || a.M <= (int64_t)sm_count() * 56;
}
template <typename T>
int forward_pairs(const FwdArgs& a, cudaStream_t st) {
  // three vectors a thread, up to 512 threads
  const int nvec = a.D / (16 / (int)sizeof(T));
  int th = 32;
  while (th < 512 && nvec > th * 3) th *= 2;
  const int c = (nvec + th - 1) / th;
  const unsigned m = (unsigned)a.M;
  if (c <= 1) forward_pairs_kernel<T, 1><<<m, th, 0, st>>>(a);
  else if (c <= 2) forward_pairs_kernel<T, 2><<<m, th, 0, st>>>(a);
  else if (c <= 3) forward_pairs_kernel<T, 3><<<m, th, 0, st>>>(a);
  else forward_pairs_kernel<T, 4><<<m, th, 0, st>>>(a);
  return launch_status();
}

template <typename T>
int forward_t(const FwdArgs& a, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool vector = a.D % V == 0 && a.xs % V == 0 && aligned16(a.x) && aligned16(a.y);
  if (vector && pairs_fit(a, V) && vector_ok<T>(a.D, {}, {}, {a.w, a.b, a.s, a.t}))
    return forward_pairs<T>(a, st);
  return vector ? forward_v<T, true>(a, st) : forward_v<T, false>(a, st);
}

template <typename T, int VEC, int C>
int backward_c(const BwdArgs& a, int64_t blocks, cudaStream_t st) {
  const size_t smem = a.partial ? (size_t)8 * 2 * a.D * sizeof(float) : 0;
  backward_kernel<T, VEC, C><<<(unsigned)blocks, 256, smem, st>>>(a);
  return launch_status();
}

template <typename T, int E, bool VECTOR>
int backward_staged_e(const BwdArgs& a, int64_t blocks, int64_t rows, int th, cudaStream_t st) {
  auto kern = backward_staged_kernel<T, E, VECTOR>;
  // the CTAs that the register file holds share the shared memory: three
  // slots at least (one read, one being freed, one in flight)
  const int per_sm = std::max(1, std::min(8, 65536 / ((th + 32) * (E <= 8 ? 72 : 128))));
  BwdPlan p;
  p.x_slot = (uint32_t)(a.D * (int)sizeof(T) + 15 + 15) / 16 * 16;
  p.last = rows - 1;
  const int slot = 4 * (int)p.x_slot;
  p.stages = std::max(3, std::min(8, (220 * 1024 / per_sm - 2048) / slot));
  const size_t smem = (size_t)p.stages * slot;
  if (smem > 226 * 1024) return GWB_E_SHAPE;
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(reinterpret_cast<const void*>(kern), ready, 226 * 1024)) return GWB_E_LAUNCH;
  kern<<<(unsigned)blocks, th + 32, smem, st>>>(a, p);
  return launch_status();
}

// Eight columns a thread up to 384 threads, sixteen up to 480, then 24 (the
// register file's shares); rows whose three slots pass the shared memory take the wide form.
inline bool staged_fits(int D, int size) { return D <= 8192 && 3 * 4 * (D * size + 30) <= 226 * 1024; }
template <typename T, bool VECTOR>
int backward_staged(const BwdArgs& a, int64_t blocks, int64_t rows, cudaStream_t st) {
  const int unit = (a.D + 7) / 8;
  if (unit <= 384)
    return backward_staged_e<T, 8, VECTOR>(a, blocks, rows, (unit + 31) / 32 * 32, st);
  if (unit <= 2 * 480)
    return backward_staged_e<T, 16, VECTOR>(a, blocks, rows, ((a.D + 15) / 16 + 31) / 32 * 32, st);
  return backward_staged_e<T, 24, VECTOR>(a, blocks, rows, ((a.D + 23) / 24 + 31) / 32 * 32, st);
}

template <typename T, int VEC>
int backward_v(const BwdArgs& a, int64_t samples, cudaStream_t st) {
  const int64_t blocks = samples * a.chunks, rows = samples * a.rows_per_mod;
  const int nvec = a.D / VEC;
  if (nvec <= 32) return backward_c<T, VEC, 1>(a, blocks, st);
  if (nvec <= 64) return backward_c<T, VEC, 2>(a, blocks, st);
  if (staged_fits(a.D, sizeof(T))) return backward_staged<T, (VEC > 1)>(a, blocks, rows, st);
  if (a.dx) {
    backward_wide_kernel<T><<<(unsigned)rows, 1024, 0, st>>>(a);
    if (int rc = launch_status()) return rc;
  }
  if (a.partial) {
    backward_wide_sums_kernel<T><<<dim3((unsigned)blocks, (a.D + 31) / 32), 256, 0, st>>>(a);
    return launch_status();
  }
  return GWB_SUCCESS;
}

template <typename T>
int backward_t(const BwdArgs& a, int64_t samples, const SumArgs& sums, bool want_sums,
               cudaStream_t st) {
  int rc = GWB_SUCCESS;
  if (a.dx || a.partial) {
    if (vector_ok<T>(a.D, {a.x, a.dy, a.dx}, {a.xs, a.dys}, {a.w, a.s}))
      rc = backward_v<T, 16 / (int)sizeof(T)>(a, samples, st);
    else
      rc = backward_v<T, 1>(a, samples, st);
  }
  if (rc || !want_sums) return rc;
  const unsigned y = (sums.ds || sums.dt ? (unsigned)std::min<int64_t>(samples, 65534) : 0u) +
                     (sums.dw || sums.db ? 1u : 0u);
  sums_kernel<T><<<dim3((a.D + 31) / 32, y), 512, 0, st>>>(sums);
  return launch_status();
}

// Chunks a sample's rows are split into for the backward pass: over all
// samples as many CTAs as run at once (two a multiprocessor for wide rows,
// four for narrow ones), no chunk under eight rows (below that the partials
// outweigh the rows).
inline int chunks_of(int64_t samples, int64_t rows_per_mod, int64_t D) {
  if (samples <= 0 || rows_per_mod <= 0) return 1;
  const int64_t want = (148 * (D > 1536 ? 2 : 4) + samples - 1) / samples;
  const int64_t most = (rows_per_mod + 7) / 8;
  const int64_t c = want < most ? want : most;
  return (int)(c < 1 ? 1 : c);
}

}  // namespace norm

int launch_layer_norm(const norm::FwdArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case GWB_F32: return norm::forward_t<float>(a, st);
    case GWB_BF16: return norm::forward_t<__nv_bfloat16>(a, st);
    case GWB_F16: return norm::forward_t<__half>(a, st);
  }
  return GWB_E_SHAPE;
}

int launch_layer_norm_backward(const norm::BwdArgs& a, int64_t samples, const norm::SumArgs& sums,
                               bool want_sums, int dtype, cudaStream_t st) {
  switch (dtype) {
    case GWB_F32: return norm::backward_t<float>(a, samples, sums, want_sums, st);
    case GWB_BF16: return norm::backward_t<__nv_bfloat16>(a, samples, sums, want_sums, st);
    case GWB_F16: return norm::backward_t<__half>(a, samples, sums, want_sums, st);
  }
  return GWB_E_SHAPE;
}

}  // namespace gwb
