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
// each output is rounded once.
//
// HBM bounds both directions: x in and y out forward, x and dy in and dx out
// backward. Column sums go through per-CTA partials and a second kernel in a
// fixed order, without atomics, so gradients are the same on every run.
#include <cuda_runtime.h>
#include "gwb.h"
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

// One row per warp (WARP, four rows per CTA) or per CTA; the row stays in
// registers, C vectors a thread, between the statistics and the output.
template <typename T, int VEC, int C, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024)
forward_kernel(const FwdArgs a) {
  __shared__ float red[2][32];
  const int lanes = WARP ? 32 : blockDim.x;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= a.M) return;
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
  const float mean = (WARP ? warp_sum(sum) : block_sum(sum, red[0])) * inv_d;
  float sq = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (t + c * lanes < nvec)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[c][j] -= mean;
        sq += v[c][j] * v[c][j];
      }
  const float var = (WARP ? warp_sum(sq) : block_sum(sq, red[1])) * inv_d;
  const float rstd = 1.0f / sqrtf(var + a.eps);
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
  const float mean = block_sum(sum, red[0]) * inv_d;
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

// CTA blockIdx.x takes one chunk of one sample's rows. WARP: its eight warps
// take rows in turn, one row a warp; else the CTA takes R rows at a time and
// each thread keeps its C vectors of columns, so S1 and S2 stay in its
// registers for the whole chunk and the 2 R row sums share two barriers.
template <typename T, int VEC, int C, int R, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
backward_kernel(const BwdArgs a) {
  extern __shared__ float part_sm[];             // WARP: [8][2][D]
  __shared__ float red[2][32][2 * R];
  const int lanes = WARP ? 32 : blockDim.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = WARP ? lane : threadIdx.x;
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
    if (t + c * lanes < nvec) gain<T, VEC>(a.w, a.s, smp, (t + c * lanes) * VEC, g[c]);
  }
  const int64_t step = WARP ? (int64_t)(blockDim.x >> 5) * R : R;
  int flip = 0;
  for (int64_t r = r0 + (WARP ? warp * R : 0); r < r1; r += step, flip ^= 1) {
    Pack<T, VEC> xv[R][C], dv[R][C];
    float mean[R], rstd[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const bool live = r + k < r1;
      const int64_t row = base + (live ? r + k : r);
      mean[k] = __ldg(a.mean + row);
      rstd[k] = __ldg(a.rstd + row);
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (t + c * lanes < nvec) {
          xv[k][c].load(static_cast<const T*>(a.x) + row * a.xs + (t + c * lanes) * VEC);
          dv[k][c].load(static_cast<const T*>(a.dy) + row * a.dys + (t + c * lanes) * VEC);
        }
    }
    float sa[R], sb[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      sa[k] = sb[k] = 0.0f;
      if (r + k < r1)
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (t + c * lanes < nvec)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const float z = (xv[k][c].get(j) - mean[k]) * rstd[k], d = dv[k][c].get(j);
              s1[c][j] += d;
              s2[c][j] += d * z;
              const float i = d * g[c][j];
              sa[k] += i;
              sb[k] += i * z;
            }
    }
    if (a.dx == nullptr) continue;
#pragma unroll
    for (int k = 0; k < R; ++k) { sa[k] = warp_sum(sa[k]); sb[k] = warp_sum(sb[k]); }
    if constexpr (!WARP) {
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < R; ++k) { red[flip][warp][2 * k] = sa[k]; red[flip][warp][2 * k + 1] = sb[k]; }
      __syncthreads();
      const int nw = blockDim.x >> 5;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        sa[k] = warp_sum(lane < nw ? red[flip][lane][2 * k] : 0.0f);
        sb[k] = warp_sum(lane < nw ? red[flip][lane][2 * k + 1] : 0.0f);
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (r + k >= r1) continue;
      const float ma = sa[k] * inv_d, mb = sb[k] * inv_d;
      T* dx = static_cast<T*>(a.dx) + (base + r + k) * a.D;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (t + c * lanes < nvec) {
          Pack<T, VEC> o;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float z = (xv[k][c].get(j) - mean[k]) * rstd[k];
            o.set(j, rstd[k] * (dv[k][c].get(j) * g[c][j] - ma - z * mb));
          }
          o.store(dx + (t + c * lanes) * VEC);
        }
    }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.D;
  if constexpr (WARP) {
    float* mine = part_sm + warp * 2 * a.D;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (t + c * lanes < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          mine[(t + c * lanes) * VEC + j] = s1[c][j];
          mine[a.D + (t + c * lanes) * VEC + j] = s2[c][j];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += blockDim.x) {
      float v = 0.0f;
      for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += part_sm[w * 2 * a.D + i];
      out[i] = v;
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (t + c * lanes < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          out[(t + c * lanes) * VEC + j] = s1[c][j];
          out[a.D + (t + c * lanes) * VEC + j] = s2[c][j];
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

// Sums the partials over each sample's chunks: 32 columns a CTA, its 16 warps
// taking chunks in turn, joined in a fixed order. One sample per blockIdx.y,
// or (weight gradients wanted) all samples in turn.
template <typename T>
__global__ void __launch_bounds__(512) sums_kernel(const SumArgs a) {
  __shared__ float acc[2][16][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const bool all = gridDim.y == 1;
  float dw = 0.0f, db = 0.0f;
  for (int64_t smp = blockIdx.y; smp < a.samples; smp += gridDim.y) {
    float s1 = 0.0f, s2 = 0.0f;
    if (c < a.D)
      for (int k = w; k < a.chunks; k += 16) {
        const float* p = a.partial + (smp * a.chunks + k) * 2 * (int64_t)a.D + c;
        s1 += __ldg(p);
        s2 += __ldg(p + a.D);
      }
    acc[0][w][lane] = s1;
    acc[1][w][lane] = s2;
    __syncthreads();
    if (w == 0 && c < a.D) {
      s1 = s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) { s1 += acc[0][k][lane]; s2 += acc[1][k][lane]; }
      float p[1], up = 1.0f;
      if (a.s.p) { load_param<T, 1>(a.s, smp, c, p); up += p[0]; }
      dw += up * s2;
      db += up * s1;
      const auto put = [&](void* o, int f32, float v) {
        if (f32) static_cast<float*>(o)[smp * a.D + c] = v;
        else static_cast<T*>(o)[smp * a.D + c] = from_f32<T>(v);
      };
      if (a.dt) put(a.dt, a.s.f32, s1);
      if (a.ds) {
        float v = s2;
        if (a.w.p) { load_param<T, 1>(a.w, 0, c, p); v *= p[0]; }
        if (a.b.p) { load_param<T, 1>(a.b, 0, c, p); v += p[0] * s1; }
        put(a.ds, a.s.f32, v);
      }
    }
    __syncthreads();
  }
  if (all && w == 0 && c < a.D) {
    const auto put = [&](void* o, float v) {
      if (a.w.f32) static_cast<float*>(o)[c] = v;
      else static_cast<T*>(o)[c] = from_f32<T>(v);
    };
    if (a.dw) put(a.dw, dw);
    if (a.db) put(a.db, db);
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

template <typename T, int VEC, int C>
int forward_c(const FwdArgs& a, int th, cudaStream_t st) {
  if (th == 32) forward_kernel<T, VEC, C, true><<<(unsigned)((a.M + 3) / 4), 128, 0, st>>>(a);
  else forward_kernel<T, VEC, C, false><<<(unsigned)a.M, th, 0, st>>>(a);
  return launch_status();
}

// Threads a row: the fewest warps that keep a thread at four vectors (one
// warp needs no barrier; more rows in flight beat more threads a row), the
// register file's limit being 1024 threads.
template <typename T, int VEC>
int forward_v(const FwdArgs& a, cudaStream_t st) {
  constexpr int CMAX = VEC == 1 ? 8 : 4;
  const int nvec = a.D / VEC;
  int th = 32;
  while (th < 1024 && nvec > th * CMAX) th *= 2;
  if (nvec > th * CMAX) {
    forward_wide_kernel<T><<<(unsigned)a.M, 1024, 0, st>>>(a);
    return launch_status();
  }
  const int c = (nvec + th - 1) / th;
  if (c <= 1) return forward_c<T, VEC, 1>(a, th, st);
  if (c <= 2) return forward_c<T, VEC, 2>(a, th, st);
  if (c <= 3) return forward_c<T, VEC, 3>(a, th, st);
  if (c <= 4) return forward_c<T, VEC, 4>(a, th, st);
  if constexpr (CMAX > 4) return forward_c<T, VEC, 8>(a, th, st);
  return GWB_E_SHAPE;
}

template <typename T>
int forward_t(const FwdArgs& a, cudaStream_t st) {
  if (vector_ok<T>(a.D, {a.x, a.y}, {a.xs}, {a.w, a.b, a.s, a.t}))
    return forward_v<T, 16 / (int)sizeof(T)>(a, st);
  return forward_v<T, 1>(a, st);
}

template <typename T, int VEC, int C, bool WARP>
int backward_c(const BwdArgs& a, int64_t blocks, int th, cudaStream_t st) {
  // rows a step: as many as keep x, dy, the gain and both sums in the 128
  // registers that 512 threads leave each other
  constexpr int E = VEC * C, WIDE = sizeof(T) == 4 || VEC == 1;
  constexpr int R = WARP ? 1 : E <= 4 ? 4 : E <= 8 ? (WIDE ? 2 : 4) : (WIDE ? 1 : 2);
  const size_t smem = WARP && a.partial ? (size_t)8 * 2 * a.D * sizeof(float) : 0;
  backward_kernel<T, VEC, C, R, WARP><<<(unsigned)blocks, th, smem, st>>>(a);
  return launch_status();
}

template <typename T, int VEC>
int backward_v(const BwdArgs& a, int64_t samples, cudaStream_t st) {
  const int64_t blocks = samples * a.chunks;
  const int nvec = a.D / VEC;
  constexpr int E = 16 / VEC;        // columns a thread: at most 16
  if (nvec > 512 * E) {
    if (a.dx) {
      backward_wide_kernel<T><<<(unsigned)(samples * a.rows_per_mod), 1024, 0, st>>>(a);
      if (int rc = launch_status()) return rc;
    }
    if (a.partial) {
      backward_wide_sums_kernel<T><<<dim3((unsigned)blocks, (a.D + 31) / 32), 256, 0, st>>>(a);
      return launch_status();
    }
    return GWB_SUCCESS;
  }
  if (nvec <= 32) return backward_c<T, VEC, 1, true>(a, blocks, 256, st);
  if (nvec <= 64) return backward_c<T, VEC, 2, true>(a, blocks, 256, st);
  int c = 1;
  while (nvec > 512 * c) c *= 2;
  const int th = ((nvec + c - 1) / c + 31) / 32 * 32;
  if (c == 1) return backward_c<T, VEC, 1, false>(a, blocks, th, st);
  if (c == 2) return backward_c<T, VEC, 2, false>(a, blocks, th, st);
  if constexpr (E >= 4)
    if (c == 4) return backward_c<T, VEC, 4, false>(a, blocks, th, st);
  if constexpr (E >= 8)
    if (c == 8) return backward_c<T, VEC, 8, false>(a, blocks, th, st);
  if constexpr (E >= 16)
    if (c == 16) return backward_c<T, VEC, 16, false>(a, blocks, th, st);
  return GWB_E_SHAPE;
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
  const bool all = sums.dw || sums.db;
  const unsigned y = all ? 1u : (unsigned)(samples < 65535 ? samples : 65535);
  sums_kernel<T><<<dim3((a.D + 31) / 32, y > 0 ? y : 1), 512, 0, st>>>(sums);
  return launch_status();
}

// Chunks a sample's rows are split into for the backward pass: four CTAs a
// multiprocessor over all samples (their barriers then overlap), no chunk
// under eight rows (below that the partials outweigh the rows).
inline int chunks_of(int64_t samples, int64_t rows_per_mod) {
  if (samples <= 0 || rows_per_mod <= 0) return 1;
  const int64_t want = (148 * 4 + samples - 1) / samples;
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
