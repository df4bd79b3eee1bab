// Rotary positions of queries and keys: feature pairs (a, b) of each head's
// first 2 n features turn by t = position * inv_freq,
//   (a, b) -> c (a cos t - b sin t, b cos t + a sin t),
// c the attention scale of a long-context extension; the remaining features
// pass through. Pairs are (i, n + i) (half layout) or (2 i, 2 i + 1)
// (interleaved). The backward pass is the same map by -t.
//
// Angles: t is reduced to a fraction of a turn in f64 (position *
// inv_freq / 2 pi minus its nearest integer), then sincospi in f32: an f32
// product would lose 2^-24 of the whole angle, 0.06 rad at position 2^20.
// Cosines and sines of a token are computed once per CTA into shared memory
// and used by all of its heads. HBM bounds it: q and k are read and written
// once; queries and keys share one launch.
#include <cuda_runtime.h>
#include "gwb.h"
#include "elem.cuh"

namespace gwb {
namespace rotary {

struct Heads {                     // q or k: [B, S, H, Dh] by strides, last dim dense
  const void* x; void* y;
  int64_t xb, xs, xh, yb, ys, yh;  // element strides
  int h;
};

struct Args {
  Heads q, k;                      // k.h == 0: no keys
  const void* pos; int pos_kind;   // 0 i64, 1 i32, 2 f32
  int64_t pb, ps, pa;              // position strides: batch, token, axis
  const double* inv_freq;          // [n]
  const int* axis;                 // [n] or null (axis 0)
  int axes;                        // position axes
  int64_t tokens; int S;           // B * S, S
  int n, dh;                       // rotated pairs, head size
  float scale; int inverse, in_place;
  int split;                       // CTAs that share a token's heads
  int per_cta;                     // tokens a CTA takes
};

constexpr double kInvTwoPi = 0.15915494309189533576888;

__device__ __forceinline__ double position_of(const Args& a, int64_t b, int64_t s, int axis) {
  const int64_t at = b * a.pb + s * a.ps + axis * a.pa;
  if (a.pos_kind == 0) return (double)static_cast<const long long*>(a.pos)[at];
  if (a.pos_kind == 1) return (double)static_cast<const int*>(a.pos)[at];
  return (double)static_cast<const float*>(a.pos)[at];
}

// Threads (x, y): x walks one head's items, y the heads. An item is one
// vector of pairs (two 16-byte accesses in the half layout, one interleaved)
// or, out of place, one vector of the features that pass through.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const Args a) {
  extern __shared__ float2 turn[];             // [per_cta][n] (c cos, c sin)
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, nthreads = blockDim.x * blockDim.y;
  const int64_t t0 = (int64_t)(blockIdx.x / a.split) * a.per_cta;
  const int part = blockIdx.x % a.split;
  const int nt = (int)(a.tokens - t0 < a.per_cta ? a.tokens - t0 : a.per_cta);
  for (int i = tid; i < nt * a.n; i += nthreads) {
    const int64_t tok = t0 + i / a.n;
    const int f = i % a.n;
    int ax = a.axis ? a.axis[f] : 0;
    ax = ax < 0 ? 0 : ax >= a.axes ? a.axes - 1 : ax;   // a bad axis reads no stray position
    const double p = position_of(a, tok / a.S, tok % a.S, ax);
    const double turns = p * a.inv_freq[f] * kInvTwoPi;
    const float frac = (float)(turns - rint(turns));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    turn[i] = make_float2(cs * a.scale, (a.inverse ? -sn : sn) * a.scale);
  }
  __syncthreads();
  // items: rotated vectors, then (out of place) pass-through vectors
  constexpr int PAIRS = INTERLEAVED && VEC > 1 ? VEC / 2 : VEC;   // pairs an item
  const int rot_items = a.n / PAIRS;
  const int rest = a.dh - 2 * a.n;
  const int items = rot_items + (a.in_place ? 0 : rest / VEC);
  const int heads = a.q.h + a.k.h;
  for (int k = 0; k < nt; ++k) {
    const int64_t tok = t0 + k, b = tok / a.S, s = tok % a.S;
    const float2* tr = turn + k * a.n;
    for (int h = part * blockDim.y + threadIdx.y; h < heads; h += blockDim.y * a.split) {
      const bool is_k = h >= a.q.h;
      const Heads& w = is_k ? a.k : a.q;
      const int hh = is_k ? h - a.q.h : h;
      const T* x = static_cast<const T*>(w.x) + b * w.xb + s * w.xs + hh * w.xh;
      T* y = static_cast<T*>(w.y) + b * w.yb + s * w.ys + hh * w.yh;
      for (int i = threadIdx.x; i < items; i += blockDim.x) {
        if (i < rot_items) {
          if constexpr (INTERLEAVED && VEC > 1) {
            Pack<T, VEC> v;
            v.load(x + i * VEC);
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
              const float2 c = tr[i * PAIRS + j / 2];
              const float p = v.get(j), r = v.get(j + 1);
              v.set(j, p * c.x - r * c.y);
              v.set(j + 1, r * c.x + p * c.y);
            }
            v.store(y + i * VEC);
          } else {
            const int ia = INTERLEAVED ? 2 * i : i * VEC, ib = INTERLEAVED ? ia + 1 : a.n + ia;
            Pack<T, VEC> va, vb;
            va.load(x + ia);
            vb.load(x + ib);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const float2 c = tr[i * VEC + j];
              const float p = va.get(j), r = vb.get(j);
              va.set(j, p * c.x - r * c.y);
              vb.set(j, r * c.x + p * c.y);
            }
            va.store(y + ia);
            vb.store(y + ib);
          }
        } else {
          const int at = 2 * a.n + (i - rot_items) * VEC;
          Pack<T, VEC> v;
          v.load(x + at);
          v.store(y + at);
        }
      }
    }
  }
}

inline bool vec_heads(const Heads& w, int V) {
  if (w.h == 0) return true;
  return ((reinterpret_cast<uintptr_t>(w.x) | reinterpret_cast<uintptr_t>(w.y)) & 15u) == 0 &&
         w.xb % V == 0 && w.xs % V == 0 && w.xh % V == 0 && w.yb % V == 0 && w.ys % V == 0 &&
         w.yh % V == 0;
}

template <typename T, int VEC, bool INTERLEAVED>
int launch_v(Args a, cudaStream_t st) {
  constexpr int PAIRS = INTERLEAVED && VEC > 1 ? VEC / 2 : VEC;
  const int items = a.n / PAIRS + (a.in_place ? 0 : (a.dh - 2 * a.n) / VEC);
  const int heads = a.q.h + a.k.h;
  const int bx = items < 256 ? (items > 0 ? items : 1) : 256;
  int by = 256 / bx;
  if (by > heads) by = heads;
  // With few tokens a token's heads are split over CTAs until the GPU has two
  // CTAs a multiprocessor (each repeats the token's angles, n of them); with
  // many, a CTA takes tokens until its threads have two items each, as far
  // as the angles fit.
  a.split = 1;
  a.per_cta = 1;
  const int most_split = (heads + by - 1) / by;
  if (a.tokens < 296) {
    const int64_t want = (296 + a.tokens - 1) / a.tokens;
    a.split = (int)(want < most_split ? want : most_split);
  } else {
    const int rows = (heads + by - 1) / by;
    const int xs = (items + bx - 1) / bx;
    while (a.per_cta < 8 && a.per_cta * rows * xs < 2 && a.tokens / (a.per_cta * 2) >= 148 * 8 &&
           (a.per_cta * 2) * a.n <= 4096)
      a.per_cta *= 2;
  }
  const int64_t blocks = (a.tokens + a.per_cta - 1) / a.per_cta * a.split;
  if (blocks > 0x7fffffff) return GWB_E_CAPACITY;
  const size_t smem = (size_t)a.per_cta * a.n * sizeof(float2);
  rotary_kernel<T, VEC, INTERLEAVED><<<(unsigned)blocks, dim3(bx, by), smem, st>>>(a);
  return launch_status();
}

template <typename T>
int launch_t(const Args& a, bool interleaved, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = vec_heads(a.q, V) && vec_heads(a.k, V) && a.dh % V == 0 &&
                   (interleaved ? (2 * a.n) % V == 0 : a.n % V == 0);
  if (interleaved) return vec ? launch_v<T, V, true>(a, st) : launch_v<T, 1, true>(a, st);
  return vec ? launch_v<T, V, false>(a, st) : launch_v<T, 1, false>(a, st);
}

}  // namespace rotary

int launch_rotary(const rotary::Args& a, bool interleaved, int dtype, cudaStream_t st) {
  switch (dtype) {
    case GWB_F32: return rotary::launch_t<float>(a, interleaved, st);
    case GWB_BF16: return rotary::launch_t<__nv_bfloat16>(a, interleaved, st);
    case GWB_F16: return rotary::launch_t<__half>(a, interleaved, st);
  }
  return GWB_E_SHAPE;
}

}  // namespace gwb
