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

// Division of n < 2^31 by a fixed d as a multiply and a shift.
struct FastDiv {
  uint32_t d, m, s;
  __host__ static FastDiv of(uint32_t d) {
    FastDiv f{d, 0, 0};
    while ((1ull << f.s) < d) ++f.s;                 // ceil(log2 d)
    f.m = (uint32_t)(((1ull << 32) * ((1ull << f.s) - d)) / d + 1);
    return f;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return (uint32_t)(((uint64_t)__umulhi(n, m) + n) >> s);
  }
};

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
  int64_t total;                   // units of all tokens
  int chunk;                       // units a CTA takes
  int items, rot_items;            // of a head
  int per_thread;                  // heads a thread
  FastDiv by_token, by_item, by_seq, by_n;   // units of a token, items, S, n
};

constexpr double kInvTwoPi = 0.15915494309189533576888;

__device__ __forceinline__ double position_of(const Args& a, int64_t b, int64_t s, int axis) {
  const int64_t at = b * a.pb + s * a.ps + axis * a.pa;
  if (a.pos_kind == 0) return (double)static_cast<const long long*>(a.pos)[at];
  if (a.pos_kind == 1) return (double)static_cast<const int*>(a.pos)[at];
  return (double)static_cast<const float*>(a.pos)[at];
}

// The rotation, with its roundings in one order in every form, so that a
// tensor's alignment does not change its bits.
__device__ __forceinline__ float first_of(float p, float r, float c, float s) {
  return fmaf(r, -s, __fmul_rn(p, c));
}
__device__ __forceinline__ float second_of(float p, float r, float c, float s) {
  return fmaf(p, s, __fmul_rn(r, c));
}

// An item is one vector of pairs (two 16-byte accesses in the half layout,
// one interleaved) or, out of place, one vector of the features that pass
// through. A thread takes one item of up to HEADS consecutive heads of a
// token: the indices and the item's cosines and sines are worked out once for
// all of them, and their loads are in flight together. A CTA takes a run of
// consecutive units (token, group of heads, item), so sizes that divide by
// nothing leave no thread idle; its loads are in flight while it works out
// the angles. (An item and head a thread spent more
// instructions on indices than on the rotation: 41 us against 22 at 4608
// tokens of 48 interleaved bf16 heads of 128, 5.0 TB/s.)
constexpr int THREADS = 256;
// heads a thread: 32 registers of loads in flight, or eight elements
template <int VEC, bool INTERLEAVED> constexpr int heads_of() {
  return INTERLEAVED && VEC > 1 ? 8 : 4;
}

template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, 4) rotary_kernel(const Args a) {
  extern __shared__ __align__(16) float turn[];          // [tokens of the run][2][n] c cos, c sin
  constexpr bool ONE = INTERLEAVED && VEC > 1;           // one access an item
  constexpr int PAIRS = ONE ? VEC / 2 : VEC;             // pairs an item
  constexpr int HEADS = heads_of<VEC, INTERLEAVED>();
  const int64_t u0 = (int64_t)blockIdx.x * a.chunk;
  const int count = (int)(a.total - u0 < a.chunk ? a.total - u0 : a.chunk);
  const uint32_t tok0 = (uint32_t)(u0 / a.by_token.d), lead = (uint32_t)(u0 % a.by_token.d);
  const uint32_t n = lead + threadIdx.x, k = a.by_token.div(n), rem = n - k * a.by_token.d;
  const uint32_t grp = a.by_item.div(rem);
  const int item = (int)(rem - grp * a.by_item.d);
  const uint32_t tok = tok0 + k, b = a.by_seq.div(tok), s = tok - b * a.by_seq.d;
  const int h0 = (int)grp * a.per_thread;
  const int hn = (int)threadIdx.x < count ? min(a.per_thread, a.q.h + a.k.h - h0) : 0;
  const bool rot = item < a.rot_items;
  // offset of the item's first vector, and of its second from there
  const int ia = rot ? (ONE ? item * VEC : INTERLEAVED ? 2 * item : item * VEC)
                     : 2 * a.n + (item - a.rot_items) * VEC;
  const int gap = INTERLEAVED ? 1 : a.n;
  Pack<T, VEC> va[HEADS], vb[ONE ? 1 : HEADS];
  {
    const T* qx = static_cast<const T*>(a.q.x) + b * a.q.xb + s * a.q.xs + ia;
    const T* kx = static_cast<const T*>(a.k.x) + b * a.k.xb + s * a.k.xs + ia;
#pragma unroll
    for (int j = 0; j < HEADS; ++j)
      if (j < hn) {
        const int h = h0 + j;
        const T* x = h < a.q.h ? qx + h * a.q.xh : kx + (h - a.q.h) * a.k.xh;
        va[j].load(x);
        if constexpr (!ONE) if (rot) vb[j].load(x + gap);
      }
  }
  // the angles, while the loads are in flight
  const int nt = (int)a.by_token.div(lead + count - 1) + 1;
  for (int i = threadIdx.x; i < nt * a.n; i += THREADS) {
    const uint32_t kk = a.by_n.div(i), f = i - kk * a.n, tk = tok0 + kk;
    const uint32_t bb = a.by_seq.div(tk), ss = tk - bb * a.by_seq.d;
    int ax = a.axis ? a.axis[f] : 0;
    ax = ax < 0 ? 0 : ax >= a.axes ? a.axes - 1 : ax;   // a bad axis reads no stray position
    const double turns = position_of(a, bb, ss, ax) * a.inv_freq[f] * kInvTwoPi;
    const float frac = (float)(turns - rint(turns));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    turn[2 * kk * a.n + f] = cs * a.scale;
    turn[(2 * kk + 1) * a.n + f] = (a.inverse ? -sn : sn) * a.scale;
  }
  __syncthreads();
  float c[PAIRS], sn[PAIRS];
  if (rot && hn > 0) {
    const float* tr = turn + 2 * k * a.n + item * PAIRS;
    if constexpr (PAIRS % 4 == 0) {
#pragma unroll
      for (int e = 0; e < PAIRS; e += 4) {
        *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(tr + e);
        *reinterpret_cast<float4*>(sn + e) = *reinterpret_cast<const float4*>(tr + a.n + e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) { c[e] = tr[e]; sn[e] = tr[a.n + e]; }
    }
  }
  T* qy = static_cast<T*>(a.q.y) + b * a.q.yb + s * a.q.ys + ia;
  T* ky = static_cast<T*>(a.k.y) + b * a.k.yb + s * a.k.ys + ia;
#pragma unroll
  for (int j = 0; j < HEADS; ++j)
    if (j < hn) {
      const int h = h0 + j;
      T* y = h < a.q.h ? qy + h * a.q.yh : ky + (h - a.q.h) * a.k.yh;
      if (rot) {
        if constexpr (VEC == 1) {
          const float p = va[j].get(0), r = vb[j].get(0);
          va[j].set(0, first_of(p, r, c[0], sn[0]));
          vb[j].set(0, second_of(p, r, c[0], sn[0]));
          vb[j].store(y + gap);
        } else if constexpr (ONE) {
          F2 v[PAIRS];
          unpack<T>(va[j].bits(), v);
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) {
            const float2 f = split(v[e]);
            v[e] = f2(first_of(f.x, f.y, c[e], sn[e]), second_of(f.x, f.y, c[e], sn[e]));
          }
          va[j].put(repack<T>(v));
        } else {
          F2 p[PAIRS / 2], r[PAIRS / 2];
          unpack<T>(va[j].bits(), p);
          unpack<T>(vb[j].bits(), r);
#pragma unroll
          for (int e = 0; e < PAIRS / 2; ++e) {
            const F2 c2 = f2(c[2 * e], c[2 * e + 1]), s2 = f2(sn[2 * e], sn[2 * e + 1]);
            const F2 n2 = f2(-sn[2 * e], -sn[2 * e + 1]);
            const F2 u = fma2(r[e], n2, mul2(p[e], c2));
            r[e] = fma2(p[e], s2, mul2(r[e], c2));
            p[e] = u;
          }
          va[j].put(repack<T>(p));
          vb[j].put(repack<T>(r));
          vb[j].store(y + gap);
        }
      }
      va[j].store(y);
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
  a.rot_items = a.n / PAIRS;
  a.items = a.rot_items + (a.in_place ? 0 : (a.dh - 2 * a.n) / VEC);
  const int heads = a.q.h + a.k.h;
  // heads a thread: as many as still give every multiprocessor four CTAs
  a.per_thread = heads_of<VEC, INTERLEAVED>();
  while (a.per_thread > 1 &&
         a.tokens * ((heads + a.per_thread - 1) / a.per_thread) * a.items < (int64_t)148 * 4 * THREADS)
    a.per_thread /= 2;
  const int64_t groups = (heads + a.per_thread - 1) / a.per_thread, per_token = groups * a.items;
  if (per_token > 1 << 24) return GWB_E_CAPACITY;
  a.total = a.tokens * per_token;
  a.by_token = FastDiv::of((uint32_t)per_token);
  a.by_item = FastDiv::of((uint32_t)a.items);
  a.by_seq = FastDiv::of((uint32_t)a.S);
  a.by_n = FastDiv::of((uint32_t)(a.n > 0 ? a.n : 1));
  // units a CTA: one a thread, as many as the angles of their tokens fit in 48 KB
  a.chunk = THREADS;
  const auto tokens = [&](int chunk) { return (chunk + per_token - 2) / per_token + 1; };
  while (a.chunk > 8 && tokens(a.chunk) * a.n * 2 * (int64_t)sizeof(float) > 48 * 1024) a.chunk /= 2;
  const int64_t blocks = (a.total + a.chunk - 1) / a.chunk;
  if (blocks > 0x7fffffff) return GWB_E_CAPACITY;
  const size_t smem = (size_t)tokens(a.chunk) * a.n * 2 * sizeof(float);
  rotary_kernel<T, VEC, INTERLEAVED><<<(unsigned)blocks, THREADS, smem, st>>>(a);
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
