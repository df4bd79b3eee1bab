// Gated feed-forward projections, bf16 or f16, forward and backward:
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u        [M, F]
//   dg = dh * u * act'(g),  du = dh * act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  db = column sums
//
// x [M, D], Wg and Wu [F, D]. Tensor cores bound all of it (4 M D F operations
// forward, 8 M D F backward) except at few rows, where reading the weights
// does. One persistent TMA-fed tcgen05 kernel serves the four products; the
// operands' majorness is a template argument, so no operand is transposed in
// memory: the backward products read W, x and dg / du as they lie, through
// MN-major shared-memory descriptors.
//
//   FORWARD  256 x (128 gate | 128 up) tile: both projections accumulate side
//            by side in TMEM, so activation and product happen in registers
//            and g and u never reach memory.
//   SAVE     FORWARD for a backward pass to come: also writes a = u act'(g) and
//            b = act(g), all that dg = dh a and du = dh b need of it.
//   DGATE    the same tile again for a caller that kept nothing; the epilogue
//            reads dh and writes dg and du (rounded to the operand type: they
//            are tensor-core operands next) and, for the bias gradients, the
//            column sums of each 32 rows before that rounding.
//   DX       dg Wg + du Wu as one chain of K = 2 F into one accumulator.
//   DW       dg^T x and du^T x, K = M.
//
// Accumulators, activations and column sums are f32. h and the bias gradients
// are rounded once; so are dx and dW, from products whose operands dg and du
// were rounded to 16 bits. a and b are kept with three bits or more beyond the
// operand type's, so that keeping them adds next to nothing to the rounding of
// dg and du: for bf16 as f16 times a power of two per row and 64 columns (4
// bytes a pair), for f16 as f32.
#include <cuda.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include "gwb.h"
#include "ptx.cuh"
#include "elem.cuh"

namespace gwb {
namespace gated {

enum Mode { FORWARD, SAVE, DGATE, DX, DW };

// A pair of CTAs shares a 256 x 256 tile: each holds its 128 rows of A, half
// of B's rows and its 128 rows of the accumulator, so a stage costs 32 KB a CTA
// where a CTA alone needs 48 KB for a 128 x 256 tile, and a third less is
// copied and read from shared memory per operation.
constexpr int BM = 128, BN = 256, BK = 64;      // BK elements = one 128-byte swizzle row
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN / 2 * BK * 2;   // of one CTA
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int MN_BOX = 64 * BK * 2;             // a 64 (MN) x 64 (K) box of an MN-major operand
constexpr int THREADS = 384, EPI0 = 4, EPI_WARPS = 8;
constexpr int PATCH = 32 * 128;                 // an epilogue warp's 32 rows of 128 bytes
// Stages, and the epilogue's patches where an epilogue has them (SAVE, and a
// product whose second template argument says so): what is left of the 256 KB
// is the L1 that direct stores go through.
template <int MODE, int ACT> constexpr bool patched() {
  return MODE == SAVE || ((MODE == DX || MODE == DW) && ACT);
}
template <int MODE, int ACT> constexpr int stages() { return patched<MODE, ACT>() ? 5 : 6; }
template <int MODE, int ACT> constexpr int smem_bytes() {
  return stages<MODE, ACT>() * STAGE_BYTES + (patched<MODE, ACT>() ? EPI_WARPS * PATCH : 0) + 1024 +
         256;
}
// Short items leave the epilogue no k-loop to hide behind: whole lines then.
// With 48 k-blocks or more the patches' shared memory costs more than it saves
// (dx and dw of 4608 x 3072 -> 12288: 1055 us with, 1037 without).
constexpr int PATCH_K = 48;
constexpr int NACC = 2, TMEM_COLS = NACC * BN;
// Tiles are walked in groups of eight row tiles: the 74 pairs at work then read
// about 8 row tiles and 9 column tiles, near the fewest operand bytes.
constexpr int GROUP = 8;

struct Args {
  const void* bg; const void* bu;     // FORWARD, DGATE: biases [F] or null
  const void* dh; int64_t dhs;        // DGATE: [M, F], row stride
  void* o0; void* o1;                 // h | dg, du | dx | dWg, dWu
  int M, D, F, act;
  void* kept; float* kept_scale;      // SAVE: a and b, planes [2][M][F], and their scales
  int tiles_m, tiles_n, half0, ntiles;
  // DX, DW with few tiles: each tile's K is split into `parts` of `part_k`
  // k-blocks, and part p's f32 tile goes to partial + p * part_stride. DGATE:
  // column sums [2][M / 32 rounded up][F], or null
  int parts, part_k; float* partial; int64_t part_stride;
};

// The type a and b are kept in, and whether each row's 64 columns have a scale.
template <typename T> struct Kept { using type = __half; static constexpr bool scaled = true; };
template <> struct Kept<__half> { using type = float; static constexpr bool scaled = false; };

// Infinities and NaN are kept as they are by any scale: finite values alone
// decide it.
__device__ __forceinline__ float finite_max(float m, float v) {
  const float a = fabsf(v);
  return a < INFINITY ? fmaxf(m, a) : m;
}

// 2^k that brings the largest magnitude into [2^13, 2^14) of f16; 1 where
// there is none.
__device__ __forceinline__ float kept_scale_of(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23);            // biased exponent, amax >= 0
  if (amax == 0.0f) return 1.0f;
  const int k = 13 + 127 - e;                                  // -114 .. 140
  return __uint_as_float((uint32_t)(min(max(k, -126), 126) + 127) << 23);
}

// ------------------------------------------------------------- activations
struct ActValue { float act, slope; };

// The normal distribution's upper tail at z >= 0, from e = exp(-z^2 / 2):
// e t P(t) with t = 1 / (1 + 0.3 z), the exponential taken out so that what is
// left (Mills' ratio over sqrt(2 pi)) is smooth and the error stays relative.
// P is the minimax polynomial of that for z up to 13.5, where the tail leaves
// f32's range, by Lawson's iteration in 64 bits: 1.3e-7 of the value. (1 + erf
// would cancel: off by 4 % at -5, by all of it from -5.6 on. erfcf holds, but
// cannot share the slope's exponential and is longer: run in turn with the erf
// form, forward calls of 4608 x 3072 -> 12288 and 1531 x 1416 -> 3880 took 9 to
// 15 % more with it; this form takes what the erf form does.)
__device__ __forceinline__ float normal_tail(float z, float e) {
  const float t = __fdividef(1.0f, fmaf(0.3f, z, 1.0f));
  float p = 0.03593185171484947f;
  p = fmaf(p, t, -0.15827642381191254f);
  p = fmaf(p, t, 0.20820726454257965f);
  p = fmaf(p, t, -0.055394381284713745f);
  p = fmaf(p, t, 0.12946945428848267f);
  p = fmaf(p, t, 0.09963742643594742f);
  p = fmaf(p, t, 0.12079837173223495f);
  p = fmaf(p, t, 0.11962638795375824f);
  return e * (t * p);
}

// act(g), and act'(g) when SLOPE. silu and the tanh form of GELU are
// g * sigmoid(t): 1 - sigmoid is taken without cancellation on either side.
// KIND is a template argument: a branch an element would keep the compiler
// from running the elements' exp and divide chains side by side.
template <int KIND, bool SLOPE>
__device__ __forceinline__ ActValue activation(float g) {
  ActValue r;
  r.slope = 0.0f;
  if constexpr (KIND == GWB_ACT_GELU) {
    const float e = __expf(-0.5f * g * g), q = normal_tail(fabsf(g), e);
    const float cdf = g < 0.0f ? q : 1.0f - q;
    r.act = g * cdf;
    if (SLOPE) r.slope = cdf + g * (0.39894228040143268f * e);
  } else {
    constexpr float c = 2.0f * 0.79788456080286536f, k = 0.044715f;   // 2 sqrt(2 / pi)
    const float t = KIND == GWB_ACT_SILU ? g : c * (g + k * g * g * g);
    const float e = __expf(-t);
    const float s = __fdividef(1.0f, 1.0f + e);
    r.act = g * s;
    if (SLOPE) {
      const float q = t >= 0.0f ? e * s : 1.0f - s;                   // 1 - s
      const float dt = KIND == GWB_ACT_SILU ? 1.0f : c * (1.0f + 3.0f * k * g * g);
      r.slope = s + g * (s * q) * dt;
    }
  }
  return r;
}

// ------------------------------------------------------------- descriptors
// MN-major operand, 128-byte swizzle: 64 MN elements are one 128-byte row,
// eight K rows a 1024-byte atom (SBO, to the next eight K), the next 64 MN
// elements `lbo` bytes on.
__device__ __forceinline__ uint64_t sdesc_mn128(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <typename T, bool A_MN, bool B_MN>
__host__ __device__ constexpr uint32_t idesc16() {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
         ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(2 * BM >> 4) << 24);
}

struct Tile { int m0, n0, half; };

template <int MODE>
__device__ __forceinline__ Tile tile_of(const Args& a, int t) {
  const int per = GROUP * a.tiles_n, first = t / per * GROUP;
  const int rows = min(a.tiles_m - first, GROUP), in = t % per;
  const int tm = first + in % rows, tn = in / rows;
  if (MODE == DW) {
    const int tf = (a.F + 2 * BM - 1) / (2 * BM);
    return {(tm % tf) * 2 * BM, tn * BN, a.half0 + tm / tf};
  }
  return {tm * 2 * BM, tn * (MODE == DX ? BN : BN / 2), 0};
}

// After a wait that ran out: a millisecond, in which any copy in flight lands
// before the CTA gives its shared memory back (the barrier that would tell is
// the other CTA's).
__device__ __forceinline__ void land_copies() {
  const long long t = clock64();
  while (clock64() - t < 2000000) { }
}

// Eight 16-bit elements <-> f32, two at a time
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  F2 v[4];
  unpack<T>(*reinterpret_cast<const uint4*>(p), v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 s = split(v[j]);
    f[2 * j] = s.x;
    f[2 * j + 1] = s.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 round8(const float (&f)[8]) {
  const F2 v[4] = {f2(f[0], f[1]), f2(f[2], f[3]), f2(f[4], f[5]), f2(f[6], f[7])};
  return repack<T>(v);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = round8<T>(f);
}

// The kept planes and the gradients leave by way of shared memory, 128 bytes of
// each of a warp's 32 rows at a time: a lane holds one row, and storing it
// directly touches 32 lines with every instruction (7473 x 304 -> 6984 f16 with
// its f32 planes: 325 us directly, 185 so; the gradients of 128 rows of 3072 ->
// 12288: 142 and 101). h is stored directly all the same: the detour cost it
// more than the lines did (41 against 47 us at 1531 x 1416 -> 3880). 16-byte
// pieces are swizzled by row, so both sides are free of bank conflicts.
__device__ __forceinline__ void patch_put(uint8_t* patch, int lane, int piece, uint4 v) {
  *reinterpret_cast<uint4*>(patch + lane * 128 + ((piece ^ (lane & 7)) << 4)) = v;
}
// rows and columns that exist; K elements of 16 or 32 bits
template <typename K>
__device__ __forceinline__ void patch_store(const uint8_t* patch, int lane, K* dst, int64_t ld,
                                            int rows, int cols) {
  constexpr int N = 16 / (int)sizeof(K);
  __syncwarp();
  const int piece = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    const uint4 v = *reinterpret_cast<const uint4*>(patch + r * 128 + ((piece ^ (r & 7)) << 4));
    if (r < rows && piece * N < cols) *reinterpret_cast<uint4*>(dst + r * ld + piece * N) = v;
  }
  __syncwarp();
}

// A warp's 32 rows (one a lane) of 32 columns, added up by column in 31
// shuffles: each step halves the columns a lane carries. Returns the sum of
// column `lane`; fixed order.
__device__ __forceinline__ float column_sums(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int half = 16; half; half /= 2) {
    const bool up = lane & half;
#pragma unroll
    for (int k = 0; k < half; ++k) {
      const float keep = up ? v[k + half] : v[k], give = up ? v[k] : v[k + half];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, give, half);
    }
  }
  return v[0];
}

template <int MODE, int ACT, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gated_kernel(const __grid_constant__ CUtensorMap tA0, const __grid_constant__ CUtensorMap tA1,
             const __grid_constant__ CUtensorMap tB0, const __grid_constant__ CUtensorMap tB1,
             const Args a) {
  constexpr bool A_MN = MODE == DW, B_MN = MODE == DX || MODE == DW, PROJ = !B_MN;
  constexpr bool PATCHED = patched<MODE, ACT>();
  constexpr int STAGES = stages<MODE, ACT>(), PATCHES = PATCHED ? EPI_WARPS * PATCH : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + PATCHES);   // the leader's count
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + NACC;                                       // the leader's count
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + NACC);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int kext = MODE == DX ? a.F : MODE == DW ? a.M : a.D;
  const int nk1 = (kext + BK - 1) / BK;               // k-blocks of one segment
  const int nk = MODE == DX ? 2 * nk1 : nk1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < NACC; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * EPI_WARPS);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tA0);
    tma_prefetch_desc(&tB0);
    if (MODE != DW) tma_prefetch_desc(&tB1);
    if (B_MN) tma_prefetch_desc(&tA1);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, TMEM_COLS);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // register hand-off as in the W8A8 kernel: 384 x 168 at launch, the first
  // warpgroup down to 40, the two epilogue warpgroups up to 232
  if (warp < EPI0) {
    regs_dec<40>();
    if (warp == 0 && lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < a.ntiles; tile += pairs) {
        const Tile t = tile_of<MODE>(a, PROJ ? tile : tile / a.parts);
        const int m0 = t.m0 + (int)rank * BM;         // this CTA's rows of A
        const int bn = (int)rank * (BN / 2);          // its part of B's rows
        const int k0b = PROJ ? 0 : tile % a.parts * a.part_k;
        const int k1b = PROJ ? nk : min(nk, k0b + a.part_k);
        for (int kb = k0b; kb < k1b; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, GWB_ERR_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * STAGE_BYTES;
          uint8_t* sb = sa + A_BYTES;
          // both CTAs' copies complete on the leader's barrier, which expects
          // them all; the other CTA's may come first, the phase still waits
          // for the leader's arrival
          const uint32_t bar = cluster_addr(&full[s], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * STAGE_BYTES);
          if constexpr (PROJ) {
            // the pair's 256 rows of B: the leader's are the gate's, the other's the up's
            tma_load_2d_pair(sa, &tA0, bar, kb * BK, m0);
            tma_load_2d_pair(sb, rank ? &tB1 : &tB0, bar, kb * BK, t.n0);
          } else if constexpr (MODE == DX) {
            const bool up = kb >= nk1;
            const int k0 = (kb - (up ? nk1 : 0)) * BK;
            tma_load_2d_pair(sa, up ? &tA1 : &tA0, bar, k0, m0);
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)
              tma_load_2d_pair(sb + j * MN_BOX, up ? &tB1 : &tB0, bar, t.n0 + bn + 64 * j, k0);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j)
              tma_load_2d_pair(sa + j * MN_BOX, t.half ? &tA1 : &tA0, bar, m0 + 64 * j, kb * BK);
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)
              tma_load_2d_pair(sb + j * MN_BOX, &tB0, bar, t.n0 + bn + 64 * j, kb * BK);
          }
        }
      }
      if (!ok) land_copies();
    } else if (warp == 1 && lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc16<T, A_MN, B_MN>();
      int it = 0, lt = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < a.ntiles; tile += pairs, ++lt) {
        const int b = lt & 1;
        if (!mbar_wait(&acc_empty[b], ((lt >> 1) & 1) ^ 1, GWB_ERR_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t d = tmem + b * BN;
        const int k0b = PROJ ? 0 : tile % a.parts * a.part_k;
        const int k1b = PROJ ? nk : min(nk, k0b + a.part_k);
        for (int kb = k0b; kb < k1b; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full[s], (it / STAGES) & 1, GWB_ERR_TIMEOUT_MMA)) { ok = false; break; }
          tc_fence_after();
          const uint32_t ab = smem_u32(smem + s * STAGE_BYTES), bb = ab + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_f16_pair(d, A_MN ? sdesc_mn128(ab + 2048 * k, MN_BOX) : sdesc_k128(ab + 32 * k),
                         B_MN ? sdesc_mn128(bb + 2048 * k, MN_BOX) : sdesc_k128(bb + 32 * k), idesc,
                         (kb > k0b || k > 0) ? 1u : 0u);
          mma_commit_pair(&empty[s]);
        }
        if (ok) mma_commit_pair(&acc_full[b]);
      }
    }
  } else {
    regs_inc<232>();
    const int q = warp & 3, side = (warp - EPI0) >> 2;
    uint8_t* patch = smem + STAGES * STAGE_BYTES + (warp - EPI0) * PATCH;
    int lt = 0;
    for (int tile = pair; tile < a.ntiles; tile += pairs, ++lt) {
      const Tile t = tile_of<MODE>(a, PROJ ? tile : tile / a.parts);
      const int b = lt & 1;
      if (!mbar_wait_warp(&acc_full[b], (lt >> 1) & 1, GWB_ERR_TIMEOUT_EPILOGUE)) break;
      tc_fence_after();
      uint32_t v[128];
      const uint32_t base = tmem + ((uint32_t)(32 * q) << 16) + b * BN;
      const int row0 = t.m0 + (int)rank * BM + 32 * q, row = row0 + lane;    // the lane's row
      if constexpr (PROJ) {
        // v[0..63] gate and v[64..127] up of columns n0 + 64 side ..
        tmem_ld32(base + 64 * side, v);
        tmem_ld32(base + 64 * side + 32, v + 32);
        tmem_ld32(base + 128 + 64 * side, v + 64);
        tmem_ld32(base + 160 + 64 * side, v + 96);
      } else {
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(base + 128 * side + c, v + c);
      }
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[b], 0));
      if constexpr (PROJ) {
        const int n0 = t.n0 + 64 * side, rows = a.M - row0, cols = a.F - n0;
        if (rows <= 0 || cols <= 0) continue;
        // SAVE's lanes store for each other, DGATE's add up columns together
        if (MODE == FORWARD && row >= a.M) continue;
        const bool live = row < a.M;
        float amax_a = 0.0f, amax_b = 0.0f;
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
          if (c >= cols) break;
          float g[8], u[8], p[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            g[j] = __uint_as_float(v[c + j]);
            u[j] = __uint_as_float(v[64 + c + j]);
          }
          if (a.bg) {
            load8(static_cast<const T*>(a.bg) + n0 + c, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += p[j];
          }
          if (a.bu) {
            load8(static_cast<const T*>(a.bu) + n0 + c, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] += p[j];
          }
          float o[8];
          if constexpr (MODE == FORWARD) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = activation<ACT, false>(g[j]).act * u[j];
          } else if constexpr (MODE == SAVE) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const ActValue f = activation<ACT, true>(g[j]);
              o[j] = f.act * u[j];
              const float fa = u[j] * f.slope;
              v[c + j] = __float_as_uint(fa);
              v[64 + c + j] = __float_as_uint(f.act);
              if (Kept<T>::scaled) {
                amax_a = finite_max(amax_a, fa);
                amax_b = finite_max(amax_b, f.act);
              }
            }
          } else {
            if (live) load8(static_cast<const T*>(a.dh) + (size_t)row * a.dhs + n0 + c, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const ActValue f = activation<ACT, true>(g[j]);
              o[j] = live ? p[j] * u[j] * f.slope : 0.0f;
              p[j] = live ? p[j] * f.act : 0.0f;
              v[c + j] = __float_as_uint(o[j]);
              v[64 + c + j] = __float_as_uint(p[j]);
            }
            if (live) store8(static_cast<T*>(a.o1) + (size_t)row * a.F + n0 + c, p);
          }
          if (live)
            store8(static_cast<T*>(a.o0) + (size_t)row * a.F + n0 + c, o);
        }
        if constexpr (MODE == SAVE) {
          using K = typename Kept<T>::type;
          // columns [0, 64) of v from `first` on, times s, to dst
          const auto put = [&](K* dst, int first, float s) {
            constexpr int N = 16 / (int)sizeof(K), WIDE = 8 * N;       // columns a patch holds
#pragma unroll
            for (int c0 = 0; c0 < 64; c0 += WIDE) {
#pragma unroll
              for (int c = 0; c < WIDE; c += N) {
                uint4 w;
                if constexpr (sizeof(K) == 2) {
                  float o[8];
#pragma unroll
                  for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(v[first + c0 + c + j]) * s;
                  w = round8<K>(o);
                } else {
                  w = make_uint4(v[first + c0 + c], v[first + c0 + c + 1], v[first + c0 + c + 2],
                                 v[first + c0 + c + 3]);
                }
                patch_put(patch, lane, c / N, w);
              }
              patch_store(patch, lane, dst + c0, a.F, rows, cols - c0);
            }
          };
          const float sa = Kept<T>::scaled ? kept_scale_of(amax_a) : 1.0f;
          const float sb = Kept<T>::scaled ? kept_scale_of(amax_b) : 1.0f;
          if (Kept<T>::scaled && live) {
            const int groups = (a.F + 63) / 64;
            a.kept_scale[(size_t)row * groups + n0 / 64] = sa;
            a.kept_scale[((size_t)a.M + row) * groups + n0 / 64] = sb;
          }
          K* ka = static_cast<K*>(a.kept) + (size_t)row0 * a.F + n0;
          put(ka, 0, sa);
          put(ka + (size_t)a.M * a.F, 64, sb);
        }
        if (MODE == DGATE && a.partial) {
          // column sums of the warp's 32 rows, before dg and du were rounded
          const int groups = (a.M + 31) / 32;
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            float s[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = __uint_as_float(v[c + j]);
            const float sum = column_sums(s);
            const int col = c % 64 + lane;
            if (col < cols)
              a.partial[((size_t)(c / 64) * groups + row0 / 32) * a.F + n0 + col] = sum;
          }
        }
      } else {
        const int total = MODE == DX ? a.M : a.F, n0 = t.n0 + 128 * side;
        const int rows = total - row0, cols = a.D - n0;
        if (rows <= 0 || cols <= 0) continue;
        if constexpr (!PATCHED) {
          if (row >= total) continue;
          T* dst = static_cast<T*>(t.half ? a.o1 : a.o0) + (size_t)row * a.D + n0;
#pragma unroll
          for (int c = 0; c < 128; c += 8) {
            if (c >= cols) break;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(v[c + j]);
            store8(dst + c, o);
          }
        } else if (a.parts > 1) {
          // this part's f32 tile; DW's two gradients are rows of one matrix
          float* dst = a.partial + (int64_t)(tile % a.parts) * a.part_stride +
                       ((int64_t)(t.half - a.half0) * a.F + row0) * a.D + n0;
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 32) {
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              patch_put(patch, lane, c / 4,
                        make_uint4(v[c0 + c], v[c0 + c + 1], v[c0 + c + 2], v[c0 + c + 3]));
            patch_store(patch, lane, dst + c0, a.D, rows, cols - c0);
          }
        } else {
          T* dst = static_cast<T*>(t.half ? a.o1 : a.o0) + (size_t)row0 * a.D + n0;
#pragma unroll
          for (int c0 = 0; c0 < 128; c0 += 64) {
#pragma unroll
            for (int c = 0; c < 64; c += 8) {
              float o[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(v[c0 + c + j]);
              patch_put(patch, lane, c / 8, round8<T>(o));
            }
            patch_store(patch, lane, dst + c0, a.D, rows, cols - c0);
          }
        }
      }
    }
  }
  // neither CTA ends while the other's MMAs, arrivals or copies may reach it
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) tmem_dealloc_pair(tmem, TMEM_COLS);
}

// ------------------------------------------------------------- few rows
// Up to 128 rows: reading the weights bounds it. The weights are the MMA's A
// operand and x its B operand with the rows rounded up to 16: features are then
// TMEM lanes, which all have work however few the rows are, and consecutive
// lanes store consecutive features. A tile has `w` features, a multiple of 8
// that gives the multiprocessors equal numbers of tiles (with 64 always, 192
// tiles of 12288 features took 39 us on 148 of them, with 88 and 140 tiles 31);
// lanes beyond w hold what is left in shared memory and store nothing.
//   FT 128  w over 64: gate and up rows are two A operands with an accumulator
//           each, side by side;
//   FT 64   up to 64: they are halves of one A operand, half the MMAs: lane
//           quarters 0 and 1 hold the gate and finish, 2 and 3 hold the up and
//           pass it through shared memory.
// Warps: 0 TMA, 1 MMA, 2-3 idle, 4-11 epilogue; each half of the eight takes 16
// rows of x in turn.
namespace few {
constexpr int MOST_ROWS = 128, MOST_STAGES = 11;
constexpr int THREADS = 384;
constexpr int SMEM_MOST = 200 * 1024;
constexpr int a_bytes(int ft) { return 2 * ft * BK * 2; }
constexpr int exchange(int ft, int n) { return ft == 64 ? n * 64 * 4 : 0; }
inline int stages_of(int ft, int n) {
  return std::min(MOST_STAGES, (SMEM_MOST - exchange(ft, n)) / (a_bytes(ft) + n * 128));
}
inline int smem_of(int ft, int n) {
  return stages_of(ft, n) * (a_bytes(ft) + n * 128) + exchange(ft, n) + 1024 + 512;
}
}  // namespace few

template <int ACT, typename T, int FT>
__global__ void __launch_bounds__(few::THREADS, 1)
few_rows_kernel(const __grid_constant__ CUtensorMap tX, const __grid_constant__ CUtensorMap tG,
                const __grid_constant__ CUtensorMap tU, const Args a, const int w, const int n,
                const int stages) {
  using namespace few;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  constexpr int A_BYTES = a_bytes(FT);
  const int stage_bytes = A_BYTES + n * 128;
  float* ups = reinterpret_cast<float*>(smem + stages * stage_bytes);        // [n][FT], FT 64
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes + exchange(FT, n));
  uint64_t* empty = full + MOST_STAGES;
  uint64_t* acc_full = empty + MOST_STAGES;
  uint64_t* acc_empty = acc_full + NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + NACC);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nk = (a.D + BK - 1) / BK;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < NACC; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 8); }
    fence_barrier_init();
    tma_prefetch_desc(&tX);
    tma_prefetch_desc(&tG);
    tma_prefetch_desc(&tU);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {
    int s = 0, phase = 1;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < a.ntiles; tile += gridDim.x)
      for (int kb = 0; kb < nk; ++kb) {
        if (!mbar_wait(&empty[s], phase, GWB_ERR_TIMEOUT_PRODUCER)) { ok = false; break; }
        uint8_t* sa = smem + s * stage_bytes;
        mbar_arrive_expect_tx(&full[s], (2 * w + n) * 128);
        tma_load_2d(sa, &tG, &full[s], kb * BK, tile * w);
        tma_load_2d(sa + A_BYTES / 2, &tU, &full[s], kb * BK, tile * w);
        tma_load_2d(sa + A_BYTES, &tX, &full[s], kb * BK, 0);
        if (++s == stages) { s = 0; phase ^= 1; }
      }
    if (!ok) land_copies();
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(n >> 3) << 17) |
                           (128u >> 4 << 24);
    int s = 0, phase = 0, lt = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < a.ntiles; tile += gridDim.x, ++lt) {
      const int b = lt & 1;
      if (!mbar_wait(&acc_empty[b], ((lt >> 1) & 1) ^ 1, GWB_ERR_TIMEOUT_MMA)) break;
      tc_fence_after();
      for (int kb = 0; kb < nk; ++kb) {
        if (!mbar_wait(&full[s], phase, GWB_ERR_TIMEOUT_MMA)) { ok = false; break; }
        tc_fence_after();
        const uint32_t ab = smem_u32(smem + s * stage_bytes), bb = ab + A_BYTES;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          const uint32_t more = (kb > 0 || k > 0) ? 1u : 0u;
          const uint64_t bd = sdesc_k128(bb + 32 * k);
          mma_f16(tmem + b * 256, sdesc_k128(ab + 32 * k), bd, idesc, more);
          if (FT == 128)
            mma_f16(tmem + b * 256 + 128, sdesc_k128(ab + A_BYTES / 2 + 32 * k), bd, idesc, more);
        }
        mma_commit(&empty[s]);
        if (++s == stages) { s = 0; phase ^= 1; }
      }
      if (ok) mma_commit(&acc_full[b]);
    }
  } else if (warp >= 4) {
    const int q = warp & 3, half = (warp - 4) >> 2;
    const int fl = 32 * (FT == 64 ? q & 1 : q) + lane;  // feature within the tile
    const int chunks = n / 16;
    int lt = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < a.ntiles; tile += gridDim.x, ++lt) {
      const int b = lt & 1;
      ok = ok && mbar_wait_warp(&acc_full[b], (lt >> 1) & 1, GWB_ERR_TIMEOUT_EPILOGUE);
      tc_fence_after();
      const int f = tile * w + fl;
      const bool mine = fl < w && f < a.F;
      const uint32_t base = tmem + ((uint32_t)(32 * q) << 16) + b * 256;
      uint32_t v[16], vu[16];
      if (FT == 64) {
        if (q >= 2)
          for (int c = half; c < chunks; c += 2) {
            tmem_ld16(base + 16 * c, v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) ups[(16 * c + j) * FT + fl] = __uint_as_float(v[j]);
          }
        asm volatile("bar.sync 1, 256;" ::: "memory");  // ups is written
      }
      if (FT == 128 || q < 2) {
        const float bg = a.bg && mine ? to_f32<T>(static_cast<const T*>(a.bg)[f]) : 0.0f;
        const float bu = a.bu && mine ? to_f32<T>(static_cast<const T*>(a.bu)[f]) : 0.0f;
        __syncwarp();
        for (int c = half; c < chunks; c += 2) {
          tmem_ld16(base + 16 * c, v);
          if (FT == 128) tmem_ld16(base + 128 + 16 * c, vu);
          tmem_wait_ld();
          float h[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float u = FT == 128 ? __uint_as_float(vu[j]) : ups[(16 * c + j) * FT + fl];
            h[j] = activation<ACT, false>(__uint_as_float(v[j]) + bg).act * (u + bu);
          }
          if (mine && ok)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (16 * c + j < a.M)
                static_cast<T*>(a.o0)[(size_t)(16 * c + j) * a.F + f] = from_f32<T>(h[j]);
          // lanes past w or F stored nothing: together again for the next
          // accumulator load and the barrier, which take whole warps
          __syncwarp();
        }
      }
      tc_fence_before();
      if (FT == 64) asm volatile("bar.sync 1, 256;" ::: "memory");   // ups is read
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[b]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------- dg, du and bias gradients
// From kept a and b: dg = dh a, du = dh b, 256 columns a CTA (eight a lane),
// its warps taking rows of one chunk in turn; with `partial`, the column sums
// [2][chunks][F] of the products before they are rounded, for
// column_join_kernel.
template <typename T>
__global__ void __launch_bounds__(256)
gradients_kernel(const T* __restrict__ dh, int64_t dhs, const void* __restrict__ kept,
                 const float* __restrict__ scale, T* __restrict__ dg, T* __restrict__ du, int M,
                 int F, int chunk_rows, float* __restrict__ partial) {
  using K = typename Kept<T>::type;
  __shared__ float acc[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x * 256 + lane * 8;
  const int r0 = blockIdx.y * chunk_rows, r1 = min(M, r0 + chunk_rows);
  const size_t plane = (size_t)M * F;
  const int groups = (F + 63) / 64;
  float sg[8] = {}, su[8] = {};
  if (c0 < F)
#pragma unroll 2
    for (int r = r0 + warp; r < r1; r += 8) {
      const size_t at = (size_t)r * F + c0;
      float g[8], u[8], d[8], ra = 1.0f, rb = 1.0f;
      load8(dh + (size_t)r * dhs + c0, d);
      const K* ka = static_cast<const K*>(kept) + at;
      if constexpr (Kept<T>::scaled) {
        load8(ka, g);
        load8(ka + plane, u);
        // the scales are powers of two: their reciprocals are exact
        ra = 1.0f / __ldg(scale + (size_t)r * groups + c0 / 64);
        rb = 1.0f / __ldg(scale + ((size_t)M + r) * groups + c0 / 64);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<float4*>(g + j) = *reinterpret_cast<const float4*>(ka + j);
          *reinterpret_cast<float4*>(u + j) = *reinterpret_cast<const float4*>(ka + plane + j);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] = d[j] * (g[j] * ra);
        u[j] = d[j] * (u[j] * rb);
      }
      store8(dg + at, g);
      store8(du + at, u);
      if (partial) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { sg[j] += g[j]; su[j] += u[j]; }
      }
    }
  if (!partial) return;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[warp][lane * 8 + j] = z ? su[j] : sg[j];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < F) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += acc[w][threadIdx.x];
      partial[((size_t)z * gridDim.y + blockIdx.y) * F + c] = t;
    }
    __syncthreads();
  }
}

// Sums a split product's parts in order: out0 [rows0][D], then out1.
template <typename T>
__global__ void __launch_bounds__(256)
parts_join_kernel(const float* __restrict__ partial, int parts, int64_t stride, int64_t n0,
                  int64_t n, T* __restrict__ out0, T* __restrict__ out1) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  float t[8] = {};
  for (int p = 0; p < parts; ++p) {
    const float4* src = reinterpret_cast<const float4*>(partial + p * stride + i);
    const float4 a = __ldcs(src), b = __ldcs(src + 1);
    t[0] += a.x; t[1] += a.y; t[2] += a.z; t[3] += a.w;
    t[4] += b.x; t[5] += b.y; t[6] += b.z; t[7] += b.w;
  }
  store8(i < n0 ? out0 + i : out1 + (i - n0), t);
}

// Bias gradients from column sums [2][chunks][F]: 32 columns a CTA, its eight
// warps taking chunks in turn, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256)
column_join_kernel(const float* __restrict__ partial, int chunks, int F, T* dbg, T* dbu) {
  __shared__ float acc[8][32];
  T* out = blockIdx.y ? dbu : dbg;
  if (out == nullptr) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  float t = 0.0f;
  if (c < F)
#pragma unroll 4
    for (int k = warp; k < chunks; k += 8) t += partial[((size_t)blockIdx.y * chunks + k) * F + c];
  acc[warp][lane] = t;
  __syncthreads();
  if (warp || c >= F) return;
  t = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += acc[w][lane];
  out[c] = from_f32<T>(t);
}

// ------------------------------------------------------------- host
// 2-D tensor of 16-bit elements, rows `ld` elements apart, box {64, by}
inline int tmap16(CUtensorMap* m, const void* base, bool bf16, int64_t cols, int64_t rows,
                  int64_t ld, int by) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return GWB_E_DRIVER;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)by}, es[2] = {1, 1};
  const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        2, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? GWB_SUCCESS : GWB_E_TMAP;
}

template <int MODE, int ACT, typename T>
int launch(const CUtensorMap& a0, const CUtensorMap& a1, const CUtensorMap& b0,
           const CUtensorMap& b1, Args a, cudaStream_t st) {
  auto kern = gated_kernel<MODE, ACT, T>;
  static std::atomic<uint64_t> ready{0};
  if (!allow_smem(reinterpret_cast<const void*>(kern), ready, smem_bytes<MODE, ACT>()))
    return GWB_E_LAUNCH;
  const int pairs = sm_count() / 2;
  kern<<<2 * (a.ntiles < pairs ? a.ntiles : pairs), THREADS, smem_bytes<MODE, ACT>(), st>>>(a0, a1, b0,
                                                                                   b1, a);
  return launch_status();
}

// Tensor maps are encoded by the driver, which wants a current context: a
// thread that has made no runtime call yet (autograd's) has none until its
// device is set.
inline int bind_context() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return GWB_E_LAUNCH;
  return GWB_SUCCESS;
}

inline int cdiv(int a, int b) { return (a + b - 1) / b; }

// Kept planes: a and b [2][M][F], 16-byte aligned end to end (F % 8 == 0),
// then (scaled) the scales f32 [2][M][F / 64 rounded up].
template <typename T> int64_t kept_bytes(int64_t M, int64_t F) {
  return 2 * M * F * (int64_t)sizeof(typename Kept<T>::type) +
         (Kept<T>::scaled ? 2 * M * ((F + 63) / 64) * 4 : 0);
}
template <typename T> float* kept_scales(void* kept, int64_t M, int64_t F) {
  return reinterpret_cast<float*>(static_cast<uint8_t*>(kept) +
                                  2 * M * F * sizeof(typename Kept<T>::type));
}

// The few-rows forward call
template <typename T>
int few_rows(const void* x, int64_t xs, const void* wg, const void* wu, Args a, cudaStream_t st) {
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  const int n = cdiv(a.M, 16) * 16;
  if (int rc = bind_context()) return rc;
  CUtensorMap tx, tg, tu;
  const int sms = sm_count(), waves = cdiv(a.F, 128 * sms);
  const int w = std::max(8, cdiv(cdiv(a.F, sms * waves), 8) * 8), ft = w > 64 ? 128 : 64;
  if (int rc = tmap16(&tx, x, bf, a.D, a.M, xs, n)) return rc;
  if (int rc = tmap16(&tg, wg, bf, a.D, a.F, a.D, w)) return rc;
  if (int rc = tmap16(&tu, wu, bf, a.D, a.F, a.D, w)) return rc;
  a.ntiles = cdiv(a.F, w);
  const auto wide = [&](auto act, auto feats) {
    auto kern = few_rows_kernel<decltype(act)::value, T, decltype(feats)::value>;
    static std::atomic<uint64_t> ready{0};
    if (!allow_smem(reinterpret_cast<const void*>(kern), ready, few::SMEM_MOST + 1024 + 512))
      return (int)GWB_E_LAUNCH;
    kern<<<std::min(a.ntiles, sms), few::THREADS, few::smem_of(ft, n), st>>>(
        tx, tg, tu, a, w, n, few::stages_of(ft, n));
    return launch_status();
  };
  const auto go = [&](auto act) {
    return ft == 128 ? wide(act, std::integral_constant<int, 128>{})
                     : wide(act, std::integral_constant<int, 64>{});
  };
  if (a.act == GWB_ACT_SILU) return go(std::integral_constant<int, GWB_ACT_SILU>{});
  if (a.act == GWB_ACT_GELU) return go(std::integral_constant<int, GWB_ACT_GELU>{});
  return go(std::integral_constant<int, GWB_ACT_GELU_TANH>{});
}

template <typename T>
int projections(Mode mode, const void* x, int64_t xs, const void* wg, const void* wu, Args a,
                cudaStream_t st) {
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  if (mode == FORWARD && a.M <= few::MOST_ROWS) return few_rows<T>(x, xs, wg, wu, a, st);
  if (int rc = bind_context()) return rc;
  CUtensorMap tx, tg, tu;
  if (int rc = tmap16(&tx, x, bf, a.D, a.M, xs, BM)) return rc;
  if (int rc = tmap16(&tg, wg, bf, a.D, a.F, a.D, BN / 2)) return rc;
  if (int rc = tmap16(&tu, wu, bf, a.D, a.F, a.D, BN / 2)) return rc;
  a.tiles_m = cdiv(a.M, 2 * BM);
  a.tiles_n = cdiv(a.F, BN / 2);
  a.ntiles = a.tiles_m * a.tiles_n;
  const auto go = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (mode == DGATE) return launch<DGATE, ACT, T>(tx, tx, tg, tu, a, st);
    if (mode == SAVE) return launch<SAVE, ACT, T>(tx, tx, tg, tu, a, st);
    return launch<FORWARD, ACT, T>(tx, tx, tg, tu, a, st);
  };
  if (a.act == GWB_ACT_SILU) return go(std::integral_constant<int, GWB_ACT_SILU>{});
  if (a.act == GWB_ACT_GELU) return go(std::integral_constant<int, GWB_ACT_GELU>{});
  return go(std::integral_constant<int, GWB_ACT_GELU_TANH>{});
}

// Chunks of rows of gradients_kernel: about eight CTAs a multiprocessor, at
// least 32 rows each.
inline int bias_chunks(int M, int F) {
  const int tiles = cdiv(F, 256), want = cdiv(148 * 8, tiles), most = cdiv(M, 32);
  return want < most ? (want > 0 ? want : 1) : (most > 0 ? most : 1);
}

// How a product of `tiles` tiles of nk k-blocks is split along K: the parts (at
// most 16, of eight k-blocks at least) for which the pairs of multiprocessors
// finish first, counting 512 cycles a k-block, 3000 an item, and the parts'
// f32 values written and read at 3400 bytes a cycle. One part wherever there
// are tiles enough; at 1000 x 256 x 8192, dx has 4 tiles of 256 k-blocks and 74
// pairs to work on them: 99 us in one part, 20 in 16.
struct Split { int parts, part_k; };
inline Split split_of(int64_t tiles, int nk, int64_t elements) {
  const int64_t pairs = sm_count() / 2;
  Split best{1, nk};
  int64_t cost = -1;
  for (int parts = 1; parts <= 16 && (parts == 1 || nk / parts >= 8); ++parts) {
    const int per = cdiv(nk, parts);
    if (cdiv(nk, per) != parts) continue;
    int64_t c = (tiles * parts + pairs - 1) / pairs * (per * 512 + 3000);
    if (parts > 1) c += elements * 8 * parts / 3400 + 6000;
    if (cost < 0 || c < cost) { cost = c; best = {parts, per}; }
  }
  return best;
}
inline Split split_dx(int M, int D, int F) {
  return split_of((int64_t)cdiv(M, 2 * BM) * cdiv(D, BN), 2 * cdiv(F, BK), (int64_t)M * D);
}
inline Split split_dw(int M, int D, int F, int halves) {
  return split_of((int64_t)halves * cdiv(F, 2 * BM) * cdiv(D, BN), cdiv(M, BK),
                  (int64_t)halves * F * D);
}
inline int64_t partial_bytes(const Split& s, int64_t elements) {
  return s.parts > 1 ? s.parts * elements * 4 : 0;
}

// Column sums of the bias gradients: of each 32 rows of the DGATE tiles, or
// (a and b kept) of gradients_kernel's chunks, which are no more.
inline int bias_groups(int M) { return cdiv(M, 32); }
inline int64_t bias_bytes(int M, int F) {
  return ((int64_t)2 * bias_groups(M) * F * 4 + 255) / 256 * 256;
}

template <typename T>
int join(const Args& a, int64_t n0, int64_t n, cudaStream_t st) {
  parts_join_kernel<T><<<(unsigned)((n / 8 + 255) / 256), 256, 0, st>>>(
      a.partial, a.parts, a.part_stride, n0, n, static_cast<T*>(a.o0), static_cast<T*>(a.o1));
  return launch_status();
}

template <typename T>
int backward(const GatedBackward& w, cudaStream_t st) {
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  const int M = w.M, D = w.D, F = w.F;
  uint8_t* p = static_cast<uint8_t*>(w.work);
  const size_t plane = ((size_t)M * F * 2 + 255) / 256 * 256;
  void* dg = p;
  void* du = p + plane;
  float* partial = reinterpret_cast<float*>(p + 2 * plane);
  float* parts = reinterpret_cast<float*>(p + 2 * plane + bias_bytes(M, F));
  Args a{};
  a.bg = w.bg; a.bu = w.bu; a.dh = w.dh; a.dhs = w.dhs; a.o0 = dg; a.o1 = du;
  a.M = M; a.D = D; a.F = F; a.act = w.act;
  const int chunks = w.kept ? bias_chunks(M, F) : bias_groups(M);
  const bool bias = w.dbg || w.dbu;
  if (int rc = bind_context()) return rc;
  if (w.kept) {
    gradients_kernel<T><<<dim3(cdiv(F, 256), chunks), 256, 0, st>>>(
        static_cast<const T*>(w.dh), w.dhs, w.kept, kept_scales<T>(w.kept, M, F),
        static_cast<T*>(dg), static_cast<T*>(du), M, F, cdiv(M, chunks), bias ? partial : nullptr);
    if (int rc = launch_status()) return rc;
  } else {
    Args d = a;
    d.partial = bias ? partial : nullptr;
    if (int rc = projections<T>(DGATE, w.x, w.xs, w.wg, w.wu, d, st)) return rc;
  }
  if (w.dx) {
    CUtensorMap ag, au, bgm, bum;
    if (int rc = tmap16(&ag, dg, bf, F, M, F, BM)) return rc;
    if (int rc = tmap16(&au, du, bf, F, M, F, BM)) return rc;
    if (int rc = tmap16(&bgm, w.wg, bf, D, F, D, BK)) return rc;
    if (int rc = tmap16(&bum, w.wu, bf, D, F, D, BK)) return rc;
    Args c = a;
    c.o0 = w.dx;
    c.tiles_m = cdiv(M, 2 * BM);
    c.tiles_n = cdiv(D, BN);
    const Split sp = split_dx(M, D, F);
    c.parts = sp.parts; c.part_k = sp.part_k;
    c.partial = parts; c.part_stride = (int64_t)M * D;
    c.ntiles = c.tiles_m * c.tiles_n * c.parts;
    const bool patch = c.parts > 1 || c.part_k < PATCH_K;
    if (int rc = patch ? launch<DX, 1, T>(ag, au, bgm, bum, c, st)
                       : launch<DX, 0, T>(ag, au, bgm, bum, c, st))
      return rc;
    if (c.parts > 1)
      if (int rc = join<T>(c, c.part_stride, c.part_stride, st)) return rc;
  }
  if (w.dwg || w.dwu) {
    CUtensorMap ag, au, bx;
    if (int rc = tmap16(&ag, dg, bf, F, M, F, BK)) return rc;
    if (int rc = tmap16(&au, du, bf, F, M, F, BK)) return rc;
    if (int rc = tmap16(&bx, w.x, bf, D, M, w.xs, BK)) return rc;
    Args c = a;
    c.o0 = w.dwg;
    c.o1 = w.dwu;
    c.half0 = w.dwg ? 0 : 1;
    c.tiles_m = cdiv(F, 2 * BM) * (w.dwg && w.dwu ? 2 : 1);
    c.tiles_n = cdiv(D, BN);
    const int halves = w.dwg && w.dwu ? 2 : 1;
    const Split sp = split_dw(M, D, F, halves);
    c.parts = sp.parts; c.part_k = sp.part_k;
    c.partial = parts; c.part_stride = (int64_t)halves * F * D;
    c.ntiles = c.tiles_m * c.tiles_n * c.parts;
    const bool patch = c.parts > 1 || c.part_k < PATCH_K;
    if (int rc = patch ? launch<DW, 1, T>(ag, au, bx, bx, c, st)
                       : launch<DW, 0, T>(ag, au, bx, bx, c, st))
      return rc;
    if (c.parts > 1)
      if (int rc = join<T>(c, w.dwg ? (int64_t)F * D : 0, c.part_stride, st)) return rc;
  }
  if (bias) {
    column_join_kernel<T><<<dim3(cdiv(F, 32), 2), 256, 0, st>>>(
        partial, chunks, F, static_cast<T*>(w.dbg), static_cast<T*>(w.dbu));
    return launch_status();
  }
  return GWB_SUCCESS;
}

}  // namespace gated

int64_t gated_backward_work(int M, int D, int F) {
  using namespace gated;
  const int64_t plane = ((int64_t)M * F * 2 + 255) / 256 * 256;
  const int64_t dx = partial_bytes(split_dx(M, D, F), (int64_t)M * D);
  const int64_t dw2 = partial_bytes(split_dw(M, D, F, 2), (int64_t)2 * F * D);
  const int64_t dw1 = partial_bytes(split_dw(M, D, F, 1), (int64_t)F * D);
  return 2 * plane + bias_bytes(M, F) + std::max(dx, std::max(dw1, dw2));
}

int64_t gated_kept_bytes(int64_t M, int64_t F, int dtype) {
  return dtype == GWB_BF16 ? gated::kept_bytes<__nv_bfloat16>(M, F) : gated::kept_bytes<__half>(M, F);
}

template <typename T>
static int gated_forward(const void* x, int64_t xs, const void* wg, const void* wu, gated::Args a,
                         void* kept, cudaStream_t st) {
  a.kept = kept;
  if (kept) a.kept_scale = gated::kept_scales<T>(kept, a.M, a.F);
  return gated::projections<T>(kept ? gated::SAVE : gated::FORWARD, x, xs, wg, wu, a, st);
}

int launch_gated_forward(const void* x, int64_t xs, const void* wg, const void* wu, const void* bg,
                         const void* bu, int M, int D, int F, int act, int dtype, void* h,
                         void* kept, cudaStream_t st) {
  gated::Args a{};
  a.bg = bg; a.bu = bu; a.o0 = h; a.M = M; a.D = D; a.F = F; a.act = act;
  return dtype == GWB_BF16 ? gated_forward<__nv_bfloat16>(x, xs, wg, wu, a, kept, st)
                           : gated_forward<__half>(x, xs, wg, wu, a, kept, st);
}

int launch_gated_backward(const GatedBackward& w, int dtype, cudaStream_t st) {
  return dtype == GWB_BF16 ? gated::backward<__nv_bfloat16>(w, st)
                           : gated::backward<__half>(w, st);
}

}  // namespace gwb
