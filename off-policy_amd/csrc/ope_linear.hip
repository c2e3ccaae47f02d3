// Linear layer with bias, activation and residual in its epilogue, and its gradients (ope_linear, ope_linear_backward; ope.h).
//
// One product kernel for all four operand types: C[m][n] = sum_k A[m][k] B[n][k]. In the forward product the contraction runs along memory in both operands;
// in the gradients' (dz w, dz^T x) over the rows of one or both, which are turned in registers (Loader). It counts in BYTES of k: a lane takes 16 bytes of one row -- 4 float32, 8 bfloat16 / float16 or 16 e4m3 values -- and feeds them to the matrix
// instructions of that type (the same permutation of k on both operands, so any grouping is right). The weight row is the instruction's A
// operand: a lane then holds 4 consecutive columns of one output row, and the epilogue reads and writes packs.
#include <type_traits>

#include "ope_elem.h"

namespace ope {

struct e4m3_t { uint8_t v; };
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_loose __attribute__((aligned(1)));
typedef uint32_t u32_loose __attribute__((aligned(2)));

template <typename T>
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 product<float>(u32x4 a, u32x4 b, f32x4 c) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int r = 0; r < 4; ++r) c = mfma16(x[r], y[r], c);
  return c;
}
template <>
__device__ __forceinline__ f32x4 product<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 product<f16_t>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 16 e4m3 values as two packs of float16 (exact: every e4m3 value, subnormals and NaN among them, is one).
__device__ __forceinline__ void widen_e4m3(u32x4 a, f16x8* out) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a[i], 1.f, false));
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a[i], 1.f, true));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      out[i / 2][4 * (i % 2) + e] = lo[e];
      out[i / 2][4 * (i % 2) + 2 + e] = hi[e];
    }
  }
}
// The matrix instructions on 8-bit operands align their products before they add them and keep about 18 bits (measured: 1.4e-5 of the result's
// norm at k = 128, against 1.8e-8 on float16 and bfloat16), so the operands are widened in registers: sums in 32 bits at the same rate as the
// 16 x 16 x 32 form on 8 bits, and the memory traffic stays that of 8 bits.
template <>
__device__ __forceinline__ f32x4 product<e4m3_t>(u32x4 a, u32x4 b, f32x4 c) {
  f16x8 x[2], y[2];
  widen_e4m3(a, x);
  widen_e4m3(b, y);
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[0], y[0], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(x[1], y[1], c, 0, 0, 0);
}

__device__ __forceinline__ int ope_cdiv_dev4(int n) { return (n + 3) / 4; }
__device__ __forceinline__ int ope_cdiv_dev64(int n) { return (n + 63) / 64; }

// 16 bytes of a row, from byte k of `len`; bytes past the row's end are zero (and not read).
__device__ __forceinline__ u32x4 row16(const uint8_t* row, int64_t k, int64_t len, int elem) {
  if (k + 16 <= len) return *reinterpret_cast<const u32x4_loose*>(row + k);
  u32x4 v = {0, 0, 0, 0};
  if (elem == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + 4 * e < len) v[e] = *reinterpret_cast<const uint32_t*>(row + k + 4 * e);
  } else if (elem == 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + 2 * e < len) v[e / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(row + k + 2 * e) << (16 * (e % 2));
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (k + e < len) v[e / 4] |= (uint32_t)row[k + e] << (8 * (e % 4));
  }
  return v;
}
// The last step of float32 rows that end inside it, for the forward product: piece g of a half (16 values) takes k = 4 r + g, so that the matrix
// instructions add what is left in ascending order of k. Whole steps go by k = 4 g + r (16 bytes a lane); with both, z was to the bit what the library's
// float32 product gives on the rows compared that neither splits (252, 480, 672 and 2048 wide), and a relu's gate falls on the same side where z is within
// rounding of 0 (one that falls otherwise moves a row of dx and a row of dw). The loads are single ones there anyway.
__device__ __forceinline__ u32x4 last16(const uint8_t* row, int64_t half, int g, int64_t len) {
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t k = half + 16 * r + 4 * g;
    if (k < len) v[r] = *reinterpret_cast<const uint32_t*>(row + k);
  }
  return v;
}

// e^-z and s = 1 / (1 + e^-z) by the hardware's 2^x and 1/x, each within one step of float32: with expf and a division the epilogue of a 4096 x 4096
// output took 20 us more than without an activation. e^-z past the range is infinite, its reciprocal 0. The rounding of the exponent z log2 e alone moves e^-z
// by |z| 2^-24 of itself: nothing beside the rounding of a 16-bit result, up to 64 half steps of a float32 one. WIDE (float32 results) makes that good
// with the exponent's low part, where e^-z is in range.
template <bool WIDE>
__device__ __forceinline__ float sigmoid(float z, float* ez = nullptr) {
  constexpr float L = -1.44269504088896341f, Llo = (float)(-1.44269504088896341 - (double)L);
  const float t = z * L;
  float e = __builtin_amdgcn_exp2f(t);
  if (WIDE) {
    const float low = fmaf(z, Llo, fmaf(z, L, -t)) * 0.69314718055994531f;
    e = fabsf(z) < 88.f ? fmaf(e, low, e) : e;
  }
  if (ez) *ez = e;
  return __builtin_amdgcn_rcpf(1.f + e);
}
template <bool WIDE>
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case OPE_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case OPE_ACT_TANH: return tanhf(z);
    case OPE_ACT_SILU: return z * sigmoid<WIDE>(z);
    case OPE_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  }
  return z;
}
template <bool WIDE>
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case OPE_ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case OPE_ACT_TANH: { const float t = tanhf(z); return 1.f - t * t; }
    case OPE_ACT_SILU: {
      float e;
      const float s = sigmoid<WIDE>(z, &e);
      return s * (1.f + z * (WIDE && z > 0.f ? e * s : 1.f - s));       // (1 - s = e^-z s, which keeps its bits where s is next to 1)
    }
    case OPE_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  }
  return 1.f;
}
template <bool WIDE>
__device__ __forceinline__ f32x4 act4(f32x4 z, int act) {          // one branch for the four
  const auto each = [&](auto a) { return f32x4{act_of<WIDE>(z[0], a()), act_of<WIDE>(z[1], a()), act_of<WIDE>(z[2], a()), act_of<WIDE>(z[3], a())}; };
  switch (act) {
    case OPE_ACT_RELU: return each(std::integral_constant<int, OPE_ACT_RELU>{});
    case OPE_ACT_TANH: return each(std::integral_constant<int, OPE_ACT_TANH>{});
    case OPE_ACT_SILU: return each(std::integral_constant<int, OPE_ACT_SILU>{});
    case OPE_ACT_GELU: return each(std::integral_constant<int, OPE_ACT_GELU>{});
  }
  return z;
}

struct Epilogue {
  const float *x_scale, *w_scale;
  const void *bias, *residual;
  void* y;
  float* z;
  int64_t residual_stride;
  int64_t M;
  int N, act;
};
// columns n .. n+3 of output row m
template <typename O>
__device__ __forceinline__ void finish4(const Epilogue& e, f32x4 acc, int64_t m, int n) {
  if (m >= e.M || n >= e.N) return;
  const int live = min(4, e.N - n);
  f32x4 z = acc, res = {0.f, 0.f, 0.f, 0.f}, b = res, sw = {1.f, 1.f, 1.f, 1.f};
  if (live == 4) {
    if (e.w_scale) sw = load_pack<float, 4>(e.w_scale + n);
    if (e.bias) b = load_pack<O, 4>((const O*)e.bias + n);
    if (e.residual) res = load_pack<O, 4>((const O*)e.residual + m * e.residual_stride + n);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < live) {
        if (e.w_scale) sw[r] = e.w_scale[n + r];
        if (e.bias) b[r] = (float)((const O*)e.bias)[n + r];
        if (e.residual) res[r] = (float)((const O*)e.residual)[m * e.residual_stride + n + r];
      }
  }
  if (e.x_scale) z *= sw * e.x_scale[m];
  z += b;
  const f32x4 y = act4<sizeof(O) == 4>(z, e.act) + res;
  const int64_t at = m * e.N + n;
  if (live == 4) {
    store_pack<O, 4>((O*)e.y + at, y);
    if (e.z) store_pack<float, 4>(e.z + at, z);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < live) {
        ((O*)e.y)[at + r] = (O)y[r];
        if (e.z) e.z[at + r] = z[r];
      }
  }
}

struct Operand {
  const uint8_t* p;
  int64_t rows, stride;            // output rows this operand has; bytes from one row of memory to the next
};

// One operand's tile of R output rows and 128 bytes of the contraction, on its way from memory through registers to LDS (TH threads). LDS rows are 8
// pieces of 16 bytes, stored at piece ^ spread(row): 8 rows behind each other, and 8 rows 4 apart, then lie in 8 different places, so neither the
// 16-row fragment reads nor the stores of turned columns collide in the banks.
//   ALONG: the contraction runs along memory; a thread moves whole pieces. LAST: by last16 in the step that the rows end in.
//   else: it runs over the rows of memory (gradients: dz^T x, dz w); a thread takes C neighbouring columns of as many rows as a piece has elements and
//   turns them in registers, so nothing is transposed in memory. 16 neighbouring lanes read one run of a row, the four rows of lanes behind them
//   other pieces: their LDS stores then spread over all eight places.
__device__ __forceinline__ int spread(int row) { return (row ^ (row >> 2)) & 7; }
template <typename T, int R, int TH, bool ALONG, bool LAST>
struct Loader {
  static constexpr int N = R * 8 / TH;                                    // pieces a thread moves
  static constexpr int E = 16 / (int)sizeof(T), C = N < 4 ? N : 4;        // elements of a piece; columns a thread takes
  static constexpr int W = C * (int)sizeof(T) / 4;                        // 4-byte words of a row it takes
  static_assert(R * 8 % TH == 0 && N % C == 0 && (ALONG || W >= 1), "tile and workgroup");
  u32x4 r[N];
  // Step s of the contraction. WHOLE: all of its 128 bytes are there, so no row of memory needs a check. Output rows past the last one read the last
  // one's bytes again; what they make is not stored.
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(const Operand& o, int64_t first, int64_t klen, int s) {
    if constexpr (ALONG) {
      const int row = threadIdx.x >> 3;
      const int64_t k = (int64_t)s * 128 + (threadIdx.x & 7) * 16;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint8_t* p = o.p + min(first + row + TH / 8 * i, o.rows - 1) * o.stride;
        if (WHOLE) r[i] = *reinterpret_cast<const u32x4_loose*>(p + k);
        else if (LAST) r[i] = last16(p, k & ~(int64_t)63, threadIdx.x & 3, klen);
        else r[i] = row16(p, k, klen, (int)sizeof(T));
      }
    } else {
      typedef uint32_t words __attribute__((ext_vector_type(W)));
      typedef words words_loose __attribute__((aligned(2)));
      const int64_t len = klen / (int)sizeof(T);                          // rows of memory
#pragma unroll
      for (int i = 0; i < N / C; ++i) {
        const int x = threadIdx.x + TH * i, col = ((x & 15) + 16 * (x >> 7)) * C, piece = (x >> 4) & 7;
        const int64_t n = first + col, m0 = (int64_t)s * (128 / (int)sizeof(T)) + piece * E;
        const int here = (int)(n < o.rows ? min(o.rows - n, (int64_t)C) : 0);                        // columns of the C that exist
        const uint8_t* p = o.p + m0 * o.stride + (here ? n : 0) * (int)sizeof(T);
        uint32_t w[E][W];
        if (WHOLE && (here == C || (here == 0 && o.rows >= C))) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const words v = *reinterpret_cast<const words_loose*>(p + e * o.stride);
#pragma unroll
            for (int c = 0; c < W; ++c) w[e][c] = ((const uint32_t*)&v)[c];
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) {
#pragma unroll
            for (int c = 0; c < W; ++c) w[e][c] = 0;
            if (m0 + e < len)
#pragma unroll
              for (int c = 0; c < C; ++c)
                if (c < here) {
                  if (sizeof(T) == 4) w[e][c % W] = *reinterpret_cast<const uint32_t*>(p + e * o.stride + 4 * c);
                  else w[e][c / 2 % W] |= (uint32_t) * reinterpret_cast<const uint16_t*>(p + e * o.stride + 2 * c) << (16 * (c % 2));
                }
          }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 4) r[C * i + c][e] = w[e][c];
            else r[C * i + c][e] = __builtin_amdgcn_perm(w[2 * e + 1][c / 2], w[2 * e][c / 2], c % 2 ? 0x07060302 : 0x05040100);
          }
      }
    }
  }
  __device__ __forceinline__ void store(u32x4 (*lds)[8]) const {
    if constexpr (ALONG) {
      const int row = threadIdx.x >> 3, piece = threadIdx.x & 7;
#pragma unroll
      for (int i = 0; i < N; ++i) lds[row + TH / 8 * i][piece ^ spread(row + TH / 8 * i)] = r[i];
    } else {
#pragma unroll
      for (int i = 0; i < N / C; ++i) {
        const int x = threadIdx.x + TH * i, col = ((x & 15) + 16 * (x >> 7)) * C, piece = (x >> 4) & 7;
#pragma unroll
        for (int c = 0; c < C; ++c) lds[col + c][piece ^ spread(col + c)] = r[C * i + c];
      }
    }
  }
};

// The tile kernel: BM x BN outputs a workgroup of WM x WN waves, 128 bytes of k a step, two LDS buffers: the next step's rows travel from
// memory to registers while this step's are multiplied (two steps ahead took the second workgroup off the CU: 135 and 206 us instead of 96 and 103 in
// the two products of 4096 x 2048 x 4096). gridDim.y > 1: split of k; part [split][M][N] takes the sums and linear_join finishes.
// Workgroups run over the XCDs in turn; each XCD gets one run of tiles, four rows of tiles high, so that its L2 sees few panels.
template <typename T, typename O, int BM, int BN, int WM, int WN, bool AA, bool BA>
__global__ __launch_bounds__(64 * WM * WN) void linear_tile(Operand A, Operand B, int64_t klen, int tiles_m, int tiles_n, int steps_per, Epilogue e,
                                                            float* __restrict__ part) {
  constexpr int TH = 64 * WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
  __shared__ u32x4 lds[2 * (BM + BN) * 8];
  u32x4(*As)[BM][8] = reinterpret_cast<u32x4(*)[BM][8]>(lds);
  u32x4(*Bs)[BN][8] = reinterpret_cast<u32x4(*)[BN][8]>(lds + 2 * BM * 8);
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const unsigned total = gridDim.x, per = total / 8, more = total % 8, xcd = blockIdx.x % 8;
  const unsigned tile = xcd * per + min(xcd, more) + blockIdx.x / 8;
  const unsigned band = tile / (4u * tiles_n), high = min(4u, tiles_m - 4 * band), in = tile - band * 4u * tiles_n;
  const int64_t m0 = (int64_t)(4 * band + in % high) * BM, n0 = (int64_t)(in / high) * BN;
  const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);
  const int steps = (int)((klen + 127) / 128), first = blockIdx.y * steps_per, last = min(first + steps_per, steps);
  constexpr bool kLast = AA && BA && sizeof(T) == 4;   // (both operands alike)
  Loader<T, BM, TH, AA, kLast> la;
  Loader<T, BN, TH, BA, kLast> lb;
  const int whole = (int)(klen / 128);                 // steps without an end in them
  auto fetch = [&](int s) {
    if (s < whole) {
      la.template fetch<true>(A, m0, klen, s);
      lb.template fetch<true>(B, n0, klen, s);
    } else {
      la.template fetch<false>(A, m0, klen, s);
      lb.template fetch<false>(B, n0, klen, s);
    }
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (first < last) fetch(first);
  for (int s = first; s < last; ++s) {
    const int buf = (s - first) & 1;
    la.store(As[buf]);
    lb.store(Bs[buf]);
    lds_barrier();
    if (s + 1 < last) fetch(s + 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 fa[MT], fb[NT];
#pragma unroll
      for (int b = 0; b < NT; ++b) fb[b] = Bs[buf][wn + 16 * b + j][(4 * h + g) ^ spread(wn + 16 * b + j)];
#pragma unroll
      for (int a = 0; a < MT; ++a) fa[a] = As[buf][wm + 16 * a + j][(4 * h + g) ^ spread(wm + 16 * a + j)];
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = product<T>(fb[b], fa[a], acc[a][b]);
    }
  }
  // The epilogue walks 16 rows at a time through the wave's own part of LDS: packs of whole rows leave (as the accumulators lie, a store would touch 16
  // rows), and the code for a pack stands once for each 16 rows.
  __syncthreads();
  constexpr int CW = 16 * NT;                          // columns of a wave
  float* mine = reinterpret_cast<float*>(lds) + w * 16 * (CW + 4);
#pragma unroll
  for (int a = 0; a < MT; ++a) {
#pragma unroll
    for (int b = 0; b < NT; ++b) *reinterpret_cast<f32x4*>(&mine[j * (CW + 4) + 16 * b + 4 * g]) = acc[a][b];
#pragma unroll 1
    for (int x = threadIdx.x & 63; x < 16 * CW / 4; x += 64) {
      const int r = x / (CW / 4), c = x % (CW / 4) * 4, n = (int)n0 + wn + c;
      const int64_t m = m0 + wm + 16 * a + r;
      const f32x4 v = *reinterpret_cast<const f32x4*>(&mine[r * (CW + 4) + c]);
      if (gridDim.y == 1) finish4<O>(e, v, m, n);
      else if (m < e.M && n < e.N) {
        float* p = part + ((int64_t)blockIdx.y * e.M + m) * e.N + n;
        if (n + 4 <= e.N) store_pack<float, 4>(p, v);
        else
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < e.N) p[i] = v[i];
      }
    }
  }
}

// Sums the splits in order and runs the epilogue: a pack of 4 outputs a thread; RUNS > 1 (many splits of a small output): 16 packs a workgroup, 16 runs
// of splits side by side, then the runs in order. (8 splits and fewer leave half of the runs idle: two of 2000 x 1500 took 37 us
// that way; a pack a thread takes 9 for two of 2048 x 2048.)
template <typename O, int RUNS>
__global__ __launch_bounds__(256) void linear_join(const float* __restrict__ part, int splits, Epilogue e) {
  constexpr int PACKS = 256 / RUNS;
  const int per = ope_cdiv_dev4(e.N), run = threadIdx.x / PACKS;
  const int64_t i = (int64_t)blockIdx.x * PACKS + (threadIdx.x % PACKS), m = i / per;
  const int n = (int)(i % per) * 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (m < e.M)
    for (int s = run; s < splits; s += RUNS) {
      const float* p = part + ((int64_t)s * e.M + m) * e.N + n;
      if (n + 4 <= e.N) acc += load_pack<float, 4>(p);
      else
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < e.N) acc[r] += p[r];
    }
  if constexpr (RUNS > 1) {
    __shared__ f32x4 lds[RUNS][PACKS + 1];
    lds[run][threadIdx.x % PACKS] = acc;
    __syncthreads();
    if (run) return;
    acc = lds[0][threadIdx.x];
    for (int r = 1; r < RUNS; ++r) acc += lds[r][threadIdx.x];
  }
  finish4<O>(e, acc, m, n);
}

// Few rows (up to 64): a workgroup has 16 columns, its eight waves every eighth 64 bytes of k, straight from memory to the matrix instructions -- the
// weights are read once and by whole lines, four loads of them in flight a wave, and nothing waits for a barrier but the last sum over the waves.
template <typename T, typename O, int MT>
__global__ __launch_bounds__(512) void linear_few(Operand A, Operand B, int64_t klen, Epilogue e) {
  constexpr int NW = 8, D = 4;
  __shared__ float lds[NW][MT][16][17];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const uint8_t* bp = B.p + min(n0 + j, B.rows - 1) * B.stride + 16 * g;
  const uint8_t* ap[MT];
#pragma unroll
  for (int a = 0; a < MT; ++a) ap[a] = A.p + min((int64_t)16 * a + j, A.rows - 1) * A.stride + 16 * g;
  f32x4 acc[MT];
#pragma unroll
  for (int a = 0; a < MT; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
  int64_t k = 64 * w;
  for (; k + 64 * NW * (D - 1) + 64 <= klen; k += 64 * NW * D) {
    u32x4 fb[D], fa[D][MT];
#pragma unroll
    for (int i = 0; i < D; ++i) {
      fb[i] = *reinterpret_cast<const u32x4_loose*>(bp + k + 64 * NW * i);
#pragma unroll
      for (int a = 0; a < MT; ++a) fa[i][a] = *reinterpret_cast<const u32x4_loose*>(ap[a] + k + 64 * NW * i);
    }
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
      for (int a = 0; a < MT; ++a) acc[a] = product<T>(fb[i], fa[i][a], acc[a]);
  }
  for (; k < klen; k += 64 * NW) {
    if (k + 64 <= klen) {
      const u32x4 fb = *reinterpret_cast<const u32x4_loose*>(bp + k);
#pragma unroll
      for (int a = 0; a < MT; ++a) acc[a] = product<T>(fb, *reinterpret_cast<const u32x4_loose*>(ap[a] + k), acc[a]);
    } else {
      const u32x4 fb = row16(bp - 16 * g, k + 16 * g, klen, (int)sizeof(T));
#pragma unroll
      for (int a = 0; a < MT; ++a) acc[a] = product<T>(fb, row16(ap[a] - 16 * g, k + 16 * g, klen, (int)sizeof(T)), acc[a]);
    }
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) lds[w][a][j][4 * g + r] = acc[a][r];
  __syncthreads();
  for (int a = w; a < MT; a += NW) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NW; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += lds[i][a][j][4 * g + r];
    finish4<O>(e, v, 16 * a + j, (int)n0 + 4 * g);
  }
}

// dz = dy act'(z), and the column sums of dz over a workgroup's kDzRows rows for dbias. 64 columns a workgroup; 4 neighbouring columns a lane, 16 rows side
// by side, all of a thread's loads before their first use. Without an activation only the sums. A kernel for each activation: with the choice inside,
// the code of all of them, unrolled, did not stay in the instruction cache (14 us for any small batch).
constexpr int kDzRows = 128;
template <typename T, int ACT>
__global__ __launch_bounds__(256) void linear_dz(const T* __restrict__ dy, const float* __restrict__ z, int64_t M, int N, T* __restrict__ dz,
                                                 float* __restrict__ sums) {
  constexpr int R = kDzRows / 16;
  __shared__ f32x4 lds[16][17];
  const int tn = ope_cdiv_dev64(N), n = (int)(blockIdx.x % tn) * 64 + (threadIdx.x & 15) * 4, r0 = threadIdx.x >> 4;
  const int64_t m0 = (int64_t)(blockIdx.x / tn) * kDzRows;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (n + 4 <= N) {
    f32x4 d[R], x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {                       // (rows past the last one read the last one's values again)
      const int64_t at = min(m0 + r0 + 16 * i, M - 1) * N + n;
      d[i] = load_pack<T, 4>(dy + at);
      if constexpr (ACT != OPE_ACT_NONE) x[i] = load_pack<float, 4>(z + at);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t m = m0 + r0 + 16 * i;
      if (m >= M) break;
      if constexpr (ACT != OPE_ACT_NONE) {
#pragma unroll
        for (int c = 0; c < 4; ++c) d[i][c] *= act_slope<sizeof(T) == 4>(x[i][c], ACT);
        store_pack<T, 4>(dz + m * N + n, d[i]);
      }
      s += d[i];
    }
  } else if (n < N) {
    for (int i = 0; i < R; ++i) {
      const int64_t m = m0 + r0 + 16 * i;
      if (m >= M) break;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (n + c < N) {
          float d = (float)dy[m * N + n + c];
          if constexpr (ACT != OPE_ACT_NONE) {
            d *= act_slope<sizeof(T) == 4>(z[m * N + n + c], ACT);
            dz[m * N + n + c] = (T)d;
          }
          s[c] += d;
        }
    }
  }
  if (!sums) return;
  lds[r0][threadIdx.x & 15] = s;
  __syncthreads();
  if (r0 || n >= N) return;
  for (int r = 1; r < 16; ++r) s += lds[r][threadIdx.x];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (n + c < N) sums[(int64_t)(blockIdx.x / tn) * N + n + c] = s[c];
}
template <typename T>
__global__ __launch_bounds__(1024) void linear_dbias(const float* __restrict__ sums, int tiles, int N, T* __restrict__ out) {
  __shared__ float lds[16][65];
  const int col = threadIdx.x & 63, run = threadIdx.x >> 6, n = blockIdx.x * 64 + col;
  float v = 0.f;
  if (n < N)
#pragma unroll 8
    for (int r = run; r < tiles; r += 16) v += sums[(int64_t)r * N + n];
  lds[run][col] = v;
  __syncthreads();
  if (run == 0 && n < N) {
    v = 0.f;
    for (int r = 0; r < 16; ++r) v += lds[r][col];
    out[n] = (T)v;
  }
}

// How one product is cut: the tile, and splits of k where the tiles alone leave CUs idle. Short contractions (under 8 steps of 128 bytes) and
// small outputs are bound by memory and latency: tiles of 64 x 64, five workgroups a CU. Otherwise the tile whose rounds over the chip cost least, in
// the time of a 64 x 64 tile's work at the rates measured for each:
//   bf16, 4096 x 4096 x 4096 : 588 / 816 / 973 TFLOP/s with tiles of 64 / 128 / 256; a tile of 128 that is alone on its CU waits for itself at every
//                              barrier (2048 x 2048 x 2048, one tile a CU: 493 against 527 with tiles of 64);
//   float32                  : 114 / 132 / 112.
struct Cut { int BM, tm, tn, steps, splits, per; bool few; };
static Cut cut_of(int64_t M, int64_t N, int64_t klen, bool may_be_few, int eb) {
  Cut c;
  c.few = may_be_few && M <= 64;
  c.steps = (int)((klen + 127) / 128);
  c.BM = 64;
  if (M > 64 && N > 64 && c.steps >= 8 && (int64_t)ope_cdiv(M, 128) * ope_cdiv(N, 128) >= 256) {
    auto rounds = [&](int t) { return ((int64_t)ope_cdiv(M, t) * ope_cdiv(N, t) + 255) / 256; };
    const int64_t n = rounds(128);
    if (eb == 4) {
      if (4 * n < rounds(64) / 0.86) c.BM = 128;
    } else {
      const double c64 = rounds(64) / 0.6, c128 = 4 * ((n - n % 2) / 0.83 + n % 2 / 0.55), c256 = 16. * rounds(256);
      if (c128 < c64) c.BM = 128;
      if (c256 < c128 && c256 < c64) c.BM = 256;
    }
  }
  c.tm = ope_cdiv(M, c.BM);
  c.tn = ope_cdiv(N, c.BM);
  const int64_t tiles = (int64_t)c.tm * c.tn;
  c.splits = 1;
  if (!c.few && c.BM == 64 && tiles && tiles < 512) {          // (no rows: no tiles)
    const int64_t want = 1024 / tiles, most = c.steps / 4;     // four workgroups a CU, four steps at least each
    c.splits = (int)(want < most ? want : most);
    if (c.splits < 1) c.splits = 1;
  }
  // One 128 x 128 tile a CU leaves it idle at every barrier; in float32 a second split pays for its join (dw of 4096 x 2048 x 2048: 393 against 293 + 9
  // us), in 16 bits the join's bytes would cost as much as the product gains.
  if (c.BM == 128 && eb == 4 && tiles < 512 && c.steps >= 32) c.splits = 2;
  c.per = ope_cdiv(c.steps, c.splits);
  if (c.per < 1) c.per = 1;
  c.splits = c.steps ? ope_cdiv(c.steps, c.per) : 1;
  return c;
}
static int64_t cut_floats(const Cut& c, int64_t M, int64_t N) { return c.splits > 1 ? (int64_t)c.splits * M * N : 0; }

// AA, BA: the contraction runs along memory in A / B
template <typename T, typename O, bool AA, bool BA>
static int launch_product(Operand A, Operand B, int64_t klen, const Epilogue& e, float* part, hipStream_t st) {
  const Cut c = cut_of(e.M, e.N, klen, AA && BA, (int)sizeof(T));
  if constexpr (AA && BA)
    if (c.few) {
      const dim3 grid((unsigned)ope_cdiv(e.N, 16));
      if (e.M <= 16) OPE_LAUNCH((linear_few<T, O, 1>), grid, dim3(512), 0, st, A, B, klen, e);
      else if (e.M <= 32) OPE_LAUNCH((linear_few<T, O, 2>), grid, dim3(512), 0, st, A, B, klen, e);
      else OPE_LAUNCH((linear_few<T, O, 4>), grid, dim3(512), 0, st, A, B, klen, e);
      OPE_CHECK_LAUNCH();
      return OPE_OK;
    }
  const dim3 grid((unsigned)((int64_t)c.tm * c.tn), (unsigned)c.splits);
  if (c.BM == 64) OPE_LAUNCH((linear_tile<T, O, 64, 64, 2, 2, AA, BA>), grid, dim3(256), 0, st, A, B, klen, c.tm, c.tn, c.per, e, part);
  else if (c.BM == 128) OPE_LAUNCH((linear_tile<T, O, 128, 128, 2, 2, AA, BA>), grid, dim3(256), 0, st, A, B, klen, c.tm, c.tn, c.per, e, part);
  else if constexpr (sizeof(T) < 4) OPE_LAUNCH((linear_tile<T, O, 256, 256, 2, 4, AA, BA>), grid, dim3(512), 0, st, A, B, klen, c.tm, c.tn, c.per, e, part);
  OPE_CHECK_LAUNCH();
  if (c.splits > 1) {
    const int64_t n = e.M * ((e.N + 3) / 4);
    if (c.splits > 8) OPE_LAUNCH((linear_join<O, 16>), dim3((unsigned)((n + 15) / 16)), dim3(256), 0, st, part, c.splits, e);
    else OPE_LAUNCH((linear_join<O, 1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, c.splits, e);
    OPE_CHECK_LAUNCH();
  }
  return OPE_OK;
}

static bool linear_ok(const ope_linear_cfg* c) {
  if (!c || c->rows < 0 || c->rows >= ((int64_t)1 << 31) || c->in_width < 1 || c->out_width < 1) return false;
  if (c->in_width > (1 << 20) || c->out_width > (1 << 20) || c->x_stride < 0 || c->residual_stride < 0) return false;
  if (c->activation < OPE_ACT_NONE || c->activation > OPE_ACT_GELU || !elem_float(c->out_dtype)) return false;
  if (c->dtype != OPE_E4M3 && (!elem_float(c->dtype) || c->dtype != c->out_dtype)) return false;
  const int64_t tm = ope_cdiv(c->rows, 64), tn = ope_cdiv(c->out_width, 64), tk = ope_cdiv(c->in_width, 64);
  return launch_fits(tm * tn, 256) && launch_fits(tm * tk, 256) && launch_fits(tn * tk * 16, 256);      // (16: the fill of dw where there are no rows)
}

// What the backward pass needs beside its outputs, as offsets in bytes
struct BwdPlan { int64_t dz, sums, part_dx, part_dw, bytes; };
static BwdPlan bwd_plan(const ope_linear_cfg* c) {
  BwdPlan p;
  const int64_t M = c->rows, N = c->out_width, K = c->in_width, eb = elem_bytes(c->dtype);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t r = o; o += (bytes + 255) & ~(int64_t)255; return r; };
  p.dz = take(c->activation != OPE_ACT_NONE ? M * N * eb : 0);
  p.sums = take((int64_t)ope_cdiv(M, kDzRows) * N * 4);
  p.part_dx = take(cut_floats(cut_of(M, K, N * eb, false, (int)eb), M, K) * 4);
  p.part_dw = take(cut_floats(cut_of(N, K, M * eb, false, (int)eb), N, K) * 4);
  p.bytes = o;
  return p;
}

template <typename T>
__global__ void linear_zero(T* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = (T)0.f;
}

}  // namespace ope
using namespace ope;

extern "C" int64_t ope_linear_workspace_bytes(const ope_linear_cfg* cfg) {
  if (!linear_ok(cfg)) return OPE_EINVAL;
  return cut_floats(cut_of(cfg->rows, cfg->out_width, (int64_t)cfg->in_width * elem_bytes(cfg->dtype), true, elem_bytes(cfg->dtype)), cfg->rows, cfg->out_width) * 4;
}

extern "C" int ope_linear(const ope_linear_cfg* cfg, const void* x, const void* w, const float* x_scale, const float* w_scale, const void* bias,
                          const void* residual, void* y, float* z_out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!linear_ok(cfg)) return OPE_EINVAL;
  if (cfg->rows == 0) return OPE_OK;
  const bool fp8 = cfg->dtype == OPE_E4M3;
  if (!x || !w || !y || fp8 != (x_scale != nullptr) || fp8 != (w_scale != nullptr)) return OPE_EINVAL;
  const int64_t need = ope_linear_workspace_bytes(cfg);
  if (workspace_bytes < need || (need && !workspace)) return OPE_ENOSPC;
  const int eb = elem_bytes(cfg->dtype);
  const Epilogue e = {x_scale, w_scale, bias, residual, y, z_out, cfg->residual_stride, cfg->rows, cfg->out_width, cfg->activation};
  const Operand A = {(const uint8_t*)x, cfg->rows, cfg->x_stride * eb}, B = {(const uint8_t*)w, cfg->out_width, (int64_t)cfg->in_width * eb};
  const int64_t klen = (int64_t)cfg->in_width * eb;
  hipStream_t st = (hipStream_t)stream;
  return with_elem(cfg->out_dtype, [&](auto t) {
    typedef decltype(t) T;
    return fp8 ? launch_product<e4m3_t, T, true, true>(A, B, klen, e, (float*)workspace, st) : launch_product<T, T, true, true>(A, B, klen, e, (float*)workspace, st);
  });
}

extern "C" int64_t ope_linear_backward_workspace_bytes(const ope_linear_cfg* cfg) {
  if (!linear_ok(cfg) || cfg->dtype == OPE_E4M3) return OPE_EINVAL;
  return bwd_plan(cfg).bytes;
}

extern "C" int ope_linear_backward(const ope_linear_cfg* cfg, const void* dy, const float* z, const void* x, const void* w, void* dx, void* dw, void* dbias,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  if (!linear_ok(cfg) || cfg->dtype == OPE_E4M3) return OPE_EINVAL;
  const int64_t M = cfg->rows;
  const int N = cfg->out_width, K = cfg->in_width, eb = elem_bytes(cfg->dtype);
  hipStream_t st = (hipStream_t)stream;
  const bool acts = cfg->activation != OPE_ACT_NONE;
  if (M && (!dy || (acts && !z) || (dw && !x) || (dx && !w))) return OPE_EINVAL;
  const BwdPlan p = bwd_plan(cfg);
  if (workspace_bytes < p.bytes || (p.bytes && !workspace)) return OPE_ENOSPC;
  uint8_t* ws = (uint8_t*)workspace;
  return with_elem(cfg->dtype, [&](auto t) {
    typedef decltype(t) T;
    if (M == 0) {            // sums over no rows
      if (dw) OPE_LAUNCH((linear_zero<T>), dim3((unsigned)(((int64_t)N * K + 255) / 256)), dim3(256), 0, st, (T*)dw, (int64_t)N * K);
      if (dbias) OPE_LAUNCH((linear_zero<T>), dim3(ope_cdiv(N, 256)), dim3(256), 0, st, (T*)dbias, (int64_t)N);
      OPE_CHECK_LAUNCH();
      return OPE_OK;
    }
    const T* dz = acts ? (const T*)(ws + p.dz) : (const T*)dy;
    const int tm = ope_cdiv(M, kDzRows);
    if (acts || dbias) {
      const dim3 grid((unsigned)((int64_t)tm * ope_cdiv(N, 64)));
      T* const out = acts ? (T*)(ws + p.dz) : nullptr;
      float* const sums = dbias ? (float*)(ws + p.sums) : nullptr;
      switch (cfg->activation) {
        case OPE_ACT_NONE: OPE_LAUNCH((linear_dz<T, OPE_ACT_NONE>), grid, dim3(256), 0, st, (const T*)dy, z, M, N, out, sums); break;
        case OPE_ACT_RELU: OPE_LAUNCH((linear_dz<T, OPE_ACT_RELU>), grid, dim3(256), 0, st, (const T*)dy, z, M, N, out, sums); break;
        case OPE_ACT_TANH: OPE_LAUNCH((linear_dz<T, OPE_ACT_TANH>), grid, dim3(256), 0, st, (const T*)dy, z, M, N, out, sums); break;
        case OPE_ACT_SILU: OPE_LAUNCH((linear_dz<T, OPE_ACT_SILU>), grid, dim3(256), 0, st, (const T*)dy, z, M, N, out, sums); break;
        case OPE_ACT_GELU: OPE_LAUNCH((linear_dz<T, OPE_ACT_GELU>), grid, dim3(256), 0, st, (const T*)dy, z, M, N, out, sums); break;
      }
      OPE_CHECK_LAUNCH();
    }
    if (dbias) {
      OPE_LAUNCH((linear_dbias<T>), dim3(ope_cdiv(N, 64)), dim3(1024), 0, st, (const float*)(ws + p.sums), tm, N, (T*)dbias);
      OPE_CHECK_LAUNCH();
    }
    if (dx) {
      const Epilogue e = {nullptr, nullptr, nullptr, nullptr, dx, nullptr, 0, M, K, OPE_ACT_NONE};
      const int rc = launch_product<T, T, true, false>({(const uint8_t*)dz, M, (int64_t)N * eb}, {(const uint8_t*)w, K, (int64_t)K * eb}, (int64_t)N * eb, e,
                                                       (float*)(ws + p.part_dx), st);
      if (rc) return rc;
    }
    if (dw) {
      const Epilogue e = {nullptr, nullptr, nullptr, nullptr, dw, nullptr, 0, N, K, OPE_ACT_NONE};
      const int rc = launch_product<T, T, false, false>({(const uint8_t*)dz, N, (int64_t)N * eb}, {(const uint8_t*)x, K, cfg->x_stride * eb}, M * eb, e,
                                                        (float*)(ws + p.part_dw), st);
      if (rc) return rc;
    }
    return OPE_OK;
  });
}
