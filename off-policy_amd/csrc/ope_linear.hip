// Linear layer with bias, activation and residual in its epilogue, and its gradients (ope_linear, ope_linear_backward; ope.h).
//
// One product kernel for all four operand types: C[m][n] = sum_k A[m][k] B[n][k], both operands with the contraction running along memory.
// It counts in BYTES of k: a lane takes 16 bytes of one row -- 4 float32, 8 bfloat16 / float16 or 16 e4m3 values -- and feeds them to the matrix
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

__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case OPE_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case OPE_ACT_TANH: return tanhf(z);
    case OPE_ACT_SILU: return z / (1.f + expf(-z));
    case OPE_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  }
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case OPE_ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case OPE_ACT_TANH: { const float t = tanhf(z); return 1.f - t * t; }
    case OPE_ACT_SILU: { const float s = 1.f / (1.f + expf(-z)); return s * (1.f + z * (1.f - s)); }
    case OPE_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  }
  return 1.f;
}

struct Epilogue {
  const float *x_scale, *w_scale;
  const void *bias, *residual;
  void *y, *z;
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
  f32x4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = act_of(z[r], e.act) + res[r];
  const int64_t at = m * e.N + n;
  if (live == 4) {
    store_pack<O, 4>((O*)e.y + at, y);
    if (e.z) store_pack<O, 4>((O*)e.z + at, z);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < live) {
        ((O*)e.y)[at + r] = (O)y[r];
        if (e.z) ((O*)e.z)[at + r] = (O)z[r];
      }
  }
}

struct Operand {
  const uint8_t* p;
  int64_t rows, stride;            // stride in bytes
};

// The tile kernel: BM x BN outputs a workgroup of 4 waves (2 x 2), 128 bytes of k a step, two LDS buffers: the next step's rows travel from
// memory to registers while this step's are multiplied. 16-byte pieces are stored at piece ^ (row & 7), so neither the stores nor the 16-row
// fragment reads collide in the banks. gridDim.y > 1: split of k; part [split][M][N] takes the sums and linear_join finishes.
template <typename T, typename O, int BM, int BN>
__global__ __launch_bounds__(256) void linear_tile(Operand A, Operand B, int64_t klen, int tiles_n, int steps_per, Epilogue e, float* __restrict__ part) {
  constexpr int MT = BM / 32, NT = BN / 32, LA = BM / 32, LB = BN / 32;
  __shared__ u32x4 As[2][BM][8], Bs[2][BN][8];
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * BM, n0 = (int64_t)(blockIdx.x % tiles_n) * BN;
  const int wm = (w >> 1) * (BM / 2), wn = (w & 1) * (BN / 2);
  const int row = threadIdx.x >> 3, piece = threadIdx.x & 7;
  const int steps = (int)((klen + 127) / 128), first = blockIdx.y * steps_per, last = min(first + steps_per, steps);
  u32x4 ra[LA], rb[LB];
  auto fetch = [&](int s) {
    const int64_t k = (int64_t)s * 128 + piece * 16;
#pragma unroll
    for (int i = 0; i < LA; ++i) ra[i] = row16(A.p + min(m0 + row + 32 * i, A.rows - 1) * A.stride, k, klen, (int)sizeof(T));
#pragma unroll
    for (int i = 0; i < LB; ++i) rb[i] = row16(B.p + min(n0 + row + 32 * i, B.rows - 1) * B.stride, k, klen, (int)sizeof(T));
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (first < last) fetch(first);
  for (int s = first; s < last; ++s) {
    const int buf = (s - first) & 1;
#pragma unroll
    for (int i = 0; i < LA; ++i) As[buf][row + 32 * i][piece ^ (row & 7)] = ra[i];
#pragma unroll
    for (int i = 0; i < LB; ++i) Bs[buf][row + 32 * i][piece ^ (row & 7)] = rb[i];
    lds_barrier();
    if (s + 1 < last) fetch(s + 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 fa[MT], fb[NT];
#pragma unroll
      for (int a = 0; a < MT; ++a) fa[a] = As[buf][wm + 16 * a + j][(4 * h + g) ^ (j & 7)];
#pragma unroll
      for (int b = 0; b < NT; ++b) fb[b] = Bs[buf][wn + 16 * b + j][(4 * h + g) ^ (j & 7)];
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = product<T>(fb[b], fa[a], acc[a][b]);
    }
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      const int64_t m = m0 + wm + 16 * a + j;
      const int n = (int)n0 + wn + 16 * b + 4 * g;
      if (gridDim.y == 1) finish4<O>(e, acc[a][b], m, n);
      else if (m < e.M && n < e.N) {
        float* p = part + ((int64_t)blockIdx.y * e.M + m) * e.N + n;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < e.N) p[r] = acc[a][b][r];
      }
    }
}

// Sums the splits in order and runs the epilogue.
template <typename O>
__global__ __launch_bounds__(256) void linear_join(const float* __restrict__ part, int splits, Epilogue e) {
  const int per = ope_cdiv_dev4(e.N);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / per;
  const int n = (int)(i % per) * 4;
  if (m >= e.M) return;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float* p = part + ((int64_t)s * e.M + m) * e.N + n;
    if (n + 4 <= e.N) acc += load_pack<float, 4>(p);
    else
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < e.N) acc[r] += p[r];
  }
  finish4<O>(e, acc, m, n);
}

// Few rows (up to 64): a workgroup has 16 columns, its four waves every fourth 64 bytes of k, straight from memory to the matrix instructions --
// the weights are read once and by whole lines, and nothing waits for a barrier but the last sum over the waves.
template <typename T, typename O, int MT>
__global__ __launch_bounds__(256) void linear_few(Operand A, Operand B, int64_t klen, Epilogue e) {
  __shared__ float lds[4][MT][16][17];
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const uint8_t* bp = B.p + min(n0 + j, B.rows - 1) * B.stride;
  const uint8_t* ap[MT];
#pragma unroll
  for (int a = 0; a < MT; ++a) ap[a] = A.p + min((int64_t)16 * a + j, A.rows - 1) * A.stride;
  f32x4 acc[MT];
#pragma unroll
  for (int a = 0; a < MT; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int64_t k0 = 64 * w; k0 < klen; k0 += 256) {
    const int64_t k = k0 + 16 * g;
    const u32x4 fb = row16(bp, k, klen, (int)sizeof(T));
#pragma unroll
    for (int a = 0; a < MT; ++a) acc[a] = product<T>(fb, row16(ap[a], k, klen, (int)sizeof(T)), acc[a]);
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int r = 0; r < 4; ++r) lds[w][a][j][4 * g + r] = acc[a][r];
  __syncthreads();
  for (int a = w; a < MT; a += 4) {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = ((lds[0][a][j][4 * g + r] + lds[1][a][j][4 * g + r]) + lds[2][a][j][4 * g + r]) + lds[3][a][j][4 * g + r];
    finish4<O>(e, v, 16 * a + j, (int)n0 + 4 * g);
  }
}

// dz = dy act'(z) in tiles of 64 x 64: dz as it lies (where act' is not 1), its transpose [N][ldt], and the tile's column sums for dbias.
// The same kernel transposes x and w (z = NULL, dz = NULL, no sums).
template <typename T>
__global__ __launch_bounds__(256) void linear_turn(const T* __restrict__ dy, int64_t stride, const T* __restrict__ z, int64_t M, int N, int act,
                                                   T* __restrict__ dz, T* __restrict__ out, int64_t ldt, float* __restrict__ sums) {
  __shared__ float tile[64][65];
  const int tn = ope_cdiv_dev64(N);
  const int64_t m0 = (int64_t)(blockIdx.x / tn) * 64;
  const int n0 = (int)(blockIdx.x % tn) * 64;
  for (int x = threadIdx.x; x < 64 * 64; x += 256) {
    const int r = x >> 6, c = x & 63;
    const int64_t m = m0 + r;
    const int n = n0 + c;
    float v = 0.f;
    if (m < M && n < N) {
      v = (float)dy[m * stride + n];
      if (z) v *= act_slope((float)z[m * (int64_t)N + n], act);
      if (dz) dz[m * (int64_t)N + n] = (T)v;
    }
    tile[r][c] = v;
  }
  __syncthreads();
  if (out)
    for (int x = threadIdx.x; x < 64 * 64; x += 256) {
      const int c = x >> 6, r = x & 63;
      if (n0 + c < N && m0 + r < M) out[(int64_t)(n0 + c) * ldt + m0 + r] = (T)tile[r][c];
    }
  if (sums && threadIdx.x < 64 && n0 + (int)threadIdx.x < N) {
    float s = 0.f;
    for (int r = 0; r < 64; ++r) s += tile[r][threadIdx.x];
    sums[(int64_t)(blockIdx.x / tn) * N + n0 + threadIdx.x] = s;
  }
}
template <typename T>
__global__ __launch_bounds__(1024) void linear_dbias(const float* __restrict__ sums, int tiles, int N, T* __restrict__ out) {
  __shared__ float lds[16][65];
  const int col = threadIdx.x & 63, run = threadIdx.x >> 6, n = blockIdx.x * 64 + col;
  float v = 0.f;
  if (n < N)
    for (int r = run; r < tiles; r += 16) v += sums[(int64_t)r * N + n];
  lds[run][col] = v;
  __syncthreads();
  if (run == 0 && n < N) {
    v = 0.f;
    for (int r = 0; r < 16; ++r) v += lds[r][col];
    out[n] = (T)v;
  }
}

// How one product is cut: tile size, and splits of k where the tiles alone leave CUs idle.
struct Cut { int BM, tm, tn, steps, splits, per; bool few; };
static Cut cut_of(int64_t M, int64_t N, int64_t klen, bool may_be_few) {
  Cut c;
  c.few = may_be_few && M <= 64;
  c.steps = (int)((klen + 127) / 128);
  c.BM = (int64_t)ope_cdiv(M, 128) * ope_cdiv(N, 128) >= 256 ? 128 : 64;
  c.tm = ope_cdiv(M, c.BM);
  c.tn = ope_cdiv(N, c.BM);
  const int64_t tiles = (int64_t)c.tm * c.tn;
  c.splits = 1;
  if (!c.few && tiles && tiles < 256) {        // (no rows: no tiles)
    const int64_t want = 512 / tiles, most = c.steps / 4;      // two workgroups a CU, four steps at least each
    c.splits = (int)(want < most ? want : most);
    if (c.splits < 1) c.splits = 1;
  }
  c.per = ope_cdiv(c.steps, c.splits);
  if (c.per < 1) c.per = 1;
  c.splits = c.steps ? ope_cdiv(c.steps, c.per) : 1;
  return c;
}
static int64_t cut_floats(const Cut& c, int64_t M, int64_t N) { return c.splits > 1 ? (int64_t)c.splits * M * N : 0; }

template <typename T, typename O>
static int launch_product(Operand A, Operand B, int64_t klen, const Epilogue& e, bool may_be_few, float* part, hipStream_t st) {
  const Cut c = cut_of(e.M, e.N, klen, may_be_few);
  if (c.few) {
    const dim3 grid((unsigned)ope_cdiv(e.N, 16));
    if (e.M <= 16) OPE_LAUNCH((linear_few<T, O, 1>), grid, dim3(256), 0, st, A, B, klen, e);
    else if (e.M <= 32) OPE_LAUNCH((linear_few<T, O, 2>), grid, dim3(256), 0, st, A, B, klen, e);
    else OPE_LAUNCH((linear_few<T, O, 4>), grid, dim3(256), 0, st, A, B, klen, e);
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  }
  const dim3 grid((unsigned)((int64_t)c.tm * c.tn), (unsigned)c.splits);
  if (c.BM == 128) OPE_LAUNCH((linear_tile<T, O, 128, 128>), grid, dim3(256), 0, st, A, B, klen, c.tn, c.per, e, part);
  else OPE_LAUNCH((linear_tile<T, O, 64, 64>), grid, dim3(256), 0, st, A, B, klen, c.tn, c.per, e, part);
  OPE_CHECK_LAUNCH();
  if (c.splits > 1) {
    const int64_t n = e.M * ((e.N + 3) / 4);
    OPE_LAUNCH((linear_join<O>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, part, c.splits, e);
    OPE_CHECK_LAUNCH();
  }
  return OPE_OK;
}

static bool linear_ok(const ope_linear_cfg* c) {
  if (!c || c->rows < 0 || c->rows >= ((int64_t)1 << 31) || c->in_width < 1 || c->out_width < 1) return false;
  if (c->in_width > (1 << 20) || c->out_width > (1 << 20) || c->x_stride < 0 || c->residual_stride < 0) return false;
  if (c->activation < OPE_ACT_NONE || c->activation > OPE_ACT_GELU || !elem_float(c->out_dtype)) return false;
  if (c->dtype != OPE_E4M3 && (!elem_float(c->dtype) || c->dtype != c->out_dtype)) return false;
  return (int64_t)ope_cdiv(c->rows, 64) * ope_cdiv(c->out_width, 64) < ((int64_t)1 << 31) &&
         (int64_t)ope_cdiv(c->rows, 64) * ope_cdiv(c->in_width, 64) < ((int64_t)1 << 31);
}
static int64_t ld_of(int64_t rows) { return (rows + 15) & ~(int64_t)15; }     // rows of a transpose start on 16-byte pieces

// What the backward pass needs beside its outputs, in elements of the type (e) and in floats (f)
struct BwdPlan { int64_t dz, dzt, xt, wt, sums, part_dx, part_dw, bytes; };
static BwdPlan bwd_plan(const ope_linear_cfg* c) {
  BwdPlan p;
  const int64_t M = c->rows, N = c->out_width, K = c->in_width, eb = elem_bytes(c->dtype);
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t r = o; o += (bytes + 255) & ~(int64_t)255; return r; };
  p.dz = take(c->activation != OPE_ACT_NONE ? M * N * eb : 0);
  p.dzt = take(N * ld_of(M) * eb);
  p.xt = take(K * ld_of(M) * eb);
  p.wt = take(K * ld_of(N) * eb);
  p.sums = take((int64_t)ope_cdiv(M, 64) * N * 4);
  p.part_dx = take(cut_floats(cut_of(M, K, N * eb, false), M, K) * 4);
  p.part_dw = take(cut_floats(cut_of(N, K, M * eb, false), N, K) * 4);
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
  return cut_floats(cut_of(cfg->rows, cfg->out_width, (int64_t)cfg->in_width * elem_bytes(cfg->dtype), true), cfg->rows, cfg->out_width) * 4;
}

extern "C" int ope_linear(const ope_linear_cfg* cfg, const void* x, const void* w, const float* x_scale, const float* w_scale, const void* bias,
                          const void* residual, void* y, void* z_out, void* workspace, int64_t workspace_bytes, void* stream) {
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
    return fp8 ? launch_product<e4m3_t, T>(A, B, klen, e, true, (float*)workspace, st) : launch_product<T, T>(A, B, klen, e, true, (float*)workspace, st);
  });
}

extern "C" int64_t ope_linear_backward_workspace_bytes(const ope_linear_cfg* cfg) {
  if (!linear_ok(cfg) || cfg->dtype == OPE_E4M3) return OPE_EINVAL;
  return bwd_plan(cfg).bytes;
}

extern "C" int ope_linear_backward(const ope_linear_cfg* cfg, const void* dy, const void* z, const void* x, const void* w, void* dx, void* dw, void* dbias,
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
    const int tm = ope_cdiv(M, 64);
    const int64_t ldm = ld_of(M), ldn = ld_of(N);
    const T* dz = acts ? (const T*)(ws + p.dz) : (const T*)dy;
    if (acts || dw || dbias) {
      OPE_LAUNCH((linear_turn<T>), dim3((unsigned)((int64_t)tm * ope_cdiv(N, 64))), dim3(256), 0, st, (const T*)dy, (int64_t)N, acts ? (const T*)z : nullptr, M, N,
                 cfg->activation, acts ? (T*)(ws + p.dz) : nullptr, dw ? (T*)(ws + p.dzt) : nullptr, ldm, dbias ? (float*)(ws + p.sums) : nullptr);
      OPE_CHECK_LAUNCH();
    }
    if (dbias) {
      OPE_LAUNCH((linear_dbias<T>), dim3(ope_cdiv(N, 64)), dim3(1024), 0, st, (const float*)(ws + p.sums), tm, N, (T*)dbias);
      OPE_CHECK_LAUNCH();
    }
    if (dx) {
      OPE_LAUNCH((linear_turn<T>), dim3((unsigned)((int64_t)ope_cdiv(N, 64) * ope_cdiv(K, 64))), dim3(256), 0, st, (const T*)w, (int64_t)K, (const T*)nullptr, (int64_t)N, K, 0,
                 (T*)nullptr, (T*)(ws + p.wt), ldn, (float*)nullptr);
      OPE_CHECK_LAUNCH();
      const Epilogue e = {nullptr, nullptr, nullptr, nullptr, dx, nullptr, 0, M, K, OPE_ACT_NONE};
      const int rc = launch_product<T, T>({(const uint8_t*)dz, M, (int64_t)N * eb}, {ws + p.wt, K, ldn * eb}, (int64_t)N * eb, e, false, (float*)(ws + p.part_dx), st);
      if (rc) return rc;
    }
    if (dw) {
      OPE_LAUNCH((linear_turn<T>), dim3((unsigned)((int64_t)tm * ope_cdiv(K, 64))), dim3(256), 0, st, (const T*)x, cfg->x_stride, (const T*)nullptr, M, K, 0, (T*)nullptr,
                 (T*)(ws + p.xt), ldm, (float*)nullptr);
      OPE_CHECK_LAUNCH();
      const Epilogue e = {nullptr, nullptr, nullptr, nullptr, dw, nullptr, 0, N, K, OPE_ACT_NONE};
      const int rc = launch_product<T, T>({ws + p.dzt, N, ldm * eb}, {ws + p.xt, K, ldm * eb}, M * eb, e, false, (float*)(ws + p.part_dw), st);
      if (rc) return rc;
    }
    return OPE_OK;
  });
}
