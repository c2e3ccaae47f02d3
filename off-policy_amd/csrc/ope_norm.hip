// RMS norm with the residual's addition, its gradients, and rows in 8 bits with one scale each (ope_rms_norm, ope_rms_norm_backward,
// ope_quantize_rows; ope.h).
//
// Bound by memory: one read of x and the residual, one write of s and y. A row lives in the registers of L lanes (L = 16, 64, 256 or 1024,
// NV packs of 16 bytes a lane), so the mean, the row's largest value and the stores need one pass. L follows the row's width alone: the
// smallest that holds it in 4 packs a lane -- narrow rows share a wave (16 lanes a row: a width of 64 in float32 keeps all lanes busy), wide
// ones get a workgroup. Rows over 1024 * 4 packs are walked again for each pass (norm_long).
// A row whose width is no multiple of the pack ends in a pack that is moved back to end with the row; the elements it shares with the pack
// in front are counted once (`first`), and written twice with the same value. Packs need no alignment beyond the element's (ope_elem.h).
#include "ope_elem.h"

#include <type_traits>

namespace ope {

constexpr float kE4m3Max = 448.f;
constexpr float kE4m3MinScale = 1.17549435e-38f;   // 2^-126: keeps y / scale finite on rows of zeros and of subnormals

__device__ __forceinline__ unsigned wave_umax(unsigned v, int width) {
  for (int m = 1; m < width; m <<= 1) v = max(v, (unsigned)__shfl_xor((int)v, m, 64));
  return v;
}
template <int L>
__device__ __forceinline__ float group_sum(float v, float* lds) {
  v = row16_sum(v);
  if (L >= 64) v = rowsum4(v);
  if (L > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[w] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < L / 64; ++i) v += lds[i];
    __syncthreads();
  }
  return v;
}
// The largest |y| by its bits: a NaN is larger than every number there, so a row that holds one gets it as its scale.
template <int L>
__device__ __forceinline__ unsigned group_umax(unsigned v, float* lds) {
  v = wave_umax(v, L >= 64 ? 64 : L);
  if (L > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[w] = __uint_as_float(v);
    __syncthreads();
    v = 0;
    for (int i = 0; i < L / 64; ++i) v = max(v, __float_as_uint(lds[i]));
    __syncthreads();
  }
  return v;
}
__device__ __forceinline__ float scale_of(unsigned amax_bits) {
  const float a = __uint_as_float(amax_bits);
  return a < kE4m3Max * kE4m3MinScale ? kE4m3MinScale : a / kE4m3Max;     // (a NaN takes the division)
}
__device__ __forceinline__ float clamp_e4m3(float v) { return v > kE4m3Max ? kE4m3Max : (v < -kE4m3Max ? -kE4m3Max : v); }   // keeps NaN
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const typename Pack<float, VEC>::fvec y, float scale) {
  typedef uint8_t bytes __attribute__((ext_vector_type(VEC)));
  typedef bytes loose __attribute__((aligned(1)));
  bytes b;
#pragma unroll
  for (int e = 0; e < VEC; e += 2) {
    const int two = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(y[e] / scale), clamp_e4m3(y[e + 1 < VEC ? e + 1 : e] / scale), 0, false);
    b[e] = (uint8_t)(two & 255);
    if (e + 1 < VEC) b[e + 1] = (uint8_t)((two >> 8) & 255);
  }
  *reinterpret_cast<loose*>(p) = b;
}
__device__ __forceinline__ void store_e4m3_1(uint8_t* p, float y, float scale) {
  *p = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(y / scale), 0.f, 0, false) & 255);
}

// Place of pack i: where it starts, and the first element that is its own.
__device__ __forceinline__ int pack_at(int i, int VEC, int D) { return min(i * VEC, D - VEC); }

// NORM: y = s w rstd; otherwise y = s (ope_quantize_rows). OUT8: 8-bit output.
template <typename T, int VEC, int L, int NV, bool NORM, bool OUT8>
__global__ __launch_bounds__(L > 256 ? L : 256) void norm_rows(ope_norm_cfg c, const T* __restrict__ x, const T* __restrict__ residual,
                                                               const T* __restrict__ weight, void* __restrict__ y, float* __restrict__ scale,
                                                               T* sum_out, float* __restrict__ rstd_out) {
  typedef typename Pack<T, VEC>::fvec fvec;
  __shared__ float lds[16];
  const int D = c.width, nvec = (D + VEC - 1) / VEC, lane = threadIdx.x % L;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / L) + threadIdx.x / L;
  const bool on = row < c.rows;                       // lanes of absent rows stay for the barriers
  fvec s[NV];
  float sq = 0.f;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = lane + n * L, p = pack_at(i, VEC, D);
    s[n] = (fvec)(0.f);
    if (on && i < nvec) {
      s[n] = load_pack<T, VEC>(x + row * c.x_stride + p);
      if (residual) s[n] += load_pack<T, VEC>(residual + row * c.residual_stride + p);
      if (NORM)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (p + e >= i * VEC) sq = fmaf(s[n][e], s[n][e], sq);
    }
  }
  float rstd = 1.f;
  if (NORM) rstd = 1.f / sqrtf(group_sum<L>(sq, lds) / (float)D + c.eps);
  if (NORM && rstd_out && on && lane == 0) rstd_out[row] = rstd;
  fvec out[NV];
  unsigned big = 0;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = lane + n * L, p = pack_at(i, VEC, D);
    out[n] = s[n];
    if (on && i < nvec) {
      if (sum_out) store_pack<T, VEC>(sum_out + row * D + p, s[n]);
      if (NORM) out[n] = s[n] * rstd * load_pack<T, VEC>(weight + p);
      if (!OUT8) store_pack<T, VEC>((T*)y + row * D + p, out[n]);
      if (OUT8)
#pragma unroll
        for (int e = 0; e < VEC; ++e) big = max(big, __float_as_uint(out[n][e]) & 0x7fffffffu);
    }
  }
  if (!OUT8) return;
  const float sc = scale_of(group_umax<L>(big, lds));
  if (on && lane == 0) scale[row] = sc;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = lane + n * L;
    if (on && i < nvec) store_e4m3<VEC>((uint8_t*)y + row * D + pack_at(i, VEC, D), out[n], sc);
  }
}

// Rows that do not fit the registers of a workgroup: one workgroup walks the row once for the mean, once for the largest value, once to write.
template <typename T, bool NORM, bool OUT8>
__global__ __launch_bounds__(1024) void norm_long(ope_norm_cfg c, const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ weight,
                                                  void* __restrict__ y, float* __restrict__ scale, T* sum_out, float* __restrict__ rstd_out) {
  __shared__ float lds[16];
  const int D = c.width;
  const int64_t row = blockIdx.x;
  auto at = [&](int d) { return (float)x[row * c.x_stride + d] + (residual ? (float)residual[row * c.residual_stride + d] : 0.f); };
  float rstd = 1.f;
  if (NORM) {
    float sq = 0.f;
    for (int d = threadIdx.x; d < D; d += 1024) { const float s = at(d); sq = fmaf(s, s, sq); }
    rstd = 1.f / sqrtf(group_sum<1024>(sq, lds) / (float)D + c.eps);
    if (rstd_out && threadIdx.x == 0) rstd_out[row] = rstd;
  }
  float sc = 1.f;
  if (OUT8) {
    unsigned big = 0;
    for (int d = threadIdx.x; d < D; d += 1024) big = max(big, __float_as_uint(NORM ? at(d) * rstd * (float)weight[d] : at(d)) & 0x7fffffffu);
    sc = scale_of(group_umax<1024>(big, lds));
    if (threadIdx.x == 0) scale[row] = sc;
  }
  for (int d = threadIdx.x; d < D; d += 1024) {
    const float s = at(d), o = NORM ? s * rstd * (float)weight[d] : s;
    if (sum_out) sum_out[row * D + d] = (T)s;
    if (OUT8) store_e4m3_1((uint8_t*)y + row * D + d, o, sc);
    else ((T*)y)[row * D + d] = (T)o;
  }
}

// Gradients. A workgroup walks every gridDim-th group of rows and keeps its share of dweight in registers; the shares go to `part`
// [gridDim][nvec * VEC] and norm_dweight adds them in order. dx needs nothing but its own row.
template <typename T, int VEC, int L, int NV>
__global__ __launch_bounds__(L > 256 ? L : 256) void norm_bwd(ope_norm_cfg c, const T* dy, const T* dsum, const T* __restrict__ s_in,
                                                              const T* __restrict__ residual, const T* __restrict__ weight, const float* __restrict__ rstd_in, T* dx,
                                                              float* __restrict__ part) {
  typedef typename Pack<T, VEC>::fvec fvec;
  constexpr int G = L > 256 ? 1 : 256 / L;             // rows a workgroup has in hand
  __shared__ float lds[16];
  __shared__ float share[G > 1 ? G * L * NV * VEC : 1];
  const int D = c.width, nvec = (D + VEC - 1) / VEC, lane = threadIdx.x % L, grp = threadIdx.x / L;
  fvec w[NV], acc[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int i = lane + n * L;
    acc[n] = (fvec)(0.f);
    w[n] = i < nvec ? load_pack<T, VEC>(weight + pack_at(i, VEC, D)) : (fvec)(0.f);
  }
  for (int64_t first = (int64_t)blockIdx.x * G; first < c.rows; first += (int64_t)gridDim.x * G) {   // the same count for every lane: barriers inside
    const int64_t row = first + grp;
    const bool on = row < c.rows;
    const float rstd = on ? rstd_in[row] : 0.f;
    fvec s[NV], d[NV];
    float dot = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = lane + n * L, p = pack_at(i, VEC, D);
      s[n] = d[n] = (fvec)(0.f);
      if (on && i < nvec) {
        s[n] = load_pack<T, VEC>(s_in + row * c.x_stride + p);
        if (residual) s[n] += load_pack<T, VEC>(residual + row * c.residual_stride + p);
        d[n] = load_pack<T, VEC>(dy + row * D + p);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (p + e >= i * VEC) {
            dot = fmaf(d[n][e] * w[n][e], s[n][e], dot);
            acc[n][e] = fmaf(d[n][e], s[n][e] * rstd, acc[n][e]);
          }
      }
    }
    const float m = group_sum<L>(dot, lds) / (float)D * rstd * rstd;
    fvec out[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = lane + n * L, p = pack_at(i, VEC, D);
      out[n] = rstd * (d[n] * w[n] - s[n] * m);
      if (on && i < nvec && dsum) out[n] += load_pack<T, VEC>(dsum + row * D + p);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = lane + n * L;
      if (on && i < nvec) store_pack<T, VEC>(dx + row * D + pack_at(i, VEC, D), out[n]);
    }
  }
  const int slots = nvec * VEC;
  if (G == 1) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = lane + n * L;
      if (i < nvec) *reinterpret_cast<typename Pack<float, VEC>::loose*>(part + (int64_t)blockIdx.x * slots + i * VEC) = acc[n];
    }
    return;
  }
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int e = 0; e < VEC; ++e) share[(grp * L * NV + lane + n * L) * VEC + e] = acc[n][e];
  __syncthreads();
  for (int k = threadIdx.x; k < slots; k += 256) {
    float v = 0.f;
    for (int g = 0; g < G; ++g) v += share[g * L * NV * VEC + k];
    part[(int64_t)blockIdx.x * slots + k] = v;
  }
}

// The same for rows that do not fit: dweight's shares are added up in global memory, by the one workgroup and lane that owns the place.
template <typename T>
__global__ __launch_bounds__(1024) void norm_bwd_long(ope_norm_cfg c, const T* dy, const T* dsum, const T* __restrict__ s_in, const T* __restrict__ residual,
                                                      const T* __restrict__ weight, const float* __restrict__ rstd_in, T* dx, float* __restrict__ part) {
  __shared__ float lds[16];
  const int D = c.width;
  float* mine = part + (int64_t)blockIdx.x * D;
  auto at = [&](int64_t row, int d) { return (float)s_in[row * c.x_stride + d] + (residual ? (float)residual[row * c.residual_stride + d] : 0.f); };
  for (int d = threadIdx.x; d < D; d += 1024) mine[d] = 0.f;
  for (int64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const float rstd = rstd_in[row];
    float dot = 0.f;
    for (int d = threadIdx.x; d < D; d += 1024) dot = fmaf((float)dy[row * D + d] * (float)weight[d], at(row, d), dot);
    const float m = group_sum<1024>(dot, lds) / (float)D * rstd * rstd;
    for (int d = threadIdx.x; d < D; d += 1024) {
      const float g = (float)dy[row * D + d], s = at(row, d);
      mine[d] = fmaf(g, s * rstd, mine[d]);
      dx[row * D + d] = (T)(rstd * (g * (float)weight[d] - s * m) + (dsum ? (float)dsum[row * D + d] : 0.f));
    }
  }
}

// dweight[d] = sum over the shares, 16 runs of rows side by side and then in order.
template <typename T>
__global__ __launch_bounds__(1024) void norm_dweight(const float* __restrict__ part, int parts, int slots, int D, int VEC, T* __restrict__ dw) {
  __shared__ float lds[16][65];
  const int col = threadIdx.x & 63, run = threadIdx.x >> 6, d = blockIdx.x * 64 + col;
  float v = 0.f;
  if (d < D) {
    const int last = slots - VEC, slot = d < last ? d : last + d - (D - VEC);
#pragma unroll 8
    for (int r = run; r < parts; r += 16) v += part[(int64_t)r * slots + slot];
  }
  lds[run][col] = v;
  __syncthreads();
  if (run == 0 && d < D) {
    v = 0.f;
    for (int r = 0; r < 16; ++r) v += lds[r][col];
    dw[d] = (T)v;
  }
}

// The width's class: lanes a row and packs a lane; L = 0 is the walk over long rows.
struct NormShape { int VEC, L, NV, nvec; };
static NormShape norm_shape(int dtype, int D) {
  NormShape s;
  s.VEC = dtype == OPE_F32 ? 4 : 8;
  if (D < s.VEC) s.VEC = 1;
  s.nvec = (D + s.VEC - 1) / s.VEC;
  s.L = s.nvec <= 64 ? 16 : s.nvec <= 256 ? 64 : s.nvec <= 1024 ? 256 : s.nvec <= 4096 ? 1024 : 0;
  const int n = s.L ? ope_cdiv(s.nvec, s.L) : 0;
  s.NV = n <= 2 ? n : 4;
  return s;
}
constexpr int kNormParts = 512;     // shares of dweight: two workgroups of 256 lanes for every CU
static int norm_parts(const ope_norm_cfg* c) {
  const NormShape s = norm_shape(c->dtype, c->width);
  const int g = s.L == 0 || s.L > 256 ? 1 : 256 / s.L;
  const int64_t need = (c->rows + g - 1) / g;
  return (int)(need < kNormParts ? need : kNormParts);
}

// calls f with the compile-time L, NV of `s`
template <typename F>
static int with_shape(const NormShape& s, F f) {
#define OPE_NV(L)                                                                     \
  return s.NV == 1 ? f(std::integral_constant<int, L>{}, std::integral_constant<int, 1>{}) \
         : s.NV == 2 ? f(std::integral_constant<int, L>{}, std::integral_constant<int, 2>{}) : f(std::integral_constant<int, L>{}, std::integral_constant<int, 4>{})
  switch (s.L) {
    case 16: OPE_NV(16);
    case 64: OPE_NV(64);
    case 256: OPE_NV(256);
    case 1024: OPE_NV(1024);
  }
#undef OPE_NV
  return OPE_EINVAL;
}

static bool norm_ok(const ope_norm_cfg* c) {
  if (!c || c->rows < 0 || c->width < 1 || c->width > (1 << 20) || !elem_float(c->dtype) || c->x_stride < 0) return false;
  const NormShape s = norm_shape(c->dtype, c->width);
  const int lanes = s.L ? s.L : 1024;                  // of one row
  return c->rows < ((int64_t)1 << 31) && launch_fits(c->rows + 16, lanes);
}

template <bool NORM, bool OUT8>
static int launch_norm(const ope_norm_cfg* c, const void* x, const void* residual, const void* weight, void* y, float* scale, void* sum_out,
                       float* rstd, hipStream_t st) {
  if (c->rows == 0) return OPE_OK;
  const NormShape s = norm_shape(c->dtype, c->width);
  return with_elem(c->dtype, [&](auto t) {
    typedef decltype(t) T;
    constexpr int W = sizeof(T) == 4 ? 4 : 8;
    if (s.L == 0) {
      OPE_LAUNCH((norm_long<T, NORM, OUT8>), dim3((unsigned)c->rows), dim3(1024), 0, st, *c, (const T*)x, (const T*)residual, (const T*)weight, y, scale, (T*)sum_out, rstd);
      OPE_CHECK_LAUNCH();
      return OPE_OK;
    }
    if (s.VEC == 1) {
      OPE_LAUNCH((norm_rows<T, 1, 16, 1, NORM, OUT8>), dim3((unsigned)ope_cdiv(c->rows, 16)), dim3(256), 0, st, *c, (const T*)x, (const T*)residual, (const T*)weight, y, scale, (T*)sum_out, rstd);
      OPE_CHECK_LAUNCH();
      return OPE_OK;
    }
    return with_shape(s, [&](auto l, auto n) {
      constexpr int L = decltype(l)::value, NV = decltype(n)::value;
      const int g = L > 256 ? 1 : 256 / L;
      OPE_LAUNCH((norm_rows<T, W, L, NV, NORM, OUT8>), dim3((unsigned)ope_cdiv(c->rows, g)), dim3(L > 256 ? L : 256), 0, st, *c, (const T*)x, (const T*)residual, (const T*)weight, y, scale, (T*)sum_out, rstd);
      OPE_CHECK_LAUNCH();
      return OPE_OK;
    });
  });
}

}  // namespace ope
using namespace ope;

extern "C" int ope_rms_norm(const ope_norm_cfg* cfg, const void* x, const void* residual, const void* weight, void* y, float* scale, void* sum_out,
                            float* rstd, void* stream) {
  if (!norm_ok(cfg) || !(cfg->eps >= 0.f) || (residual && cfg->residual_stride < 0)) return OPE_EINVAL;
  if (cfg->out_dtype != cfg->dtype && cfg->out_dtype != OPE_E4M3) return OPE_EINVAL;
  const bool out8 = cfg->out_dtype == OPE_E4M3;
  if (cfg->rows && (!x || !weight || !y || (out8 && !scale))) return OPE_EINVAL;
  return out8 ? launch_norm<true, true>(cfg, x, residual, weight, y, scale, sum_out, rstd, (hipStream_t)stream)
              : launch_norm<true, false>(cfg, x, residual, weight, y, scale, sum_out, rstd, (hipStream_t)stream);
}

extern "C" int ope_quantize_rows(const ope_norm_cfg* cfg, const void* x, void* q, float* scale, void* stream) {
  if (!norm_ok(cfg) || (cfg->rows && (!x || !q || !scale))) return OPE_EINVAL;
  return launch_norm<false, true>(cfg, x, nullptr, nullptr, q, scale, nullptr, nullptr, (hipStream_t)stream);
}

extern "C" int64_t ope_rms_norm_backward_workspace_bytes(const ope_norm_cfg* cfg) {
  if (!norm_ok(cfg)) return OPE_EINVAL;
  const NormShape s = norm_shape(cfg->dtype, cfg->width);
  return (int64_t)norm_parts(cfg) * (s.L ? s.nvec * s.VEC : cfg->width) * 4;
}

extern "C" int ope_rms_norm_backward(const ope_norm_cfg* cfg, const void* dy, const void* dsum, const void* x, const void* residual, const void* weight,
                                     const float* rstd, void* dx, void* dweight, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = ope_rms_norm_backward_workspace_bytes(cfg);
  if (need < 0 || !dweight || (residual && cfg->residual_stride < 0)) return OPE_EINVAL;
  if (cfg->rows && (!dy || !x || !weight || !rstd || !dx || !workspace)) return OPE_EINVAL;
  if (workspace_bytes < need) return OPE_ENOSPC;
  const NormShape s = norm_shape(cfg->dtype, cfg->width);
  const int parts = norm_parts(cfg), D = cfg->width, slots = s.L ? s.nvec * s.VEC : D;
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  return with_elem(cfg->dtype, [&](auto t) {
    typedef decltype(t) T;
    constexpr int W = sizeof(T) == 4 ? 4 : 8;
    if (parts) {
      int rc = OPE_OK;
      if (s.L == 0)
        OPE_LAUNCH((norm_bwd_long<T>), dim3(parts), dim3(1024), 0, st, *cfg, (const T*)dy, (const T*)dsum, (const T*)x, (const T*)residual, (const T*)weight, rstd, (T*)dx, part);
      else if (s.VEC == 1)
        OPE_LAUNCH((norm_bwd<T, 1, 16, 1>), dim3(parts), dim3(256), 0, st, *cfg, (const T*)dy, (const T*)dsum, (const T*)x, (const T*)residual, (const T*)weight, rstd, (T*)dx, part);
      else
        rc = with_shape(s, [&](auto l, auto n) {
          constexpr int L = decltype(l)::value, NV = decltype(n)::value;
          OPE_LAUNCH((norm_bwd<T, W, L, NV>), dim3(parts), dim3(L > 256 ? L : 256), 0, st, *cfg, (const T*)dy, (const T*)dsum, (const T*)x, (const T*)residual, (const T*)weight, rstd, (T*)dx, part);
          return OPE_OK;
        });
      if (rc) return rc;
      OPE_CHECK_LAUNCH();
    }
    OPE_LAUNCH((norm_dweight<T>), dim3(ope_cdiv(D, 64)), dim3(1024), 0, st, part, parts, slots, D, s.L ? s.VEC : 1, (T*)dweight);
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  });
}
