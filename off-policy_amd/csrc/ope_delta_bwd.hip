// Gated delta rule, gradients (ope_delta_backward, ope.h). With P = scale tril(q k^T decay), d_i the decay from i to the chunk's end, S the
// state in front of a chunk and dS' the gradient of the one behind it:
//   dU = P^T dO + diag(d) k dS';   dS = e^G_63 dS' + scale (e^G q)^T dO - W^T dU;   dR = (I + A)^-T dU  (R = beta (v - e^G k S))
//   dv = beta dR;  dP = dO U^T;  dA = -dR U^T (strictly lower)
//   dq = scale e^G dO S^T + (dP scale decay) k
//   dk = -beta e^G dR S^T + (dA beta decay) k + (dA beta decay)^T k + (dP scale decay)^T q + diag(d) U dS'^T
//   dbeta_t = dR_t.v_t + k_t.(-e^G dR S^T + (dA decay) k)_t
//   dG_t = q_t.dq_t + k_t.(the first two terms of dk_t) - k_t.(the last three), dG_63 += sum_t k_t.(last term of dk_t) + e^G_63 <dS', S>;
//   dg is the sum of dG from t to the end of t's segment of the chunk: no sum reaches over a reset or over more than one chunk.
//
//   delta_bwd_prep  parallel over chunks: P^T dO, N = scale (e^G q)^T dO, diag(d) k
//   delta_scan      (ope_delta.hip) serial over chunks, backwards: dU and dS'
//   delta_bwd_main  parallel over chunks: the rest
//   delta_heads     sum over the value heads that share a query / key head
#include "ope_delta.h"

namespace ope {

int launch_delta_scan(const DeltaDims& d, bool bwd, const int32_t* lengths, const float* M1, const float* M2, float* UT, float* ST, const float* gC,
                      const float* first, float* last, hipStream_t st);
void delta_saved(const DeltaDims& d, float* saved, float** ST, float** UT, float** WT, float** gC);
__global__ void delta_keep_state(const float* __restrict__ from, float* __restrict__ to, int64_t n);

template <typename T, int KT>
__global__ __launch_bounds__(256) void delta_bwd_prep(ope_delta_cfg cfg, DeltaDims d, const T* __restrict__ q_in, const T* __restrict__ k_in,
                                                      const float* __restrict__ g_in, const float* __restrict__ beta_in, const int32_t* __restrict__ lengths,
                                                      const T* __restrict__ dO, float* __restrict__ Kd, float* __restrict__ dUT, float* __restrict__ dST) {
  constexpr int Kp = 16 * KT;
  __shared__ float q[kC][Kp + 4], k[kC][Kp + 4], PT[kC][kC + 4];
  __shared__ Gates gt;
  const ChunkAt a = chunk_at(d, lengths, blockIdx.x);
  if (a.nv == 0) return;
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  if (w == 0) load_gates(gt, cfg, a, g_in, beta_in);
  const int hk = a.h / (d.H / d.Hk);
  load_rows<T, KT>(q, q_in, cfg.q_stride, a, hk, d.K);
  load_rows<T, KT>(k, k_in, cfg.k_stride, a, hk, d.K);
  __syncthreads();
  for (int x = threadIdx.x; x < kC * KT * 4; x += 256) {
    const int t = x / (KT * 4), f = (x % (KT * 4)) * 4;
    put4(&Kd[(a.c * kC + t) * Kp + f], at4(&k[t][f]) * gt.tail[t]);
  }
  const int s = 16 * w + j;
  for (int it = w; it < 4; ++it) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KT; ++c) acc = mfma4(at4(&q[16 * it + j][16 * c + 4 * g]), at4(&k[s][16 * c + 4 * g]), acc);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * it + 4 * g + r;
      acc[r] = t >= s ? cfg.scale * decay(gt, t, s) * acc[r] : 0.f;
    }
    put4(&PT[s][16 * it + 4 * g], acc);
  }
  __syncthreads();
  const T* o0 = dO + a.b * cfg.o_stride[0] + (int64_t)a.t0 * cfg.o_stride[1] + a.h * cfg.o_stride[2];
  for (int vt = w; vt < d.VT; vt += 4) {
    const int v = 16 * vt + j;
    f32x4 x[4], y[4];
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * it + 4 * g + r;
        x[it][r] = t < a.nv && v < d.V ? (float)o0[(int64_t)t * cfg.o_stride[1] + v] : 0.f;
        y[it][r] = x[it][r] * cfg.scale * gt.head[t];
      }
#pragma unroll
    for (int is = 0; is < 4; ++is) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int it = is; it < 4; ++it) acc = mfma4(at4(&PT[16 * is + j][16 * it + 4 * g]), x[it], acc);
      put4(&dUT[(a.c * d.Vp + v) * kC + 16 * is + 4 * g], acc);
    }
    for (int kt = 0; kt < KT; ++kt) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int it = 0; it < 4; ++it) acc = mfma4(col4(&q[16 * it + 4 * g][16 * kt + j], Kp + 4), y[it], acc);
      put4(&dST[(a.c * d.Vp + v) * Kp + 16 * kt + 4 * g], acc);
    }
  }
}

// Wave w owns the tokens 16w.. as data rows; the three products over the value columns keep 3 * KT accumulators in registers, so S, dS' and U
// are read once a wave. One workgroup a CU at Kp = 128 (130 KB of LDS).
template <typename T, int KT>
__global__ __launch_bounds__(256) void delta_bwd_main(ope_delta_cfg cfg, DeltaDims d, const T* __restrict__ q_in, const T* __restrict__ k_in,
                                                      const T* __restrict__ v_in, const float* __restrict__ g_in, const float* __restrict__ beta_in,
                                                      const int32_t* __restrict__ lengths, const float* __restrict__ ST, const float* __restrict__ UT,
                                                      const T* __restrict__ dO, float* dUT, const float* __restrict__ dST, T* __restrict__ dq,
                                                      T* __restrict__ dk, float* __restrict__ dqp, float* __restrict__ dkp, T* __restrict__ dv,
                                                      float* __restrict__ dg, float* __restrict__ dbeta) {
  constexpr int Kp = 16 * KT;
  __shared__ float q[kC][Kp + 4], k[kC][Kp + 4], NA[kC][kC + 4], inv[4][16][20], dPs[kC][kC + 4], dAs[kC][kC + 4];
  __shared__ float dbv[4][kC], dG[kC], dEnd[kC], dots[4];
  __shared__ Gates gt;
  const ChunkAt a = chunk_at(d, lengths, blockIdx.x);
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int rows = min(d.T - a.t0, kC), hk = a.h / (d.H / d.Hk);
  const bool own = d.H == d.Hk;
  T* dv0 = dv + a.b * cfg.dv_stride[0] + (int64_t)a.t0 * cfg.dv_stride[1] + a.h * cfg.dv_stride[2];
  float* dg0 = dg + a.b * cfg.dg_stride[0] + (int64_t)a.t0 * cfg.dg_stride[1] + a.h * cfg.dg_stride[2];
  float* db0 = dbeta + a.b * cfg.dbeta_stride[0] + (int64_t)a.t0 * cfg.dbeta_stride[1] + a.h * cfg.dbeta_stride[2];
  // four elements of dq / dk at (t, f): of the type itself, or this value head's float32 share
  auto put_k = [&](T* out, const int64_t* stride, float* share, int t, int f, f32x4 x) {
    if (t >= rows) return;
    if (own) {
      T* p = out + a.b * stride[0] + (int64_t)(a.t0 + t) * stride[1] + hk * stride[2] + f;
      if (f + 4 <= d.K) store_pack<T, 4>(p, x);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (f + e < d.K) p[e] = (T)x[e];
    } else {
      float* p = share + (((int64_t)a.b * d.T + a.t0 + t) * d.H + a.h) * d.K + f;
      if (f + 4 <= d.K) store_pack<float, 4>(p, x);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (f + e < d.K) p[e] = x[e];
    }
  };
  if (a.nv == 0) {
    for (int x = threadIdx.x; x < rows * d.V; x += 256) dv0[(int64_t)(x / d.V) * cfg.dv_stride[1] + x % d.V] = (T)0.f;
    for (int x = threadIdx.x; x < kC * KT * 4; x += 256) {
      const int t = x / (KT * 4), f = (x % (KT * 4)) * 4;
      put_k(dq, cfg.dq_stride, dqp, t, f, f32x4{0.f, 0.f, 0.f, 0.f});
      put_k(dk, cfg.dk_stride, dkp, t, f, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    if (threadIdx.x < rows) {
      dg0[threadIdx.x * cfg.dg_stride[1]] = 0.f;
      db0[threadIdx.x * cfg.dbeta_stride[1]] = 0.f;
    }
    return;
  }
  if (w == 0) load_gates(gt, cfg, a, g_in, beta_in);
  load_rows<T, KT>(q, q_in, cfg.q_stride, a, hk, d.K);
  load_rows<T, KT>(k, k_in, cfg.k_stride, a, hk, d.K);
  __syncthreads();
  minus_A<KT>(NA, k, gt);
  __syncthreads();
  if (w == 0) diag_inverse(inv, NA);
  __syncthreads();
  // dR = (I + A)^-T dU, block backward substitution, 16 value columns a wave at a time; dv; the part of dbeta that v gives
  {
    const T* v0 = v_in + a.b * cfg.v_stride[0] + (int64_t)a.t0 * cfg.v_stride[1] + a.h * cfg.v_stride[2];
    f32x4 part[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) part[it] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int vt = w; vt < d.VT; vt += 4) {
      const int v = 16 * vt + j;
      f32x4 x[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) x[it] = at4(&dUT[(a.c * d.Vp + v) * kC + 16 * it + 4 * g]);
#pragma unroll
      for (int it = 3; it >= 0; --it) {
        f32x4 acc = x[it];
#pragma unroll
        for (int kt = it + 1; kt < 4; ++kt) acc = mfma4(col4(&NA[16 * kt + 4 * g][16 * it + j], kC + 4), x[kt], acc);
        x[it] = mfma4(col4(&inv[it][4 * g][j], 20), acc, f32x4{0.f, 0.f, 0.f, 0.f});
        put4(&dUT[(a.c * d.Vp + v) * kC + 16 * it + 4 * g], x[it]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = 16 * it + 4 * g + r;
          if (t < rows && v < d.V) dv0[(int64_t)t * cfg.dv_stride[1] + v] = (T)(t < a.nv ? gt.beta[t] * x[it][r] : 0.f);
          if (t < a.nv && v < d.V) part[it][r] = fmaf(x[it][r], (float)v0[(int64_t)t * cfg.v_stride[1] + v], part[it][r]);
        }
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = row16_sum(part[it][r]);
        if (j == 0) dbv[w][16 * it + 4 * g + r] = x;
      }
  }
  __syncthreads();     // dR of all columns is in dUT
  const int t = 16 * w + j;
  f32x4 X1[KT], X2[KT], X3[KT], P[4], A[4];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) X1[kt] = X2[kt] = X3[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int is = 0; is < 4; ++is) P[is] = A[is] = f32x4{0.f, 0.f, 0.f, 0.f};
  float dot = 0.f;
  const T* o0 = dO + a.b * cfg.o_stride[0] + (int64_t)(a.t0 + t) * cfg.o_stride[1] + a.h * cfg.o_stride[2];
  for (int vt = 0; vt < d.VT; ++vt) {
    const int v = 16 * vt + 4 * g;
    f32x4 bo = {0.f, 0.f, 0.f, 0.f};
    if (t < a.nv) {
      if (v + 4 <= d.V) bo = load_pack<T, 4>(o0 + v);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v + e < d.V) bo[e] = (float)o0[v + e];
    }
    const float* S0 = ST + (a.c * d.Vp + v) * Kp + j;
    const float* D0 = dST + (a.c * d.Vp + v) * Kp + j;
    const float* U0 = UT + (a.c * d.Vp + v) * kC + j;
    const f32x4 br = col4(dUT + (a.c * d.Vp + v) * kC + t, kC), bu = col4(U0 + 16 * w, kC);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const f32x4 s = col4(S0 + 16 * kt, Kp), ds = col4(D0 + 16 * kt, Kp);
      X1[kt] = mfma4(s, bo, X1[kt]);
      X2[kt] = mfma4(s, br, X2[kt]);
      X3[kt] = mfma4(ds, bu, X3[kt]);
      if ((kt & 3) == w) dot += s[0] * ds[0] + s[1] * ds[1] + s[2] * ds[2] + s[3] * ds[3];
    }
#pragma unroll
    for (int is = 0; is < 4; ++is)
      if (is <= w) {
        const f32x4 u = col4(U0 + 16 * is, kC);
        P[is] = mfma4(u, bo, P[is]);
        A[is] = mfma4(u, br, A[is]);
      }
  }
  dot = rowsum4(row16_sum(dot));
  if ((threadIdx.x & 63) == 0) dots[w] = dot;
#pragma unroll
  for (int is = 0; is < 4; ++is) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int s = 16 * is + 4 * g + r;
      const float dec = s <= t ? decay(gt, t, s) : 0.f;
      P[is][r] = P[is][r] * cfg.scale * dec;
      A[is][r] = s < t ? -A[is][r] * dec : 0.f;
    }
    put4(&dPs[t][16 * is + 4 * g], P[is]);
    put4(&dAs[t][16 * is + 4 * g], A[is] * gt.beta[t]);
  }
  const float fq = cfg.scale * gt.head[t], fr = gt.head[t];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    X1[kt] *= fq;
    X2[kt] *= -fr;
#pragma unroll
    for (int is = 0; is < 4; ++is)
      if (is <= w) {
        const f32x4 kc = col4(&k[16 * is + 4 * g][16 * kt + j], Kp + 4);
        X1[kt] = mfma4(kc, P[is], X1[kt]);        // dq
        X2[kt] = mfma4(kc, A[is], X2[kt]);        // the terms of dk that carry beta_t, without it
      }
  }
  __syncthreads();
  float pq = 0.f, pr = 0.f, pc = 0.f, ps = 0.f;
  const float bt = gt.beta[t], tail = gt.tail[t];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
    for (int it = w; it < 4; ++it) {
      c = mfma4(col4(&q[16 * it + 4 * g][16 * kt + j], Kp + 4), col4(&dPs[16 * it + 4 * g][t], kC + 4), c);
      c = mfma4(col4(&k[16 * it + 4 * g][16 * kt + j], Kp + 4), col4(&dAs[16 * it + 4 * g][t], kC + 4), c);
    }
    const int f = 16 * kt + 4 * g;
    const f32x4 kv = at4(&k[t][f]), qv = at4(&q[t][f]), e = X3[kt] * tail;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      pq = fmaf(qv[r], X1[kt][r], pq);
      pr = fmaf(kv[r], X2[kt][r], pr);
      pc = fmaf(kv[r], c[r], pc);
      ps = fmaf(kv[r], e[r], ps);
    }
    put_k(dq, cfg.dq_stride, dqp, t, f, X1[kt]);
    put_k(dk, cfg.dk_stride, dkp, t, f, X2[kt] * bt + c + e);
  }
  pq = rowsum4(pq); pr = rowsum4(pr); pc = rowsum4(pc); ps = rowsum4(ps);
  if (g == 0) {
    dG[t] = pq + bt * pr - pc - ps;
    dEnd[t] = ps;
    if (t < rows) db0[(int64_t)t * cfg.dbeta_stride[1]] = t < a.nv ? pr + dbv[0][t] + dbv[1][t] + dbv[2][t] + dbv[3][t] : 0.f;
  }
  __syncthreads();
  if (w == 0) {
    const int l = threadIdx.x, seg = gt.seg[l];
    double x = dG[l], end = dEnd[l];
    for (int m = 1; m < 64; m <<= 1) {
      const double o = __shfl_down(x, m, 64);
      const int so = __shfl_down(seg, m, 64);
      if (l + m < 64 && so == seg) x += o;
      end += __shfl_xor(end, m, 64);
    }
    end += (double)gt.whole * ((double)dots[0] + dots[1] + dots[2] + dots[3]);
    if (seg == gt.seg[63]) x += end;
    const bool cut = seg != (l > 0 ? gt.seg[l - 1] : 0);       // g = -inf here
    if (l < rows) dg0[(int64_t)l * cfg.dg_stride[1]] = l < a.nv && !cut ? (float)x : 0.f;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void delta_heads(ope_delta_cfg cfg, DeltaDims d, const float* __restrict__ dqp, const float* __restrict__ dkp,
                                                   T* __restrict__ dq, T* __restrict__ dk) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / d.K;       // row: (b, t, hk)
  if (row >= (int64_t)d.B * d.T * d.Hk) return;
  const int f = (int)(i % d.K), hk = (int)(row % d.Hk), r = d.H / d.Hk;
  const int64_t bt = row / d.Hk, b = bt / d.T, t = bt % d.T;
  const int64_t from = (bt * d.H + (int64_t)hk * r) * d.K + f;
  float x = 0.f, y = 0.f;
  for (int h = 0; h < r; ++h) {
    x += dqp[from + (int64_t)h * d.K];
    y += dkp[from + (int64_t)h * d.K];
  }
  dq[b * cfg.dq_stride[0] + t * cfg.dq_stride[1] + hk * cfg.dq_stride[2] + f] = (T)x;
  dk[b * cfg.dk_stride[0] + t * cfg.dk_stride[1] + hk * cfg.dk_stride[2] + f] = (T)y;
}

}  // namespace ope
using namespace ope;

extern "C" int ope_delta_backward(const ope_delta_cfg* cfg, const void* q, const void* k, const void* v, const float* g, const float* beta,
                                  const int32_t* lengths, const void* saved, int64_t saved_bytes, const void* d_o, const float* d_state, void* dq,
                                  void* dk, void* dv, float* dg, float* dbeta, float* d_state0, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!delta_ok(cfg)) return OPE_EINVAL;
  const DeltaDims d = delta_dims(cfg);
  hipStream_t st = (hipStream_t)stream;
  if (d.B == 0) return OPE_OK;
  if (d.T == 0) {
    const int64_t n = (int64_t)d.B * d.H * d.K * d.V;
    if (!d_state0) return OPE_OK;
    OPE_LAUNCH(delta_keep_state, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, d_state, d_state0, n);
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  }
  if (!q || !k || !v || !g || !beta || !saved || !d_o || !dq || !dk || !dv || !dg || !dbeta || !workspace) return OPE_EINVAL;
  if (saved_bytes < ope_delta_saved_bytes(cfg) || workspace_bytes < ope_delta_workspace_bytes(cfg, 1)) return OPE_ENOSPC;
  float *ST, *UT, *WT, *gC;
  delta_saved(d, (float*)saved, &ST, &UT, &WT, &gC);
  float* Kd = (float*)workspace;
  float* dUT = Kd + d.chunks * kC * d.Kp;
  float* dST = dUT + d.chunks * d.Vp * kC;
  float* dqp = dST + d.chunks * d.Vp * d.Kp;
  float* dkp = dqp + (int64_t)d.B * d.T * d.H * d.K;
  return with_elem(cfg->dtype, [&](auto t) {
    typedef decltype(t) T;
    const dim3 grid((unsigned)d.chunks);
#define OPE_BPREP(KT) \
  case KT: OPE_LAUNCH((delta_bwd_prep<T, KT>), grid, dim3(256), 0, st, *cfg, d, (const T*)q, (const T*)k, g, beta, lengths, (const T*)d_o, Kd, dUT, dST); break
    switch (d.KT) { OPE_BPREP(1); OPE_BPREP(2); OPE_BPREP(4); OPE_BPREP(8); }
#undef OPE_BPREP
    OPE_CHECK_LAUNCH();
    const int rc = launch_delta_scan(d, true, lengths, Kd, WT, dUT, dST, gC, d_state, d_state0, st);
    if (rc) return rc;
#define OPE_BMAIN(KT)                                                                                                                                  \
  case KT: OPE_LAUNCH((delta_bwd_main<T, KT>), grid, dim3(256), 0, st, *cfg, d, (const T*)q, (const T*)k, (const T*)v, g, beta, lengths, ST, UT,        \
                      (const T*)d_o, dUT, dST, (T*)dq, (T*)dk, dqp, dkp, (T*)dv, dg, dbeta); break
    switch (d.KT) { OPE_BMAIN(1); OPE_BMAIN(2); OPE_BMAIN(4); OPE_BMAIN(8); }
#undef OPE_BMAIN
    OPE_CHECK_LAUNCH();
    if (d.H != d.Hk) {
      const int64_t n = (int64_t)d.B * d.T * d.Hk * d.K;
      OPE_LAUNCH((delta_heads<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, *cfg, d, dqp, dkp, (T*)dq, (T*)dk);
      OPE_CHECK_LAUNCH();
    }
    return OPE_OK;
  });
}
