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

int launch_delta_scan(int dtype, const DeltaDims& d, bool bwd, const int32_t* lengths, const void* M1, const void* M2, float* UT, float* ST,
                      const float* gC, const float* tails, const float* first, float* last, hipStream_t st);
int64_t delta_saved(const DeltaDims& d, float* saved, float** ST, float** UT, float** WT, float** gC, float** tails);
__global__ void delta_keep_state(const float* __restrict__ from, float* __restrict__ to, int64_t n);

template <typename T, int KT>
__global__ __launch_bounds__(64 * chunk_waves<KT>(), KT >= 4 ? 4 : 3) void delta_bwd_prep(
    ope_delta_cfg cfg, DeltaDims d, const T* __restrict__ q_in, const T* __restrict__ k_in, const float* __restrict__ g_in, const float* __restrict__ beta_in,
    const int32_t* __restrict__ lengths, const T* __restrict__ dO, T* __restrict__ Ks, float* __restrict__ dUT, float* __restrict__ dST) {
  constexpr int NW = chunk_waves<KT>(), RS = Rows<T, KT>::kStride, kPair = KT % 2 ? 1 : 2;
  __shared__ Rows<T, KT> q, k;
  __shared__ float PT[kC][kC + 4];
  __shared__ Gates gt;
  const ChunkAt a = chunk_at(d, lengths, blockIdx.x);
  if (a.nv == 0) return;
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  if (w == 0) load_gates(gt, cfg, a, g_in, beta_in);
  const int hk = a.h / (d.H / d.Hk);
  load_rows<T, KT, 64 * NW>(q, q_in, cfg.q_stride, a, hk, d.K);
  load_rows<T, KT, 64 * NW>(k, k_in, cfg.k_stride, a, hk, d.K);
  __syncthreads();
  for (int x = w; x < 4 * KT; x += NW)                   // k, a tile a wave
    *reinterpret_cast<typename Pack<T, 4>::vec*>(Ks + (a.c * 4 * KT + x) * 256 + tile_lane()) =
        *reinterpret_cast<const typename Pack<T, 4>::vec*>(&k.v[16 * (x / KT) + j][16 * (x % KT) + 4 * g]);
  for (int x = w; x < 10; x += NW) {
    int it, is;
    lower_tile(x, it, is);
    const int s = 16 * is + j;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KT; ++c) acc = dot4(&q.v[16 * it + j][16 * c + 4 * g], &k.v[s][16 * c + 4 * g], acc);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * it + 4 * g + r;
      const float dec = t >= s ? decay(gt, t, s) : 0.f;
      acc[r] = dec == 0.f ? 0.f : cfg.scale * dec * acc[r];
    }
    put4(&PT[s][16 * it + 4 * g], acc);
  }
  __syncthreads();
  const int last = gt.last();
  for (int vt = w; vt < d.VT; vt += NW) {
    const int v = 16 * vt + j;
    f32x4 x[4];
    load_columns(x, dO, cfg.o_stride, a, v, d.V);
#pragma unroll
    for (int is = 0; is < 4; ++is) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int it = is; it < 4; ++it) acc = mfma4(at4(&PT[16 * is + j][16 * it + 4 * g]), x[it], acc);
      if (last && __any(!finite(acc))) {                // one segment at a time
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int s = gt.first(); s <= last; ++s) {
          f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int it = is; it < 4; ++it) part = mfma4(at4(&PT[16 * is + j][16 * it + 4 * g]), only(gt, s, 16 * it + 4 * g, x[it]), part);
          acc += only(gt, s, 16 * is + 4 * g, part);
        }
      }
      put4(&dUT[((a.c * d.VT + vt) * 4 + is) * 256 + tile_lane()], acc);
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) x[it] = gated(at4(&gt.head[16 * it + 4 * g]) * cfg.scale, x[it]);
#pragma unroll kPair                                     // (all of an odd number of tiles would be unrolled, into scratch memory)
    for (int kt = 0; kt < KT; ++kt) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int it = 0; it < 4; ++it) acc = mfma4(column4(&q.v[16 * it + 4 * g][16 * kt + j], RS), x[it], acc);
      if (last && __any(!finite(acc))) {                // nothing of the tokens behind a reset
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int it = 0; it < 4; ++it) acc = mfma4(only(gt, 0, 16 * it + 4 * g, column4(&q.v[16 * it + 4 * g][16 * kt + j], RS)), x[it], acc);
      }
      put4(&dST[((a.c * d.VT + vt) * KT + kt) * 256 + tile_lane()], acc);
    }
  }
}

// Eight waves: wave w owns the tokens 16 (w & 3).. as data rows and one half (w >> 2) of the key tiles, so the three products over the value
// columns keep 3 * KT / 2 accumulators in registers. The first half makes dP, the second dA; they change hands through LDS.
template <typename T, int KT>
__global__ __launch_bounds__(512, KT * sizeof(T) > 16 ? 2 : 4) void delta_bwd_main(ope_delta_cfg cfg, DeltaDims d, const T* __restrict__ q_in, const T* __restrict__ k_in,
                                                      const T* __restrict__ v_in, const float* __restrict__ g_in, const float* __restrict__ beta_in,
                                                      const int32_t* __restrict__ lengths, const float* __restrict__ ST, const float* __restrict__ UT,
                                                      const T* __restrict__ dO, float* dUT, const float* __restrict__ dST, T* __restrict__ dq,
                                                      T* __restrict__ dk, float* __restrict__ dqp, float* __restrict__ dkp, T* __restrict__ dv,
                                                      float* __restrict__ dg, float* __restrict__ dbeta) {
  constexpr int RS = Rows<T, KT>::kStride, KH = (KT + 1) / 2;      // KH: key tiles of a half
  __shared__ Rows<T, KT> q, k;
  // One pool, three lives: A and the diagonal's inverses for the solve; the tiles of S, dS' and U of 16 columns (rows of 20 floats: stores of whole
  // lanes and reads along columns both spread over the banks); dP and dA.
  constexpr int kTiles = 2 * KT + 4, kTile = 16 * 20, kPool = 2 * kC * (kC + 4) + 4 * 16 * 20;
  static_assert(kTiles * kTile <= kPool, "LDS pool");
  __shared__ float pool[kPool];
  float(*NA)[kC + 4] = reinterpret_cast<float(*)[kC + 4]>(pool);
  float(*dPs)[kC + 4] = NA;
  float(*dAs)[kC + 4] = reinterpret_cast<float(*)[kC + 4]>(pool + kC * (kC + 4));
  float(*inv)[16][20] = reinterpret_cast<float(*)[16][20]>(pool + 2 * kC * (kC + 4));
  __shared__ float dbv[2][kC], sums[2][4][kC], dots[8];
  __shared__ Gates gt;
  __shared__ unsigned long long odd;                   // segments that hold a key or query that is not finite, counted from the first token's
  const ChunkAt a = chunk_at(d, lengths, blockIdx.x);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int rows = min(d.T - a.t0, kC), hk = a.h / (d.H / d.Hk);
  const bool own = d.H == d.Hk;
  T* dv0 = dv + a.b * cfg.dv_stride[0] + (int64_t)a.t0 * cfg.dv_stride[1] + a.h * cfg.dv_stride[2];
  float* dg0 = dg + a.b * cfg.dg_stride[0] + (int64_t)a.t0 * cfg.dg_stride[1] + a.h * cfg.dg_stride[2];
  float* db0 = dbeta + a.b * cfg.dbeta_stride[0] + (int64_t)a.t0 * cfg.dbeta_stride[1] + a.h * cfg.dbeta_stride[2];
  // four elements of dq / dk at (t, f): of the type itself, or this value head's float32 share. 0 behind the last live token: what was computed there is
  // 0 times a state, which need not be finite.
  auto put_k = [&](T* out, const int64_t* stride, float* share, int t, int f, f32x4 x) {
    if (t >= rows) return;
    if (t >= a.nv) x = f32x4{0.f, 0.f, 0.f, 0.f};
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
    for (int x = threadIdx.x; x < rows * d.V; x += 512) dv0[(int64_t)(x / d.V) * cfg.dv_stride[1] + x % d.V] = (T)0.f;
    for (int x = threadIdx.x; x < kC * KT * 4; x += 512) {
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
  load_rows<T, KT, 512>(q, q_in, cfg.q_stride, a, hk, d.K);
  load_rows<T, KT, 512>(k, k_in, cfg.k_stride, a, hk, d.K);
  if (threadIdx.x == 0) odd = 0;
  __syncthreads();
  minus_A<T, KT>(NA, k, gt);
  const int last_seg = gt.last();
  const int first_seg = gt.first();
  auto each4 = [&](auto f) {                           // four elements of q and k at (t, f), threads side by side
    for (int x = threadIdx.x; x < kC * KT * 4; x += 512) f(x / (KT * 4), (x % (KT * 4)) * 4);
  };
  if (last_seg)
    each4([&](int t, int f) {
      bool fine = true;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (float)q.v[t][f + e], y = (float)k.v[t][f + e];
        fine &= x - x == 0.f && y - y == 0.f;
      }
      if (!fine) atomicOr(&odd, 1ull << (gt.seg[t] - first_seg));
    });
  __syncthreads();
  if (w == 0) diag_inverse(inv, NA, gt);
  if (odd)                                             // A has them; the products over the chunk's tokens below go without (poison)
    each4([&](int t, int f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (float)q.v[t][f + e], y = (float)k.v[t][f + e];
        if (x - x != 0.f) q.v[t][f + e] = (T)0.f;
        if (y - y != 0.f) k.v[t][f + e] = (T)0.f;
      }
    });
  __syncthreads();
  // dR = (I + A)^-T dU, block backward substitution, 16 value columns a wave at a time; left in dUT with its tiles transposed
  auto solve = [&](f32x4* x, auto apart, int seg) {    // as in delta_prep
#pragma unroll
    for (int it = 3; it >= 0; --it) {
      f32x4 acc = x[it];
#pragma unroll
      for (int kt = it + 1; kt < 4; ++kt) acc = mfma4(col4(&NA[16 * kt + 4 * g][16 * it + j], kC + 4), x[kt], acc);
      if (apart()) acc = only(gt, seg, 16 * it + 4 * g, acc);
      x[it] = mfma4(col4(&inv[it][4 * g][j], 20), acc, f32x4{0.f, 0.f, 0.f, 0.f});
      if (apart()) x[it] = only(gt, seg, 16 * it + 4 * g, x[it]);
    }
  };
  for (int vt = w; vt < d.VT; vt += 8) {
    float* at = dUT + (a.c * d.VT + vt) * 4 * 256;
    f32x4 x[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) x[it] = at4(at + it * 256 + tile_lane());
    solve(x, std::false_type{}, 0);
    if (last_seg && __any(!finite<4>(x))) {
      f32x4 b[4], y[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        b[it] = at4(at + it * 256 + tile_lane());
        x[it] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll 1
      for (int s = gt.first(); s <= last_seg; ++s) {
#pragma unroll
        for (int it = 0; it < 4; ++it) y[it] = only(gt, s, 16 * it + 4 * g, b[it]);
        solve(y, std::true_type{}, s);
#pragma unroll
        for (int it = 0; it < 4; ++it) x[it] += y[it];
      }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it) put4(at + it * 256 + turned_lane(), turn4(x[it]));
  }
  __syncthreads();     // dR of all columns is in dUT; A is done with
  const int wt = __builtin_amdgcn_readfirstlane(w & 3), half = __builtin_amdgcn_readfirstlane(w >> 2), k0 = half * KH, t = 16 * wt + j;
  f32x4 X1[KH], X2[KH], X3[KH], M[4];
#pragma unroll
  for (int q = 0; q < KH; ++q) X1[q] = X2[q] = X3[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int is = 0; is < 4; ++is) M[is] = f32x4{0.f, 0.f, 0.f, 0.f};
  float dot = 0.f, rv = 0.f;                          // <dS', S> and dR.v of the tiles this wave counts
  const T* o0 = dO + a.b * cfg.o_stride[0] + (int64_t)(a.t0 + t) * cfg.o_stride[1] + a.h * cfg.o_stride[2];
  const T* v0 = v_in + a.b * cfg.v_stride[0] + (int64_t)(a.t0 + t) * cfg.v_stride[1] + a.h * cfg.v_stride[2];
  // four values of a row from column v on; nothing is read past the row's end or behind the last live token
  const int back = t - min(t, a.nv - 1);              // a token that is not live reads the last live one's row
  auto value4 = [&](const T* row, int64_t stride, int v) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (d.V == d.Vp) {
      const f32x4 y = load_pack<T, 4>(row - back * stride + v);
      x = back ? x : y;
    } else if (t < a.nv) {
      if (v + 4 <= d.V) x = load_pack<T, 4>(row + v);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v + e < d.V) x[e] = (float)row[v + e];
    }
    return x;
  };
  // The tiles of 16 columns reach LDS once (each wave loads its share of the next ones while these are multiplied) and are read from there
  // transposed: 334 us at 4 x 4096 x 8 x 128 x 128. Loaded by the waves that multiply them, four times over, they kept the L2 at 7 TB/s: 420 us.
  constexpr int kShare = (kTiles + 7) / 8;
  f32x4 pre[kShare], br, bo;
  const int64_t first = a.c * d.VT;
  auto fetch = [&](int vt) {                           // past the end: the last columns again
    const int64_t at = first + min(vt, d.VT - 1);
    const int v = 16 * min(vt, d.VT - 1) + 4 * g;
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
      const int x = min(w + 8 * i, kTiles - 1);
      const float* p = x < KT ? ST + (at * KT + x) * 256 : (x < 2 * KT ? dST + (at * KT + x - KT) * 256 : UT + (at * 4 + x - 2 * KT) * 256);
      pre[i] = at4(p + tile_lane());
    }
    br = at4(dUT + (at * 4 + wt) * 256 + tile_lane());
    bo = value4(o0, cfg.o_stride[1], v);
  };
  auto tile = [&](int x) { return col4(&pool[x * kTile + 4 * g * 20 + j], 20); };
  fetch(0);
  for (int vt = 0; vt < d.VT; ++vt) {
    const int v = 16 * vt + 4 * g;
#pragma unroll
    for (int i = 0; i < kShare; ++i)
      if (w + 8 * i < kTiles) put4(&pool[(w + 8 * i) * kTile + j * 20 + 4 * g], pre[i]);
    const f32x4 r = br, o = bo, x = value4(v0, cfg.v_stride[1], v);
    lds_barrier();
    fetch(vt + 1);
    const f32x4 bu = tile(2 * KT + wt), bm = half ? r : o;
#pragma unroll
    for (int q = 0; q < KH; ++q)
      if (KT % 2 == 0 || k0 + q < KT) {
        const f32x4 st = tile(k0 + q), dt = tile(KT + k0 + q);
        X1[q] = mfma4(st, o, X1[q]);
        X2[q] = mfma4(st, r, X2[q]);
        X3[q] = mfma4(dt, bu, X3[q]);
        if ((q & 3) == wt) dot += st[0] * dt[0] + st[1] * dt[1] + st[2] * dt[2] + st[3] * dt[3];
        if (q & 1) __builtin_amdgcn_sched_barrier(0);  // no more tiles in registers than two pairs: 128 are what two workgroups a CU leave
      }
#pragma unroll
    for (int is = 0; is < 4; ++is)
      if (is <= wt) M[is] = mfma4(tile(2 * KT + is), bm, M[is]);
    if ((vt & 1) == half) {                            // one half writes dv and counts dR.v
      const f32x4 y = t < a.nv ? r * gt.beta[t] : f32x4{0.f, 0.f, 0.f, 0.f};
      rv += r[0] * x[0] + r[1] * x[1] + r[2] * x[2] + r[3] * x[3];
      T* p = dv0 + (int64_t)t * cfg.dv_stride[1] + v;
      if (t < rows) {
        if (v + 4 <= d.V) store_pack<T, 4>(p, y);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (v + e < d.V) p[e] = (T)y[e];
      }
    }
    lds_barrier();
  }
  dot = rowsum4(row16_sum(dot));
  if ((threadIdx.x & 63) == 0) dots[w] = dot;
  rv = rowsum4(rv);
  if (g == 0) dbv[half][t] = rv;
#pragma unroll
  for (int is = 0; is < 4; ++is) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int s = 16 * is + 4 * g + r;
      const float dec = s <= t ? decay(gt, t, s) : 0.f;
      M[is][r] = dec == 0.f || (half && s == t) ? 0.f : M[is][r] * (half ? -dec : cfg.scale * dec);
    }
    put4(half ? &dAs[t][16 * is + 4 * g] : &dPs[t][16 * is + 4 * g], M[is]);      // dP scale decay, dA decay (without beta_t)
  }
  __syncthreads();
  const float fq = cfg.scale * gt.head[t], fr = gt.head[t], bt = gt.beta[t], tail = gt.tail[t];
#pragma unroll
  for (int q = 0; q < KH; ++q) {
    X1[q] = fr == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : X1[q] * fq;
    X2[q] = fr == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : X2[q] * -fr;
  }
  for (int is = 0; is <= wt; ++is) {
    const f32x4 bp = at4(&dPs[t][16 * is + 4 * g]), ba = at4(&dAs[t][16 * is + 4 * g]);
#pragma unroll
    for (int q = 0; q < KH; ++q)
      if (k0 + q < KT) {
        const f32x4 kc = column4(&k.v[16 * is + 4 * g][16 * (k0 + q) + j], RS);
        X1[q] = mfma4(kc, bp, X1[q]);              // dq
        X2[q] = mfma4(kc, ba, X2[q]);              // the terms of dk that carry beta_t, without it
      }
  }
  // A token whose segment holds a key or query that is not finite: NaN, in place of the terms that were left out
  const float poison = odd >> (gt.seg[t] - first_seg) & 1 ? NAN : 0.f;
  f32x4 C[KH];
#pragma unroll
  for (int q = 0; q < KH; ++q) C[q] = f32x4{poison, poison, poison, poison};
  for (int it = wt; it < 4; ++it) {
    const f32x4 bp = col4(&dPs[16 * it + 4 * g][t], kC + 4), ba = gated(col4(&dAs[16 * it + 4 * g][t], kC + 4), at4(&gt.beta[16 * it + 4 * g]));
#pragma unroll
    for (int i = 0; i < KH; ++i)
      if (k0 + i < KT) {
        C[i] = mfma4(column4(&q.v[16 * it + 4 * g][16 * (k0 + i) + j], RS), bp, C[i]);
        C[i] = mfma4(column4(&k.v[16 * it + 4 * g][16 * (k0 + i) + j], RS), ba, C[i]);
      }
  }
  float pq = 0.f, pr = 0.f, pc = 0.f, ps = 0.f;
#pragma unroll
  for (int i = 0; i < KH; ++i)
    if (k0 + i < KT) {
      const int f = 16 * (k0 + i) + 4 * g;
      const f32x4 kv = row4(&k.v[t][f]), qv = row4(&q.v[t][f]), e = tail == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : X3[i] * tail;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        pq = fmaf(qv[r], X1[i][r], pq);
        pr = fmaf(kv[r], X2[i][r], pr);
        pc = fmaf(kv[r], C[i][r], pc);
        ps = fmaf(kv[r], e[r], ps);
      }
      put_k(dq, cfg.dq_stride, dqp, t, f, X1[i] + poison);
      put_k(dk, cfg.dk_stride, dkp, t, f, X2[i] * bt + C[i] + e);
    }
  pq = rowsum4(pq); pr = rowsum4(pr); pc = rowsum4(pc); ps = rowsum4(ps);
  if (g == 0) {
    sums[half][0][t] = pq;
    sums[half][1][t] = pr;
    sums[half][2][t] = pc;
    sums[half][3][t] = ps;
  }
  __syncthreads();
  if (w == 0) {
    const int l = threadIdx.x, seg = gt.seg[l];
    const float r = sums[0][1][l] + sums[1][1][l];
    const float db = r + dbv[0][l] + dbv[1][l];
    if (l < rows) db0[(int64_t)l * cfg.dbeta_stride[1]] = l < a.nv ? db : 0.f;
    double end = gt.tail[l] == 0.f ? 0.0 : (double)sums[0][3][l] + sums[1][3][l];
    double x = (double)sums[0][0][l] + sums[1][0][l] + gt.beta[l] * (double)r - sums[0][2][l] - sums[1][2][l] - end;
    for (int m = 1; m < 64; m <<= 1) {
      const double o = __shfl_down(x, m, 64);
      const int so = __shfl_down(seg, m, 64);
      if (l + m < 64 && so == seg) x += o;
      end += __shfl_xor(end, m, 64);
    }
    double dot_all = 0.0;
    for (int i = 0; i < 8; ++i) dot_all += dots[i];
    if (gt.whole != 0.f) end += (double)gt.whole * dot_all;
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
  float *ST, *UT, *WT, *gC, *tails;
  delta_saved(d, (float*)saved, &ST, &UT, &WT, &gC, &tails);
  void* Ks = workspace;
  float* dUT = (float*)workspace + d.chunks * kC * d.Kp;
  float* dST = dUT + d.chunks * d.Vp * kC;
  float* dqp = dST + d.chunks * d.Vp * d.Kp;
  float* dkp = dqp + (int64_t)d.B * d.T * d.H * d.K;
  return with_elem(cfg->dtype, [&](auto t) {
    typedef decltype(t) T;
    const dim3 grid((unsigned)d.chunks);
#define OPE_BPREP(KT) \
  case KT: OPE_LAUNCH((delta_bwd_prep<T, KT>), grid, dim3(64 * chunk_waves<KT>()), 0, st, *cfg, d, (const T*)q, (const T*)k, g, beta, lengths, (const T*)d_o, (T*)Ks, dUT, dST); break
    switch (d.KT) { OPE_BPREP(1); OPE_BPREP(2); OPE_BPREP(3); OPE_BPREP(4); OPE_BPREP(5); OPE_BPREP(6); OPE_BPREP(8); }
#undef OPE_BPREP
    OPE_CHECK_LAUNCH();
    const int rc = launch_delta_scan(cfg->dtype, d, true, lengths, Ks, WT, dUT, dST, gC, tails, d_state, d_state0, st);
    if (rc) return rc;
#define OPE_BMAIN(KT)                                                                                                                                  \
  case KT: OPE_LAUNCH((delta_bwd_main<T, KT>), grid, dim3(512), 0, st, *cfg, d, (const T*)q, (const T*)k, (const T*)v, g, beta, lengths, ST, UT,        \
                      (const T*)d_o, dUT, dST, (T*)dq, (T*)dk, dqp, dkp, (T*)dv, dg, dbeta); break
    switch (d.KT) { OPE_BMAIN(1); OPE_BMAIN(2); OPE_BMAIN(3); OPE_BMAIN(4); OPE_BMAIN(5); OPE_BMAIN(6); OPE_BMAIN(8); }
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
