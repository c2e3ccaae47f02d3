// Gated delta rule, forward: chunked over time for training and long inputs, one token at a time for acting (ope.h).
//
//   delta_prep   parallel over chunks: decays, A, the triangular solve for W and U0
//   delta_scan   serial over chunks, parallel over (sequence, head, 16 value columns): U = U0 - W S, S' = e^G S + k^T e^.. U
//   delta_out    parallel over chunks: o = scale (e^G q S + tril(q k^T decay) U)
//   delta_step   one token: state read and written once
#include "ope_delta.h"

namespace ope {

bool delta_ok(const ope_delta_cfg* c) {
  if (!c || c->batch < 0 || c->seq_len < 0 || c->n_heads < 1 || c->n_qk_heads < 1 || c->n_heads % c->n_qk_heads) return false;
  if (c->key_dim < 1 || c->key_dim > 128 || c->value_dim < 1 || c->value_dim > 1024 || !elem_float(c->dtype)) return false;
  const DeltaDims d = delta_dims(c);
  const int64_t bh = (int64_t)d.B * d.H;                // (below 2^62; so are the products, each factor being checked first)
  if (!launch_fits(bh, 512) || !launch_fits(bh * d.VT, 256) || !launch_fits(bh * d.n, 512) || !launch_fits(bh * d.K * d.V / 256 + 1, 256)) return false;
  return d.H == d.Hk || launch_fits((int64_t)d.B * d.T * d.Hk * d.K / 256 + 1, 256);
}

// Rows of one chunk-head: W = (I + A)^-1 beta e^G k, U0 = (I + A)^-1 beta v by block forward substitution, 16 columns a wave at a time.
template <typename T, int KT>
__global__ __launch_bounds__(64 * chunk_waves<KT>(), KT >= 4 ? 4 : 3) void delta_prep(ope_delta_cfg cfg, DeltaDims d, const T* __restrict__ k_in,
                                                                    const T* __restrict__ v_in, const float* __restrict__ g_in, const float* __restrict__ beta_in,
                                                                    const int32_t* __restrict__ lengths, float* __restrict__ W, float* __restrict__ WT,
                                                                    T* __restrict__ KTs, float* __restrict__ UT, float* __restrict__ gC,
                                                                    float* __restrict__ tails) {
  constexpr int NW = chunk_waves<KT>();
  __shared__ Rows<T, KT> k;
  __shared__ float NA[kC][kC + 4], inv[4][16][20];
  __shared__ Gates gt;
  const ChunkAt a = chunk_at(d, lengths, blockIdx.x);
  if (a.nv == 0) return;
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  if (w == 0) load_gates(gt, cfg, a, g_in, beta_in);
  load_rows<T, KT, 64 * NW>(k, k_in, cfg.k_stride, a, a.h / (d.H / d.Hk), d.K);
  __syncthreads();
  minus_A<T, KT>(NA, k, gt);
  if (threadIdx.x == 0) gC[a.c] = gt.whole;
  if (threadIdx.x < kC) tails[a.c * kC + threadIdx.x] = copysignf(gt.tail[threadIdx.x], gt.seg[threadIdx.x] ? -1.f : 1.f);
  __syncthreads();
  if (w == 0) diag_inverse(inv, NA, gt);
  for (int x = w; x < 4 * KT; x += NW) {                 // k transposed, a tile a wave; 0 where the token does not reach the chunk's end
    const int kt = x >> 2, it = x & 3;
    typename Pack<T, 4>::vec v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = gt.tail[16 * it + 4 * g + r] == 0.f ? (T)0.f : k.v[16 * it + 4 * g + r][16 * kt + j];
    *reinterpret_cast<typename Pack<T, 4>::vec*>(KTs + (a.c * KT * 4 + x) * 256 + tile_lane()) = v;
  }
  __syncthreads();
  auto put = [&](int cg, int it, f32x4 x) {
    if (cg < KT) {
      put4(&WT[((a.c * KT + cg) * 4 + it) * 256 + tile_lane()], x);
      put4(&W[((a.c * 4 + it) * KT + cg) * 256 + turned_lane()], turn4(x));
    } else {
      put4(&UT[((a.c * d.VT + cg - KT) * 4 + it) * 256 + tile_lane()], x);
    }
  };
  auto right = [&](int cg, f32x4* x) {                   // the right-hand side
    if (cg < KT) {
#pragma unroll
      for (int it = 0; it < 4; ++it)
        x[it] = gated(at4(&gt.head[16 * it + 4 * g]), column4(&k.v[16 * it + 4 * g][16 * cg + j], Rows<T, KT>::kStride) * at4(&gt.beta[16 * it + 4 * g]));
    } else {
      load_columns(x, v_in, cfg.v_stride, a, 16 * (cg - KT) + j, d.V);
#pragma unroll
      for (int it = 0; it < 4; ++it) x[it] *= at4(&gt.beta[16 * it + 4 * g]);
    }
  };
  const int last = gt.last();
  unsigned again = 0;                                    // this wave's column groups with something that is not finite
  int mine = 0;
  for (int cg = w; cg < KT + d.VT; cg += NW, ++mine) {
    f32x4 x[4];
    right(cg, x);
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      f32x4 acc = x[it];
#pragma unroll
      for (int kt = 0; kt < it; ++kt) acc = mfma4(at4(&NA[16 * it + j][16 * kt + 4 * g]), x[kt], acc);
      x[it] = mfma4(at4(&inv[it][j][4 * g]), acc, f32x4{0.f, 0.f, 0.f, 0.f});
      put(cg, it, x[it]);
    }
    if (last && __any(!finite<4>(x))) again |= 1u << mine;
  }
  if (!again) return;
  mine = 0;
#pragma unroll 1
  for (int cg = w; cg < KT + d.VT; cg += NW, ++mine)
    if (again >> mine & 1) {
      f32x4 b[4], x[4] = {};
      right(cg, b);
#pragma unroll 1
      for (int s = gt.first(); s <= (cg < KT ? 0 : last); ++s) {      // one segment at a time (W is 0 behind a reset, whatever A holds there)
        f32x4 y[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          f32x4 acc = only(gt, s, 16 * it + 4 * g, b[it]);
#pragma unroll
          for (int kt = 0; kt < it; ++kt) acc = mfma4(at4(&NA[16 * it + j][16 * kt + 4 * g]), y[kt], acc);
          acc = only(gt, s, 16 * it + 4 * g, acc);
          y[it] = only(gt, s, 16 * it + 4 * g, mfma4(at4(&inv[it][j][4 * g]), acc, f32x4{0.f, 0.f, 0.f, 0.f}));
          x[it] += y[it];
        }
      }
#pragma unroll
      for (int it = 0; it < 4; ++it) put(cg, it, x[it]);
    }
}

// The scan, forward or backward in time. Four waves share 16 value columns of one (sequence, head): wave w makes the 16 tokens 16w.. of
// P = M1 S (64 x Kp times Kp x 16), then its share of the state's tiles of 16 keys. S lives in registers; it and U cross between the waves
// through LDS, two barriers a chunk. The chain of a chunk is what bounds it, so every chunk's operands are loaded two chunks ahead into their own
// registers (two sets, the loop is unrolled by two).
//   forward : U = U0 - W S;            S' = gC S + k^T (tail U)          M1 = W (float32),   M2 = KTs
//   backward: dU = dU0 + tail (k dS'); dS = gC dS' + N - WT dU           M1 = Ks,            M2 = WT (float32)
// (a row of tail scales a product's result or its operand: the keys themselves stay in their own type, at half the bytes.)
// A token behind a reset in its chunk (a minus sign on its tail) sees nothing of the state in front of the chunk and passes nothing back to it; one whose tail
// is 0, nothing of the state behind it: what is not finite does not get through either.
template <typename T, int KT, bool BWD>
struct ScanOperands {
  static constexpr int NK = (KT + 3) / 4;             // tiles of keys a wave
  typedef typename std::conditional<BWD, T, float>::type T1;
  typedef typename std::conditional<BWD, float, T>::type T2;
  typename Pack<T1, 4>::vec m1[KT];
  typename Pack<T2, 4>::vec m2[NK][4];
  f32x4 u, add[NK], tail;
  float whole;
};
template <typename T, int KT, bool BWD>
__global__ __launch_bounds__(256) void delta_scan(DeltaDims d, const int32_t* __restrict__ lengths, const void* M1v, const void* M2v, float* UT, float* ST,
                                                  const float* gC, const float* tails, const float* __restrict__ first, float* __restrict__ last) {
  constexpr int Kp = 16 * KT, NK = (KT + 3) / 4;
  typedef ScanOperands<T, KT, BWD> Ops;
  const typename Ops::T1* M1 = (const typename Ops::T1*)M1v;
  const typename Ops::T2* M2 = (const typename Ops::T2*)M2v;
  __shared__ float SL[16][Kp + 4], UL[16][kC + 4];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  // Workgroups of one (sequence, head) read the same M1 and M2: they are dealt to one XCD (workgroup index mod 8) in whole groups of 8 heads.
  const unsigned VT = d.VT, group = blockIdx.x / (8 * VT), in = blockIdx.x % (8 * VT);
  const bool grouped = (group + 1) * 8ull <= (unsigned long long)d.B * d.H;
  const int vt = grouped ? in / 8 : blockIdx.x % VT;
  const int64_t bh = grouped ? group * 8ll + in % 8 : blockIdx.x / VT;
  const int b = (int)(bh / d.H), v = 16 * vt + j, lane = tile_lane();
  const int n = ope_cdiv_dev(live_len(lengths, b, d.T), kC);
  f32x4 S[NK];
#pragma unroll
  for (int q = 0; q < NK; ++q)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 16 * (w + 4 * q) + 4 * g + r;
      S[q][r] = first && k < d.K && v < d.V ? first[(bh * d.K + k) * d.V + v] : 0.f;
    }
  typedef decltype(Ops().m1[0] + Ops().m1[0]) V1;
  typedef decltype(Ops().m2[0][0] + Ops().m2[0][0]) V2;
  auto at = [&](int s) { return bh * d.n + (BWD ? n - 1 - min(s, n - 1) : min(s, n - 1)); };     // chunk of step s; past the end: the last one again
  auto get1 = [&](Ops& o, int64_t c, int q) { o.m1[q] = *reinterpret_cast<const V1*>(M1 + ((c * 4 + w) * KT + q) * 256 + lane); };
  auto get2 = [&](Ops& o, int64_t c, int q, int p) { o.m2[q][p] = *reinterpret_cast<const V2*>(M2 + ((c * KT + min(w + 4 * q, KT - 1)) * 4 + p) * 256 + lane); };
  auto get_rest = [&](Ops& o, int64_t c) {
    o.u = at4(&UT[((c * VT + vt) * 4 + w) * 256 + lane]);
    if (BWD)
#pragma unroll
      for (int q = 0; q < NK; ++q) o.add[q] = at4(&ST[((c * VT + vt) * KT + min(w + 4 * q, KT - 1)) * 256 + lane]);
    o.tail = at4(&tails[c * kC + 16 * w + 4 * g]);
    o.whole = gC[c];
  };
  // The operands of the step after next are loaded one by one, each behind the product that read its registers last: in one burst they hold up
  // the wave until the CU has taken them all (measured: 2.4 us a chunk at Kp = 128, 1.3 without any loads), and left to itself the compiler moves
  // them to the front, into registers of their own, and waits for the copies. (M1, M2 are not __restrict__ for the same reason.)
  auto step = [&](Ops& o, int s) {
    const int64_t c = at(s), next = at(s + 2);
#pragma unroll
    for (int q = 0; q < NK; ++q)
      if (KT % 4 == 0 || w + 4 * q < KT) {
        put4(&SL[j][16 * (w + 4 * q) + 4 * g], S[q]);
        put4(&ST[((c * VT + vt) * KT + w + 4 * q) * 256 + lane], S[q]);
      }
    lds_barrier();
    f32x4 p0 = {0.f, 0.f, 0.f, 0.f}, p1 = p0, x[KT > 4 ? KT : 4];
#pragma unroll
    for (int q = 0; q < KT; ++q) x[q] = at4(&SL[j][16 * q + 4 * g]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < KT; ++q) {
      f32x4& p = q & 1 ? p1 : p0;
      p = mfma4(__builtin_convertvector(o.m1[q], f32x4), x[q], p);
      get1(o, next, q);
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 u, pass;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool behind = __float_as_uint(o.tail[r]) >> 31;
      const float tail = fabsf(o.tail[r]), p = p0[r] + p1[r];
      u[r] = BWD ? o.u[r] + gated(tail, p) : (behind ? o.u[r] : o.u[r] - p);
      pass[r] = BWD ? (behind ? 0.f : u[r]) : gated(tail, u[r]);
    }
    put4(&UL[j][16 * w + 4 * g], pass);
    put4(&UT[((c * VT + vt) * 4 + w) * 256 + lane], u);
    lds_barrier();
#pragma unroll
    for (int p = 0; p < 4; ++p) x[p] = at4(&UL[j][16 * p + 4 * g]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < NK; ++q)
      if (KT % 4 == 0 || w + 4 * q < KT) {
        f32x4 a0 = {0.f, 0.f, 0.f, 0.f}, a1 = a0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          f32x4& acc = p & 1 ? a1 : a0;
          acc = mfma4(__builtin_convertvector(o.m2[q][p], f32x4), x[p], acc);
          get2(o, next, q, p);
          __builtin_amdgcn_sched_barrier(0);
        }
        const f32x4 kept = o.whole == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o.whole * S[q];
        S[q] = BWD ? kept + o.add[q] - (a0 + a1) : kept + (a0 + a1);
      }
    __builtin_amdgcn_sched_barrier(0);
    get_rest(o, next);
  };
  auto fetch = [&](Ops& o, int s) {
    const int64_t c = at(s);
#pragma unroll
    for (int q = 0; q < KT; ++q) get1(o, c, q);
#pragma unroll
    for (int q = 0; q < NK; ++q)
#pragma unroll
      for (int p = 0; p < 4; ++p) get2(o, c, q, p);
    get_rest(o, c);
  };
  if (n > 0) {
    Ops even, odd;
    fetch(even, 0);
    fetch(odd, 1);
    int s = 0;
    for (; s + 1 < n; s += 2) {
      step(even, s);
      step(odd, s + 1);
    }
    if (s < n) step(even, s);
  }
#pragma unroll
  for (int q = 0; q < NK; ++q)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 16 * (w + 4 * q) + 4 * g + r;
      if (last && k < d.K && v < d.V) last[(bh * d.K + k) * d.V + v] = S[q][r];
    }
}

// o of one chunk-head. Wave w owns the tokens 16w..: its rows of scale tril(q k^T decay) and of scale e^G q stay in registers while it walks
// the value columns. The tiles of S and U of 16 columns reach LDS once, in two buffers where q and k were: each wave loads a quarter of the next ones
// while these are multiplied.
template <typename T, int KT>
__global__ __launch_bounds__(256, KT * sizeof(T) > 16 ? 2 : 4) void delta_out(ope_delta_cfg cfg, DeltaDims d, const T* __restrict__ q_in, const T* __restrict__ k_in,
                                                 const float* __restrict__ g_in, const float* __restrict__ beta_in, const int32_t* __restrict__ lengths,
                                                 const float* __restrict__ ST, const float* __restrict__ UT, T* __restrict__ o) {
  constexpr int kTiles = KT + 4, kShare = (kTiles + 3) / 4;
  constexpr int kRows = 2 * (int)sizeof(Rows<T, KT>), kStage = 2 * kTiles * 1024;
  __shared__ __attribute__((aligned(16))) uint8_t pool[kRows > kStage ? kRows : kStage];
  Rows<T, KT>&k = reinterpret_cast<Rows<T, KT>*>(pool)[0], &q = reinterpret_cast<Rows<T, KT>*>(pool)[1];
  float* stage = reinterpret_cast<float*>(pool);
  __shared__ Gates gt;
  const ChunkAt a = chunk_at(d, lengths, blockIdx.x);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  T* o0 = o + a.b * cfg.o_stride[0] + (int64_t)a.t0 * cfg.o_stride[1] + a.h * cfg.o_stride[2];
  const int rows = min(d.T - a.t0, kC);
  if (a.nv == 0) {
    for (int e = threadIdx.x; e < rows * d.V; e += 256) o0[(int64_t)(e / d.V) * cfg.o_stride[1] + e % d.V] = (T)0.f;
    return;
  }
  f32x4 pre[kShare];
  auto fetch = [&](int vt) {                           // past the end: the last columns again
    const int64_t at = a.c * d.VT + min(vt, d.VT - 1);
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
      const int x = min(w + 4 * i, kTiles - 1);
      pre[i] = at4((x < KT ? ST + (at * KT + x) * 256 : UT + (at * 4 + x - KT) * 256) + tile_lane());
    }
  };
  fetch(0);
  if (w == 0) load_gates(gt, cfg, a, g_in, beta_in);
  const int hk = a.h / (d.H / d.Hk);
  load_rows<T, KT, 256>(q, q_in, cfg.q_stride, a, hk, d.K);
  load_rows<T, KT, 256>(k, k_in, cfg.k_stride, a, hk, d.K);
  __syncthreads();
  const int t = 16 * w + j;
  f32x4 qs[KT], P[4];
#pragma unroll
  for (int is = 0; is < 4; ++is) {
    P[is] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (is <= w) {
#pragma unroll
      for (int c = 0; c < KT; ++c) P[is] = dot4(&k.v[16 * is + j][16 * c + 4 * g], &q.v[t][16 * c + 4 * g], P[is]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int s = 16 * is + 4 * g + r;
        const float dec = s <= t ? decay(gt, t, s) : 0.f;
        P[is][r] = dec == 0.f ? 0.f : cfg.scale * dec * P[is][r];
      }
    }
  }
  const float f = cfg.scale * gt.head[t];
  const int last = gt.last();
#pragma unroll
  for (int c = 0; c < KT; ++c) qs[c] = row4(&q.v[t][16 * c + 4 * g]) * f;
  __syncthreads();                                     // q and k are done with
  for (int vt = 0; vt < d.VT; ++vt) {
    float* tiles = stage + (vt & 1) * kTiles * 256 + tile_lane();
#pragma unroll
    for (int i = 0; i < kShare; ++i)
      if (w + 4 * i < kTiles) put4(tiles + (w + 4 * i) * 256, pre[i]);
    lds_barrier();
    fetch(vt + 1);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f}, acc2 = acc;
#pragma unroll
    for (int c = 0; c < KT; ++c) acc = mfma4(qs[c], at4(tiles + c * 256), acc);
#pragma unroll
    for (int is = 0; is < 4; ++is)
      if (is <= w) acc2 = mfma4(P[is], at4(tiles + (KT + is) * 256), acc2);
    if (last && __any(!finite(acc + acc2))) {       // tokens 16w + 4g .. + 3: no state behind a reset, and one segment's updates at a time
      f32x4 sum = only(gt, 0, 16 * w + 4 * g, acc);
#pragma unroll 1
      for (int s = gt.first(); s <= last; ++s) {
        acc2 = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int is = 0; is < 4; ++is)
          if (is <= w) acc2 = mfma4(P[is], only(gt, s, 16 * is + 4 * g, at4(tiles + (KT + is) * 256)), acc2);
        sum += only(gt, s, 16 * w + 4 * g, acc2);
      }
      acc = sum;
    } else {
      acc += acc2;
    }
    acc = turn4(acc);                      // four columns of one token a lane
    const int tt = 16 * w + 4 * g + (j & 3), v4 = 16 * vt + 4 * (j >> 2);
    if (tt >= a.nv) acc = f32x4{0.f, 0.f, 0.f, 0.f};   // (behind the last live token q is 0, but its product with a state that is not finite is not)
    if (tt < rows) {
      T* p = o0 + (int64_t)tt * cfg.o_stride[1] + v4;
      if (v4 + 4 <= d.V) store_pack<T, 4>(p, acc);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v4 + e < d.V) p[e] = (T)acc[e];
    }
  }
}

// One token. A workgroup has 64 value columns of one (row, head): lane l of a wave 4 columns (l & 15), the keys dealt out over 16 groups of
// 16 lanes. S passes through registers once: S^T k and S^T q in the same walk (o = e^g q.S + (q.k) u), then the update. Bound by memory.
template <typename T, int NK>
__global__ __launch_bounds__(256) void delta_step(ope_delta_cfg cfg, const T* __restrict__ q_in, const T* __restrict__ k_in, const T* __restrict__ v_in,
                                                  const float* __restrict__ g_in, const float* __restrict__ beta_in, float* __restrict__ state,
                                                  T* __restrict__ o) {
  __shared__ float red[2][16][64];
  __shared__ float qk_sh;
  const int K = cfg.key_dim, V = cfg.value_dim, H = cfg.n_heads;
  const int vb = ope_cdiv_dev(V, 64);
  const int64_t bh = blockIdx.x / vb;
  const int b = (int)(bh / H), h = (int)(bh % H), hk = h / (H / cfg.n_qk_heads);
  const int grp = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4, v0 = (int)(blockIdx.x % vb) * 64 + c;
  const T* qp = q_in + b * cfg.q_stride[0] + hk * cfg.q_stride[2];
  const T* kp = k_in + b * cfg.k_stride[0] + hk * cfg.k_stride[2];
  const float a = expf(g_in[b * cfg.g_stride[0] + h * cfg.g_stride[2]]);
  const float beta = beta_in[b * cfg.beta_stride[0] + h * cfg.beta_stride[2]];
  float* S0 = state + bh * K * V;
  f32x4 S[NK], sk = {0.f, 0.f, 0.f, 0.f}, sq = sk;
  float kk[NK], qk = 0.f;
  const bool whole = v0 + 4 <= V;
  if (whole) {
#pragma unroll
    for (int n = 0; n < NK; ++n) S[n] = load_pack<float, 4>(S0 + (int64_t)min(grp + 16 * n, K - 1) * V + v0);
  } else {
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[n][e] = v0 + e < V ? S0[(int64_t)min(grp + 16 * n, K - 1) * V + v0 + e] : 0.f;
  }
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int k = grp + 16 * n, kc = min(k, K - 1);      // keys past the last one: read again, weighted with 0 and not written
    kk[n] = k < K ? (float)kp[kc] : 0.f;
    const float qq = k < K ? (float)qp[kc] : 0.f;
    qk = fmaf(qq, kk[n], qk);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      S[n][e] = a == 0.f || k >= K ? 0.f : S[n][e] * a;   // (a reset forgets whatever the state holds)
      sk[e] = fmaf(S[n][e], kk[n], sk[e]);
      sq[e] = fmaf(S[n][e], qq, sq[e]);
    }
  }
  put4(&red[0][grp][c], sk);
  put4(&red[1][grp][c], sq);
  __shared__ float qks[16];
  if ((threadIdx.x & 15) == 0) qks[grp] = qk;
  __syncthreads();
  if (threadIdx.x == 0) {
    float v = 0.f;
    for (int i = 0; i < 16; ++i) v += qks[i];
    qk_sh = v;
  }
  f32x4 u = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < 16; ++i) u += at4(&red[0][i][c]);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (v0 + e < V) u[e] = beta * ((float)v_in[b * cfg.v_stride[0] + h * cfg.v_stride[2] + v0 + e] - u[e]);
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) S[n][e] = fmaf(kk[n], u[e], S[n][e]);
  if (whole) {
#pragma unroll
    for (int n = 0; n < NK; ++n)
      if (grp + 16 * n < K) store_pack<float, 4>(S0 + (int64_t)(grp + 16 * n) * V + v0, S[n]);
  } else {
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (grp + 16 * n < K && v0 + e < V) S0[(int64_t)(grp + 16 * n) * V + v0 + e] = S[n][e];
  }
  if (grp == 0) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 16; ++i) s += at4(&red[1][i][c]);
    T* op = o + b * cfg.o_stride[0] + h * cfg.o_stride[2] + v0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v0 + e < V) op[e] = (T)(cfg.scale * fmaf(qk_sh, u[e], s[e]));
  }
}

__global__ void delta_keep_state(const float* __restrict__ from, float* __restrict__ to, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

int launch_delta_scan(int dtype, const DeltaDims& d, bool bwd, const int32_t* lengths, const void* M1, const void* M2, float* UT, float* ST,
                      const float* gC, const float* tails, const float* first, float* last, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)d.B * d.H * d.VT));
  return with_elem(dtype, [&](auto t) {
    typedef decltype(t) T;
#define OPE_SCAN(KT)                                                                                                               \
  case KT:                                                                                                                         \
    if (bwd) OPE_LAUNCH((delta_scan<T, KT, true>), grid, dim3(256), 0, st, d, lengths, M1, M2, UT, ST, gC, tails, first, last);     \
    else OPE_LAUNCH((delta_scan<T, KT, false>), grid, dim3(256), 0, st, d, lengths, M1, M2, UT, ST, gC, tails, first, last);        \
    break
    switch (d.KT) { OPE_SCAN(1); OPE_SCAN(2); OPE_SCAN(3); OPE_SCAN(4); OPE_SCAN(5); OPE_SCAN(6); OPE_SCAN(8); }
#undef OPE_SCAN
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  });
}

}  // namespace ope
using namespace ope;

namespace ope {
// the arrays of `saved`, in the order the header of ope_delta.h names them; returns its floats
int64_t delta_saved(const DeltaDims& d, float* saved, float** ST, float** UT, float** WT, float** gC, float** tails) {
  const int64_t ut = d.chunks * d.Vp * d.Kp, wt = ut + d.chunks * d.Vp * kC, tl = wt + d.chunks * d.Kp * kC, gc = tl + d.chunks * kC;
  *ST = saved; *UT = saved + ut; *WT = saved + wt; *tails = saved + tl; *gC = saved + gc;
  return gc + ((d.chunks + 3) & ~(int64_t)3);
}
int64_t delta_bwd_floats(const DeltaDims& d) {
  return d.chunks * ((int64_t)kC * d.Kp + (int64_t)d.Vp * kC + (int64_t)d.Vp * d.Kp) + (d.H != d.Hk ? 2 * (int64_t)d.B * d.T * d.H * d.K : 0);
}
}

extern "C" int64_t ope_delta_saved_bytes(const ope_delta_cfg* cfg) {
  if (!delta_ok(cfg)) return OPE_EINVAL;
  float *a, *b, *c, *e, *f;
  return 4 * delta_saved(delta_dims(cfg), nullptr, &a, &b, &c, &e, &f);
}

extern "C" int64_t ope_delta_workspace_bytes(const ope_delta_cfg* cfg, int32_t backward) {
  if (!delta_ok(cfg)) return OPE_EINVAL;
  const DeltaDims d = delta_dims(cfg);
  return 4 * (backward ? delta_bwd_floats(d) : d.chunks * 2 * kC * d.Kp);
}

extern "C" int ope_delta_forward(const ope_delta_cfg* cfg, const void* q, const void* k, const void* v, const float* g, const float* beta,
                                 const float* state0, const int32_t* lengths, void* o, float* state_out, void* saved, int64_t saved_bytes,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  if (!delta_ok(cfg)) return OPE_EINVAL;
  const DeltaDims d = delta_dims(cfg);
  hipStream_t st = (hipStream_t)stream;
  if (d.B == 0) return OPE_OK;
  if (!state_out) return OPE_EINVAL;
  if (d.T == 0) {
    const int64_t n = (int64_t)d.B * d.H * d.K * d.V;
    OPE_LAUNCH(delta_keep_state, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, state0, state_out, n);
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  }
  if (!q || !k || !v || !g || !beta || !o || !saved || !workspace) return OPE_EINVAL;
  if (saved_bytes < ope_delta_saved_bytes(cfg) || workspace_bytes < ope_delta_workspace_bytes(cfg, 0)) return OPE_ENOSPC;
  float *ST, *UT, *WT, *gC, *tails;
  delta_saved(d, (float*)saved, &ST, &UT, &WT, &gC, &tails);
  float* W = (float*)workspace;
  void* KTs = W + d.chunks * kC * d.Kp;
  return with_elem(cfg->dtype, [&](auto t) {
    typedef decltype(t) T;
    const dim3 grid((unsigned)d.chunks);
#define OPE_PREP(KT) \
  case KT: OPE_LAUNCH((delta_prep<T, KT>), grid, dim3(64 * chunk_waves<KT>()), 0, st, *cfg, d, (const T*)k, (const T*)v, g, beta, lengths, W, WT, (T*)KTs, UT, gC, tails); break
    switch (d.KT) { OPE_PREP(1); OPE_PREP(2); OPE_PREP(3); OPE_PREP(4); OPE_PREP(5); OPE_PREP(6); OPE_PREP(8); }
#undef OPE_PREP
    OPE_CHECK_LAUNCH();
    const int rc = launch_delta_scan(cfg->dtype, d, false, lengths, W, KTs, UT, ST, gC, tails, state0, state_out, st);
    if (rc) return rc;
#define OPE_OUT(KT) \
  case KT: OPE_LAUNCH((delta_out<T, KT>), grid, dim3(256), 0, st, *cfg, d, (const T*)q, (const T*)k, g, beta, lengths, ST, UT, (T*)o); break
    switch (d.KT) { OPE_OUT(1); OPE_OUT(2); OPE_OUT(3); OPE_OUT(4); OPE_OUT(5); OPE_OUT(6); OPE_OUT(8); }
#undef OPE_OUT
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  });
}

extern "C" int ope_delta_step(const ope_delta_cfg* cfg, const void* q, const void* k, const void* v, const float* g, const float* beta, float* state,
                              void* o, void* stream) {
  if (!delta_ok(cfg)) return OPE_EINVAL;
  if (cfg->batch == 0) return OPE_OK;
  if (!q || !k || !v || !g || !beta || !state || !o) return OPE_EINVAL;
  const int64_t blocks = (int64_t)cfg->batch * cfg->n_heads * ope_cdiv(cfg->value_dim, 64);
  if (blocks >= ((int64_t)1 << 31)) return OPE_EINVAL;
  return with_elem(cfg->dtype, [&](auto t) {
    typedef decltype(t) T;
#define OPE_STEP(NK) \
  OPE_LAUNCH((delta_step<T, NK>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *cfg, (const T*)q, (const T*)k, (const T*)v, g, beta, state, (T*)o)
    if (cfg->key_dim <= 16) OPE_STEP(1);
    else if (cfg->key_dim <= 32) OPE_STEP(2);
    else if (cfg->key_dim <= 64) OPE_STEP(4);
    else OPE_STEP(8);
#undef OPE_STEP
    OPE_CHECK_LAUNCH();
    return OPE_OK;
  });
}
