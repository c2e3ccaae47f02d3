// Shared pieces of the gated delta rule's kernels (ope_delta.hip: forward and one-token step; ope_delta_bwd.hip: gradients).
//
// Names: a CHUNK is 64 tokens of one (sequence, head) = "chunk-head" c = (b * H + h) * n + i. Kp / Vp are the key and value widths padded to the
// tiles of 16 the kernels work in (Kp to 16, 32, 64 or 128). Arithmetic is float32 throughout, on the f32 matrix instruction of ope_common.h:
// its "transposed chain" (lane (j, g) holds features 4g .. 4g+3 of data row j) is both the form a product leaves and the form the next one
// reads, so the triangular solve and the scan need no shuffles.
//
// Arrays in `saved` (S, kept for the backward pass) and in the workspace (W), all float32:
//   ST  [c][Vp][Kp]   S  the state in front of the chunk, transposed          UT [c][Vp][64]  S  u of the chunk's tokens (U0 before the scan)
//   WT  [c][Kp][64]   S  W transposed                                         gC [c]          S  decay over the whole chunk (0 behind a reset)
//   W   [c][64][Kp]   W                                                       KdT [c][Kp][64] W  k_t * decay from t to the chunk's end
//   backward: Kd [c][64][Kp], dUT [c][Vp][64] (dU0, then dU, then dR), dST [c][Vp][Kp] (N, then the gradient of the state BEHIND the chunk),
//   dqp, dkp [b][t][H][K] where query / key heads are shared
#pragma once
#include <type_traits>

#include "ope_elem.h"

namespace ope {

constexpr int kC = 64;            // tokens a chunk
__device__ __forceinline__ int ope_cdiv_dev(int a, int b) { return (a + b - 1) / b; }

struct DeltaDims {
  int B, T, H, Hk, K, V, n, KT, VT, Kp, Vp;
  int64_t chunks;                 // B * H * n
};

static inline DeltaDims delta_dims(const ope_delta_cfg* c) {
  DeltaDims d;
  d.B = c->batch; d.T = c->seq_len; d.H = c->n_heads; d.Hk = c->n_qk_heads; d.K = c->key_dim; d.V = c->value_dim;
  d.n = ope_cdiv(d.T, kC);
  d.KT = d.K <= 16 ? 1 : d.K <= 32 ? 2 : d.K <= 64 ? 4 : 8;
  d.VT = ope_cdiv(d.V, 16);
  d.Kp = 16 * d.KT; d.Vp = 16 * d.VT;
  d.chunks = (int64_t)d.B * d.H * d.n;
  return d;
}

bool delta_ok(const ope_delta_cfg* c);

// One chunk-head: where it is and how many of its tokens are live.
struct ChunkAt {
  int64_t c;
  int b, h, i, t0, nv;            // nv live tokens from t0 on (0 behind the sequence's end)
};
__device__ __forceinline__ int live_len(const int32_t* lengths, int b, int T) { return lengths ? min(max(lengths[b], 0), T) : T; }
__device__ __forceinline__ ChunkAt chunk_at(const DeltaDims& d, const int32_t* lengths, int64_t c) {
  ChunkAt a;
  a.c = c;
  a.i = (int)(c % d.n);
  const int64_t bh = c / d.n;
  a.h = (int)(bh % d.H);
  a.b = (int)(bh / d.H);
  a.t0 = a.i * kC;
  a.nv = min(max(live_len(lengths, a.b, d.T) - a.t0, 0), kC);
  return a;
}

// The chunk's gates in LDS. G is the running sum of g inside a segment of the chunk, as a pair of floats (hi + lo: differences of long sums
// keep their last bits); a reset (g = -inf) starts a new segment with G = 0, and decays across segments are exactly 0: what lies behind a reset
// does not depend on what lies in front of it, to the last bit.
struct Gates {
  float hi[kC], lo[kC], beta[kC], head[kC], tail[kC];   // head: decay from the chunk's start through t; tail: from t to its end
  int seg[kC];
  float whole;                                          // decay over the whole chunk
};
__device__ __forceinline__ float decay(const Gates& s, int t, int u) {   // from u through t (u <= t)
  return s.seg[t] == s.seg[u] ? expf((s.hi[t] - s.hi[u]) + (s.lo[t] - s.lo[u])) : 0.f;
}
// By one wave; the caller puts a barrier behind it. Tokens that are not live: g = 0, beta = 0.
__device__ __forceinline__ void load_gates(Gates& s, const ope_delta_cfg& c, const ChunkAt& a, const float* g, const float* beta) {
  const int t = threadIdx.x & 63;
  const bool on = t < a.nv;
  const float gt = on ? g[a.b * c.g_stride[0] + (int64_t)(a.t0 + t) * c.g_stride[1] + a.h * c.g_stride[2]] : 0.f;
  const float bt = on ? beta[a.b * c.beta_stride[0] + (int64_t)(a.t0 + t) * c.beta_stride[1] + a.h * c.beta_stride[2]] : 0.f;
  const bool cut = gt == -INFINITY;
  const unsigned long long cuts = __ballot(cut);
  const int seg = __popcll(cuts & (~0ull >> (63 - t)));
  double G = cut ? 0.0 : (double)gt;
  for (int m = 1; m < 64; m <<= 1) {
    const double o = __shfl_up(G, m, 64);
    const int so = __shfl_up(seg, m, 64);
    if (t >= m && so == seg) G += o;
  }
  const double end = __shfl(G, 63, 64);
  const int last = __popcll(cuts);
  s.hi[t] = (float)G;
  s.lo[t] = (float)(G - (double)(float)G);
  s.seg[t] = seg;
  s.beta[t] = bt;
  s.head[t] = seg == 0 ? expf((float)G) : 0.f;
  s.tail[t] = seg == last ? expf((float)(end - G)) : 0.f;
  if (t == 63) s.whole = seg == 0 ? expf((float)G) : 0.f;
}

// A chunk of q or k as float32 in LDS [64][Kp + 4]; what lies outside (tokens that are not live, columns past K) is 0. 256 threads.
template <typename T, int KT>
__device__ __forceinline__ void load_rows(float (*dst)[16 * KT + 4], const T* p, const int64_t* stride, const ChunkAt& a, int head, int K) {
  const T* base = p + a.b * stride[0] + (int64_t)a.t0 * stride[1] + head * stride[2];
  for (int q = threadIdx.x; q < kC * KT * 4; q += 256) {
    const int t = q / (KT * 4), k = (q % (KT * 4)) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (t < a.nv) {
      const T* row = base + (int64_t)t * stride[1];
      if (k + 4 <= K) v = load_pack<T, 4>(row + k);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < K) v[e] = (float)row[k + e];
    }
    *reinterpret_cast<f32x4*>(&dst[t][k]) = v;
  }
}

__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {   // 16 x 16 x 16: four steps of the f32 matrix instruction
#pragma unroll
  for (int r = 0; r < 4; ++r) c = mfma16(a[r], b[r], c);
  return c;
}
__device__ __forceinline__ f32x4 at4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ void put4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ f32x4 col4(const float* p, int64_t stride) {   // four elements `stride` apart
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = p[r * stride];
  return v;
}

// -A (strictly lower, -A_ij = -beta_i decay(i, j) k_i.k_j) of the chunk in LDS, zero elsewhere. 4 waves, one row of tiles each; barrier behind.
template <int KT>
__device__ __forceinline__ void minus_A(float (*NA)[kC + 4], const float (*k)[16 * KT + 4], const Gates& gt) {
  const int w = threadIdx.x >> 6, j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int t = 16 * w + j;
  for (int is = 0; is < 4; ++is) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (is <= w) {
      for (int c = 0; c < KT; ++c) acc = mfma4(at4(&k[16 * is + j][16 * c + 4 * g]), at4(&k[t][16 * c + 4 * g]), acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int s = 16 * is + 4 * g + r;
        acc[r] = s < t ? -gt.beta[t] * decay(gt, t, s) * acc[r] : 0.f;
      }
    }
    put4(&NA[t][16 * is + 4 * g], acc);
  }
}
// Inverses of the four unit lower triangular 16 x 16 blocks on the diagonal of I + A, by forward substitution: lane (column c, block). One wave.
__device__ __forceinline__ void diag_inverse(float (*inv)[16][20], const float (*NA)[kC + 4]) {
  const int c = threadIdx.x & 15, blk = (threadIdx.x >> 4) & 3;
  float t[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float v = i == c ? 1.f : 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (4 * q < i) {
        const f32x4 a = at4(&NA[16 * blk + i][16 * blk + 4 * q]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (4 * q + r < i) v = fmaf(a[r], t[4 * q + r], v);
      }
    t[i] = v;
    inv[blk][i][c] = v;
  }
}

}  // namespace ope
