// Shared pieces of the gated delta rule's kernels (ope_delta.hip: forward and one-token step; ope_delta_bwd.hip: gradients).
//
// Names: a CHUNK is 64 tokens of one (sequence, head) = "chunk-head" c = (b * H + h) * n + i. Kp / Vp are the key and value widths padded to the
// tiles of 16 the kernels work in (Kp: 16 to 96, or 128). Every sum is float32. What touches a state, a decay or a solve runs on the f32 matrix
// instruction of ope_common.h: its "transposed chain" (lane (j, g) holds features 4g .. 4g+3 of data row j) is both the form a product leaves and the
// form the next one reads, so the triangular solve and the scan need no shuffles. q k^T and k k^T of 16-bit inputs run on the bf16 / f16 one (dot4).
//
// Arrays in `saved` (S, kept for the backward pass) and in the workspace (W). All lie in TILES of 16 x 16, in the order in which the lanes of a
// wave hold them: lane (j, g) has row j, columns 4g .. 4g+3, tile after tile, so that every access of a wave is one run of whole cache lines (rows
// of the matrices themselves took twice the time: a CU's requests in flight, not its bytes, bound the scan). turn4 gives a tile transposed. The
// last two indexes below count tiles; float32 unless said otherwise.
//   ST [c][VT][KT]  S  the state in front of the chunk: rows v, columns k
//   UT [c][VT][4]   S  U0 before the scan, u of the chunk's tokens after it: rows v, columns t
//   WT [c][KT][4]   S  W transposed: rows k, columns t
//   gC [c]          S  decay over the whole chunk (0 behind a reset);   tails [c][64]  S  decay from t to the chunk's end, with a minus sign where a
//                      reset lies between the chunk's start and t
//   W  [c][4][KT]   W  rows t, columns k;   KTs [c][KT][4]  W  of the inputs' type: k transposed, rows k, columns t
//   backward: Ks [c][4][KT]  W  of the inputs' type: k, rows t, columns k;   dUT like UT (dU0, then dU, then dR with its tiles transposed);
//   dST like ST (N, then the gradient of the state BEHIND the chunk);   dqp, dkp [b][t][H][K] where query / key heads are shared
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
  d.KT = d.K > 96 ? 8 : ope_cdiv(d.K, 16);            // (seven tiles spill more registers of the backward pass than eight)
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
// keep their last bits); a reset (e^g = 0 in float32: -inf, and every g under -103.97, so that no finite stand-in for -inf swallows the small gates
// that are added behind it) starts a new segment with G = 0, and decays across segments are exactly 0: what lies behind a reset
// does not depend on what lies in front of it, to the last bit.
//
// Nor does it where values are not finite. A product by a mask's zeros lets them through (0 times NaN), so (1) what a decay scales is dropped where the
// decay is 0 (gated), and (2) a matrix product whose contraction runs over the tokens of several segments is done again one segment at a time where
// its result is not finite (only), or goes without the values that are not (delta_bwd_main). That costs the few chunks it happens in; without a reset in
// the chunk nothing is asked. Inside its segment such a value may spread to the chunk's tokens in front of it.
struct Gates {
  float hi[kC], lo[kC], beta[kC], head[kC], tail[kC];   // head: decay from the chunk's start through t; tail: from t to its end
  int seg[kC];
  float whole;                                          // decay over the whole chunk
  __device__ __forceinline__ int first() const { return __builtin_amdgcn_readfirstlane(seg[0]); }
  __device__ __forceinline__ int last() const { return __builtin_amdgcn_readfirstlane(seg[kC - 1]); }      // 0: no reset in the chunk
};
__device__ __forceinline__ float gated(float decay, float x) { return decay == 0.f ? 0.f : decay * x; }
__device__ __forceinline__ f32x4 gated(f32x4 decay, f32x4 x) {
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = gated(decay[r], x[r]);
  return x;
}
// x of the tokens t .. t + 3, 0 where they belong to another segment than s. (The index is opaque: left to itself the compiler reads the segments of every
// use far ahead, on the way that hardly ever comes here too, and spills.)
__device__ __forceinline__ f32x4 only(const Gates& gt, int s, int t, f32x4 x) {
  asm volatile("" : "+v"(t));
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = gt.seg[t + r] == s ? x[r] : 0.f;
  return x;
}
// Whether all of x[0 .. N) are finite, by one sum (where that alone leaves the range, no: asked again at no harm). z - z is 0 for finite numbers alone.
template <int N>
__device__ __forceinline__ bool finite(const f32x4* x) {
  f32x4 z = x[0];
#pragma unroll
  for (int n = 1; n < N; ++n) z += x[n];
  const float s = (z[0] + z[1]) + (z[2] + z[3]);
  return s - s == 0.f;
}
__device__ __forceinline__ bool finite(f32x4 x) { return finite<1>(&x); }
__device__ __forceinline__ float decay(const Gates& s, int t, int u) {   // from u through t (u <= t)
  return s.seg[t] == s.seg[u] ? expf((s.hi[t] - s.hi[u]) + (s.lo[t] - s.lo[u])) : 0.f;
}
// By one wave; the caller puts a barrier behind it. Tokens that are not live: g = 0, beta = 0.
__device__ __forceinline__ void load_gates(Gates& s, const ope_delta_cfg& c, const ChunkAt& a, const float* g, const float* beta) {
  const int t = threadIdx.x & 63;
  const bool on = t < a.nv;
  const float gt = on ? g[a.b * c.g_stride[0] + (int64_t)(a.t0 + t) * c.g_stride[1] + a.h * c.g_stride[2]] : 0.f;
  const float bt = on ? beta[a.b * c.beta_stride[0] + (int64_t)(a.t0 + t) * c.beta_stride[1] + a.h * c.beta_stride[2]] : 0.f;
  const bool cut = expf(gt) == 0.f;                     // as the one-token step decides it
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

// A chunk of q or k in LDS, in its own type, rows 16 bytes longer than the padded width (16 rows read at one column then hit different banks).
template <typename T, int KT>
struct Rows {
  static constexpr int kStride = 16 * KT + 16 / (int)sizeof(T);
  T v[kC][kStride];
};
// What lies outside (tokens that are not live, columns past K) is 0. Lanes outside load the nearest row (and column) inside, so that all of a
// thread's loads are in flight together. TH threads.
template <typename T, int KT, int TH>
__device__ __forceinline__ void load_rows(Rows<T, KT>& dst, const T* p, const int64_t* stride, const ChunkAt& a, int head, int K) {
  typedef typename Pack<T, 4>::vec vec;
  constexpr int all = kC * KT * 4, N = (all + TH - 1) / TH;
  const T* base = p + a.b * stride[0] + (int64_t)a.t0 * stride[1] + head * stride[2];
  vec v[N];
  if (K == 16 * KT) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = min((int)threadIdx.x + TH * i, all - 1), t = q / (KT * 4), k = (q % (KT * 4)) * 4;
      v[i] = *reinterpret_cast<const typename Pack<T, 4>::loose*>(base + (int64_t)min(t, a.nv - 1) * stride[1] + k);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = min((int)threadIdx.x + TH * i, all - 1), t = q / (KT * 4), k = (q % (KT * 4)) * 4;
      const T* row = base + (int64_t)min(t, a.nv - 1) * stride[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = row[min(k + e, K - 1)];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int q = threadIdx.x + TH * i, t = q / (KT * 4), k = (q % (KT * 4)) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i][e] = t < a.nv && k + e < K ? v[i][e] : (T)0.f;
    if (q < all) *reinterpret_cast<vec*>(&dst.v[t][k]) = v[i];
  }
}
// four elements of a row / of a column, as float32
template <typename T>
__device__ __forceinline__ f32x4 row4(const T* p) {
  return __builtin_convertvector(*reinterpret_cast<const typename Pack<T, 4>::vec*>(p), f32x4);
}
template <typename T>
__device__ __forceinline__ f32x4 column4(const T* p, int stride) {
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = (float)p[r * stride];
  return v;
}

// Column `col` of a chunk of v or dO at the tokens 16 it + 4 g + r, it = 0..3: x[it][r], 0 outside the live tokens and the width. Every lane loads
// (the nearest element inside where its own is outside): 16 loads in flight instead of 16 branches that each wait for one.
template <typename T>
__device__ __forceinline__ void load_columns(f32x4* x, const T* p, const int64_t* stride, const ChunkAt& a, int col, int V) {
  const int g = (threadIdx.x >> 4) & 3;
  const T* base = p + a.b * stride[0] + (int64_t)a.t0 * stride[1] + a.h * stride[2] + min(col, V - 1);
  T raw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) raw[i] = base[(int64_t)min(16 * (i >> 2) + 4 * g + (i & 3), a.nv - 1) * stride[1]];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i >> 2][i & 3] = 16 * (i >> 2) + 4 * g + (i & 3) < a.nv && col < V ? (float)raw[i] : 0.f;
}

__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {   // 16 x 16 x 16: four steps of the f32 matrix instruction
#pragma unroll
  for (int r = 0; r < 4; ++r) c = mfma16(a[r], b[r], c);
  return c;
}
// The same product of two rows as they lie in LDS. Products of bfloat16 and float16 are exact in float32 and their matrix instructions add them in
// float32 (measured: 1.8e-8 of the result's norm, as the f32 instruction), at 8 times its rate: nothing is lost by not widening first.
__device__ __forceinline__ f32x4 dot4(const float* a, const float* b, f32x4 c) { return mfma4(row4(a), row4(b), c); }
__device__ __forceinline__ f32x4 dot4(const bf16_t* a, const bf16_t* b, f32x4 c) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(*reinterpret_cast<const s16x4*>(a), *reinterpret_cast<const s16x4*>(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 dot4(const f16_t* a, const f16_t* b, f32x4 c) {
  typedef Pack<f16_t, 4>::vec vec;
  return __builtin_amdgcn_mfma_f32_16x16x16f16(*reinterpret_cast<const vec*>(a), *reinterpret_cast<const vec*>(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 at4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ void put4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
// A lane's place in a tile, and its place in the same tile read or written transposed (turn4 on the far side).
__device__ __forceinline__ int tile_lane() { return (threadIdx.x & 63) * 4; }
__device__ __forceinline__ int turned_lane() {
  const int j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  return (4 * g + (j & 3) + 16 * (j >> 2)) * 4;
}
// Transpose of the 4 x 4 that four neighbouring lanes hold: result[e] = lane e's x[own place in the four].
__device__ __forceinline__ f32x4 turn4(f32x4 x) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    const float got = OPE_DPP_F(odd ? x[e] : x[e + 1], 0xB1);
    x[e] = odd ? got : x[e];
    x[e + 1] = odd ? x[e + 1] : got;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float got = OPE_DPP_F(high ? x[e] : x[e + 2], 0x4E);
    x[e] = high ? got : x[e];
    x[e + 2] = high ? x[e + 2] : got;
  }
  return x;
}
__device__ __forceinline__ f32x4 col4(const float* p, int64_t stride) {   // four elements `stride` apart
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = p[r * stride];
  return v;
}

// tile x of the 10 on and below the diagonal of a chunk's 4 x 4
__device__ __forceinline__ void lower_tile(int x, int& it, int& is) {
  it = x < 1 ? 0 : (x < 3 ? 1 : (x < 6 ? 2 : 3));
  is = x - it * (it + 1) / 2;
}
// -A (strictly lower, -A_ij = -beta_i decay(i, j) k_i.k_j) of the chunk in LDS: the 10 tiles on and below the diagonal, zeros above it in the
// diagonal tiles (the tiles above are neither written nor read). Tiles are dealt out to the waves; barrier behind.
template <typename T, int KT>
__device__ __forceinline__ void minus_A(float (*NA)[kC + 4], const Rows<T, KT>& k, const Gates& gt) {
  const int j = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  for (int x = threadIdx.x >> 6; x < 10; x += blockDim.x >> 6) {
    int it, is;
    lower_tile(x, it, is);
    const int t = 16 * it + j;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KT; ++c) acc = dot4(&k.v[16 * is + j][16 * c + 4 * g], &k.v[t][16 * c + 4 * g], acc);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int s = 16 * is + 4 * g + r;
      const float d = decay(gt, t, s);
      acc[r] = s < t && d != 0.f ? -gt.beta[t] * d * acc[r] : 0.f;
    }
    put4(&NA[t][16 * is + 4 * g], acc);
  }
}
// Inverses of the four unit lower triangular 16 x 16 blocks on the diagonal of I + A, by forward substitution: lane (column c, block). One wave.
__device__ __forceinline__ void diag_inverse(float (*inv)[16][20], const float (*NA)[kC + 4], const Gates& gt) {
  const int c = threadIdx.x & 15, blk = (threadIdx.x >> 4) & 3;
  float t[16];
  bool fine = true;
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
    fine &= v - v == 0.f;
    inv[blk][i][c] = v;
  }
  if (gt.last() == 0 || !__any(!fine)) return;
  // rows of A that are not finite: again, with the zeros above the diagonal and between segments kept
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    float v = i == c ? 1.f : 0.f;
    if (i > c && gt.seg[16 * blk + i] == gt.seg[16 * blk + c])
#pragma unroll 1
      for (int q = c; q < i; ++q)
        if (gt.seg[16 * blk + q] == gt.seg[16 * blk + c]) v = fmaf(NA[16 * blk + i][16 * blk + q], inv[blk][q][c], v);
    inv[blk][i][c] = v;
  }
}

// waves of a workgroup in the kernels that work on whole chunks: 4, or 8 where the keys are wide enough to keep them busy
template <int KT>
constexpr int chunk_waves() { return KT >= 4 ? 8 : 4; }

}  // namespace ope
