// The gated delta rule over whole sequences, forward and backward, in chunks of C tokens.
//
//   S_t = e^g_t S_{t-1} + k_t beta_t (v_t - e^g_t S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t      (S [128 x 128])
//
// With G the running sum of g within a chunk, D_ij = e^(G_i - G_j), S0 the state before the chunk:
//   A_ij = beta_i (k_i . k_j) D_ij (j < i)     Tm = (I + A)^-1      P_ij = scale (q_i . k_j) D_ij (j <= i)
//   R = beta (V - e^G K S0)     U = Tm R       O = scale e^G Q S0 + P U
//   S1 = e^G_C S0 + sum_j e^(G_C - G_j) k_j u_j^T
// and backwards, with dS1 the gradient of the state behind the chunk:
//   dU = P^T dO + e^(G_C - G) K dS1     dR = Tm^T dU     dV = beta dR
//   dS0 = e^G_C dS1 + Q^T (scale e^G dO) - K^T (beta e^G dR)
//
// Three kinds of kernels: what does not depend on the state (delta_chunk_kernel: Tm and P, every
// chunk at once), the state from chunk to chunk (delta_scan_kernel, delta_scan_bwd_kernel), and
// the gradients of q, k, g and beta (delta_grads_kernel, every chunk at once).
//
// Precision: all sums are fp32 on the matrix cores.  bf16 inputs enter the products as they are;
// every fp32 operand (states, U, R, Tm, P, fp32 inputs) enters as the sum of three bf16 parts,
// which hold its 24 bits, and the products of parts down to 2^-16 of the largest are added
// (mma): an error of fp32's own size, at 3 (one operand exact) or 6 bf16 instructions where one
// fp32 instruction takes the time of 16.
#include "gsa_common.h"

namespace gsa {

constexpr int kHead = 128;

// ---------------------------------------------------------------------------
// Operands.  v_mfma_f32_16x16x32_bf16: lane l holds row (A) or column (B) l % 16, elements
// 8 (l / 16) .. + 7 of the 32 summed over; the result's column l % 16, rows 4 (l / 16) .. + 3.
//
// Row `m` of tile `t` of a product stands for index tile_row(t, m): of two tiles (a pair, 32
// indices) a lane of the result then holds 8 consecutive ones, the ones that it has to hold
// as the B operand of the next product.  So a wave that owns 16 columns of the state goes from
// product to product in its own registers.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int tile_row(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

template <int N> struct Parts { bf16x8 p[N]; };

__device__ __forceinline__ Parts<3> split3(const float (&x)[8]) {
  Parts<3> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __bf16 a = (__bf16)x[i];
    const float e = x[i] - (float)a;
    const __bf16 b = (__bf16)e;
    r.p[0][i] = a;
    r.p[1][i] = b;
    r.p[2][i] = (__bf16)(e - (float)b);
  }
  return r;
}
template <int N> __device__ __forceinline__ Parts<N> parts_of(const float (&x)[8]) {
  if constexpr (N == 3) {
    return split3(x);
  } else {
    Parts<1> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.p[0][i] = (__bf16)x[i];
    return r;
  }
}
__device__ __forceinline__ Parts<3> split_pair(const floatx4& a, const floatx4& b) {
  const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return split3(x);
}

// acc += a b: the products of parts i, j with i + j < 3, the smallest first.
template <int NA, int NB>
__device__ __forceinline__ void mma(floatx4& acc, const Parts<NA>& a, const Parts<NB>& b) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == o) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
}

template <typename T> struct DeltaType;
template <> struct DeltaType<uint16_t> { static constexpr int kParts = 1, kChunk = 64; };
template <> struct DeltaType<float> { static constexpr int kParts = 3, kChunk = 32; };

template <typename T> __device__ __forceinline__ float to_f32(T x) {
  if constexpr (sizeof(T) == 2) return bf16lo(x); else return x;
}
template <typename T> __device__ __forceinline__ T from_f32(float x) {
  if constexpr (sizeof(T) == 2) return (T)f32_to_bf16_bits(x); else return x;
}

// ---------------------------------------------------------------------------
// Sequences, chunks and what is kept of a chunk
// ---------------------------------------------------------------------------
struct Rows { const void* p; int64_t sb, st, sh; };         // [B, T, heads, ...]

// Sequences: N rows of a batch of T tokens each, or (cu) N packed one behind the other in T
// tokens, sequence n from cu[n] to cu[n + 1].  Chunk c of sequence n is kept in slot
// first(n) + c; packed sequences leave slots empty (start / C + n, so no sums over lengths are
// needed).  Offsets are held within [0, T]: whatever cu says, nothing outside is touched.
struct Seqs {
  const void* cu;
  int cu64, N, T, slots;
  __device__ int64_t at(int n) const {
    const int64_t x = cu64 ? static_cast<const int64_t*>(cu)[n] : static_cast<const int32_t*>(cu)[n];
    return x < 0 ? 0 : x > T ? T : x;
  }
};
struct Span { int n, b, t0, len, slot0; };                   // sequence n: tokens t0 .. t0 + len - 1 of row b
template <int C> __device__ __forceinline__ Span span_of(const Seqs& s, int n) {
  if (!s.cu) return Span{n, n, 0, s.T, n * ((s.T + C - 1) / C)};
  const int64_t a = s.at(n), e = s.at(n + 1);
  return Span{n, 0, (int)a, e > a ? (int)(e - a) : 0, (int)(a / C) + n};
}
// The sequence and chunk of a slot; c < 0: an empty slot.
template <int C> __device__ __forceinline__ Span slot_of(const Seqs& s, int slot, int& c) {
  if (!s.cu) {
    const int nc = (s.T + C - 1) / C, n = slot / nc;
    c = slot - n * nc;
    return span_of<C>(s, n);
  }
  int lo = 0, hi = s.N - 1;                                  // the last n whose first slot is not behind
  while (lo < hi) {
    const int m = (lo + hi + 1) / 2;
    if ((int)(s.at(m) / C) + m <= slot) lo = m; else hi = m - 1;
  }
  const Span r = span_of<C>(s, lo);
  c = slot - r.slot0;
  if (c < 0 || c >= (r.len + C - 1) / C) c = -1;
  return r;
}

struct DeltaArgs {
  Seqs s;
  Rows q, k, v, g, beta;
  int beta_bf16, Hk, Hv;
  float scale;
  const float* state_in;      // [N, Hv, 128, 128], nullable
  void* o;                    // [B, T, Hv, 128]
  float* state_out;           // nullable
  // a chunk's, [slots][Hv] each
  float* tm;                  // [C][C]: Tm, rows i
  float* pm;                  // [C][C]: P
  float* gates;               // [5][C]: e^G, e^(G_C - G), beta, G (upper and lower part)
  // kept for the backward pass (nullable)
  float* s0;                  // [128][128]: the state before the chunk
  float* u;                   // [C][128]
  // backward
  Rows dout;
  const float* dstate_out;    // nullable
  float* ds1;                 // [128][128]
  float* dr;                  // [C][128]
  void *dq, *dk, *dv;         // [B, T, heads, 128]
  float* dg;                  // [B, T, Hv]
  void* dbeta;
  float* dstate_in;           // nullable
};

template <typename T> __device__ __forceinline__ const T* row_at(const Rows& x, const Span& s, int64_t t, int h) {
  return static_cast<const T*>(x.p) + s.b * x.sb + (s.t0 + t) * x.st + h * x.sh;
}

// 8 consecutive elements of a row as an operand (zeros where !ok).
template <typename T> __device__ __forceinline__ Parts<DeltaType<T>::kParts> operand(const T* p, bool ok) {
  if constexpr (sizeof(T) == 2) {
    u32x4 r = {0, 0, 0, 0};
    if (ok) r = *reinterpret_cast<const u32x4*>(p);
    return {__builtin_bit_cast(bf16x8, r)};
  } else {
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (ok) load8(p, x);
    return split3(x);
  }
}

// ---------------------------------------------------------------------------
// Tm and P of every chunk and v head.  256 threads.
// ---------------------------------------------------------------------------
// 16x16 tile a b of LDS matrices, summed over K (fp32 matrix instruction).
__device__ __forceinline__ floatx4 tile_f32(const float* a, int lda, const float* b, int ldb, int K) {
  const int l = lane_id(), m = l & 15, kk = l >> 4;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < K; s += 4)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m * lda + s + kk], b[(s + kk) * ldb + m], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ void tile_put(float* d, int ld, const floatx4& x, float f) {
  const int l = lane_id();
#pragma unroll
  for (int r = 0; r < 4; ++r) d[(4 * (l >> 4) + r) * ld + (l & 15)] = x[r] * f;
}

template <typename T>
__global__ __launch_bounds__(256) void delta_chunk_kernel(DeltaArgs a) {
  constexpr int C = DeltaType<T>::kChunk, MT = C / 16, LD = C + 4;
  __shared__ float am[C][LD], xm[C][LD], ym[C][LD];
  __shared__ float gh[C], gl[C], bt[C];
  const int slot = blockIdx.x, h = blockIdx.y, hk = h / (a.Hv / a.Hk), tid = threadIdx.x, wave = tid >> 6, l = lane_id();
  int c;
  const Span sp = slot_of<C>(a.s, slot, c);
  if (c < 0) return;
  const int64_t t0 = (int64_t)c * C;
  const int left = sp.len - (int)t0;                         // tokens of the chunk (more than C: C)
  const int64_t at = (int64_t)slot * a.Hv + h;

  if (wave == 0) {
    const bool ok = l < C && l < left;
    float g = 0.f, b = 0.f;
    if (ok) {
      g = *row_at<float>(a.g, sp, t0 + l, h);
      b = a.beta_bf16 ? bf16lo(*row_at<uint16_t>(a.beta, sp, t0 + l, h)) : *row_at<float>(a.beta, sp, t0 + l, h);
      // e^-128 is 0 in fp32: a lower g (down to -inf, a reset) gives the same, without inf - inf
      if (g < -128.f) g = -128.f;
    }
    double G = g;                                            // differences of sums keep fp32's precision
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(G, o, 64);
      if (l >= o) G += y;
    }
    const double Ge = __shfl(G, C - 1, 64);
    const float hi = (float)G, lo = (float)(G - (double)hi);
    if (l < C) {
      gh[l] = hi;
      gl[l] = lo;
      bt[l] = b;
      float* gates = a.gates + at * 5 * C;
      gates[l] = expf((float)G);
      gates[C + l] = expf((float)(Ge - G));
      gates[2 * C + l] = b;
      gates[3 * C + l] = hi;
      gates[4 * C + l] = lo;
    }
  }
  for (int i = tid; i < C * LD; i += 256) (&xm[0][0])[i] = 0.f;
  __syncthreads();

  // row tile mt of K K^T (into am) and of Q K^T (to pm)
  for (int job = wave; job < 2 * MT; job += 4) {
    const int mt = job % MT;
    const bool qk = job >= MT;
    Parts<DeltaType<T>::kParts> x[4];
    {
      const int t = 16 * mt + (l & 15);
      const T* p = qk ? row_at<T>(a.q, sp, t0 + t, hk) : row_at<T>(a.k, sp, t0 + t, hk);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) x[ks] = operand<T>(p + 32 * ks + 8 * (l >> 4), t < left);
    }
    for (int nt = 0; nt < MT; ++nt) {
      const int j = 16 * nt + (l & 15);
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
      if (nt <= mt) {
        const T* p = row_at<T>(a.k, sp, t0 + j, hk);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) mma(acc, x[ks], operand<T>(p + 32 * ks + 8 * (l >> 4), j < left));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * mt + 4 * (l >> 4) + r;
        const float d = expf((gh[i] - gh[j]) + (gl[i] - gl[j]));
        if (qk) a.pm[(at * C + i) * C + j] = j <= i ? a.scale * acc[r] * d : 0.f;
        else am[i][j] = j < i ? bt[i] * acc[r] * d : 0.f;
      }
    }
  }
  __syncthreads();

  // (I + A)^-1: blocks of 16 by substitution, a lane a column; then pairs of blocks, and of pairs:
  // the lower left of the inverse is -Y A21 X with X, Y the inverses above and below it.  (Doubling
  // products of I - A would cancel: for equal keys its terms grow like binomials.)
  if (wave < MT && l < 16) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == l ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) s = __builtin_fmaf(-am[16 * wave + i][16 * wave + m], x[m], s);
      x[i] = s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) xm[16 * wave + i][16 * wave + l] = x[i];
  }
  __syncthreads();
  if (wave < C / 32) {
    const int p = 32 * wave;
    tile_put(&ym[p][p], LD, tile_f32(&am[p + 16][p], LD, &xm[p][p], LD, 16), 1.f);
  }
  __syncthreads();
  if (wave < C / 32) {
    const int p = 32 * wave;
    tile_put(&xm[p + 16][p], LD, tile_f32(&xm[p + 16][p + 16], LD, &ym[p][p], LD, 16), -1.f);
  }
  __syncthreads();
  if constexpr (C == 64) {
    const int i = 16 * (wave >> 1), j = 16 * (wave & 1);
    tile_put(&ym[i][j], LD, tile_f32(&am[32 + i][0], LD, &xm[0][j], LD, 32), 1.f);
    __syncthreads();
    tile_put(&xm[32 + i][j], LD, tile_f32(&xm[32 + i][32], LD, &ym[0][j], LD, 32), -1.f);
    __syncthreads();
  }
  for (int i = tid; i < C * C; i += 256) a.tm[at * C * C + i] = xm[i / C][i % C];
}

// ---------------------------------------------------------------------------
// The state from chunk to chunk.  512 threads: a wave owns 16 columns of one head's state,
// tile 2 ks + e of its registers the rows tile_row(2 ks + e, .).  A chunk's operands lie in LDS
// in the order in which the lanes take them: [tile][step][part][lane] of 16 bytes.
// ---------------------------------------------------------------------------
// Rows of tokens (tile_row), summed over the 128 elements.
template <typename T>
__device__ __forceinline__ void stage_rows(bf16x8* dst, const Rows& x, const Span& sp, int64_t t0, int left, int h, int tid) {
  constexpr int C = DeltaType<T>::kChunk, NP = DeltaType<T>::kParts;
  for (int u = tid; u < C * 16; u += 512) {
    const int d8 = u & 15, t = u >> 4;
    const int tile = 2 * (t >> 5) + ((t >> 2) & 1), m = 4 * ((t >> 3) & 3) + (t & 3);
    const Parts<NP> p = operand<T>(row_at<T>(x, sp, t0 + t, h) + 8 * d8, t < left);
#pragma unroll
    for (int i = 0; i < NP; ++i) dst[((tile * 4 + (d8 >> 2)) * NP + i) * 64 + 16 * (d8 & 3) + m] = p.p[i];
  }
}
// Rows of the 128 elements (tile_row), summed over tokens.
template <typename T>
__device__ __forceinline__ void stage_cols(bf16x8* dst, const Rows& x, const Span& sp, int64_t t0, int left, int h, int tid,
                                           int threads) {
  constexpr int C = DeltaType<T>::kChunk, NP = DeltaType<T>::kParts, JS = C / 32;
  for (int u = tid; u < C * 4; u += threads) {
    const int d4 = u & 31, oct = u >> 5;
    float v[4][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 8 * oct + e;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      if (t < left) {
        const T* p = row_at<T>(x, sp, t0 + t, h) + 4 * d4;
        if constexpr (sizeof(T) == 2) {
          const uint2 r = *reinterpret_cast<const uint2*>(p);
          y[0] = bf16lo(r.x); y[1] = bf16hi(r.x); y[2] = bf16lo(r.y); y[3] = bf16hi(r.y);
        } else {
          const floatx4 r = *reinterpret_cast<const floatx4*>(p);
          y[0] = r[0]; y[1] = r[1]; y[2] = r[2]; y[3] = r[3];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i][e] = y[i];
    }
    const int tile = 2 * (d4 >> 3) + (d4 & 1), m = 4 * ((d4 >> 1) & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Parts<NP> p = parts_of<NP>(v[i]);
#pragma unroll
      for (int n = 0; n < NP; ++n) dst[((tile * JS + (oct >> 2)) * NP + n) * 64 + 16 * (oct & 3) + m + i] = p.p[n];
    }
  }
}
// A [C][C] fp32 matrix, or its transpose: rows of tokens (tile_row), summed over tokens.
template <int C, bool kTransposed>
__device__ __forceinline__ void stage_square(bf16x8* dst, const float* x, int tid) {
  constexpr int JS = C / 32;
  for (int u = tid; u < C * C / 8; u += 512) {
    int t, oct;
    float y[8];
    if constexpr (kTransposed) {
      t = u % C;
      oct = u / C;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[(8 * oct + e) * C + t];
    } else {
      oct = u % (C / 8);
      t = u / (C / 8);
      load8(x + t * C + 8 * oct, y);
    }
    const int tile = 2 * (t >> 5) + ((t >> 2) & 1), m = 4 * ((t >> 3) & 3) + (t & 3);
    const Parts<3> p = split3(y);
#pragma unroll
    for (int n = 0; n < 3; ++n) dst[((tile * JS + (oct >> 2)) * 3 + n) * 64 + 16 * (oct & 3) + m] = p.p[n];
  }
}
template <int N> __device__ __forceinline__ Parts<N> staged(const bf16x8* src, int frag, int l) {
  Parts<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.p[i] = src[(frag * N + i) * 64 + l];
  return r;
}

template <typename T> struct ScanLds {
  static constexpr int C = DeltaType<T>::kChunk, NP = DeltaType<T>::kParts, MT = C / 16, JS = C / 32;
  static constexpr int kRows = MT * 4 * NP * 64, kCols = 8 * JS * NP * 64, kSquare = MT * JS * 3 * 64;
  static constexpr int kGates = 0;                           // floats [3][C]
  static constexpr size_t kFwd = 16 * (size_t)(2 * kRows + kCols + 2 * kSquare) + 3 * C * 4;
  static constexpr size_t kBwd = 16 * (size_t)(kRows + 2 * kCols + 2 * kSquare) + 3 * C * 4;
};

template <typename T>
__global__ __launch_bounds__(512) void delta_scan_kernel(DeltaArgs a) {
  using L = ScanLds<T>;
  constexpr int C = L::C, NP = L::NP, MT = L::MT, JS = L::JS;
  extern __shared__ __align__(16) char lds[];
  bf16x8* sk = reinterpret_cast<bf16x8*>(lds);
  bf16x8* sq = sk + L::kRows;
  bf16x8* skt = sq + L::kRows;
  bf16x8* st = skt + L::kCols;
  bf16x8* sp_ = st + L::kSquare;
  float* gates = reinterpret_cast<float*>(sp_ + L::kSquare);
  const int h = blockIdx.y, hk = h / (a.Hv / a.Hk), tid = threadIdx.x, l = lane_id(), g = l >> 4;
  const int col = 16 * (tid >> 6) + (l & 15);
  const Span sp = span_of<C>(a.s, blockIdx.x);
  const int64_t sn = ((int64_t)sp.n * a.Hv + h) * kHead * kHead;

  floatx4 S[8];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) S[t][r] = a.state_in ? a.state_in[sn + tile_row(t, 4 * g + r) * kHead + col] : 0.f;

  const int chunks = (sp.len + C - 1) / C;
  for (int c = 0; c < chunks; ++c) {
    const int64_t t0 = (int64_t)c * C, at = (int64_t)(sp.slot0 + c) * a.Hv + h;
    const int left = sp.len - (int)t0;
    float v[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = tile_row(mt, 4 * g + r);
        v[mt][r] = t < left ? to_f32(row_at<T>(a.v, sp, t0 + t, h)[col]) : 0.f;
      }
    __syncthreads();
    stage_rows<T>(sk, a.k, sp, t0, left, hk, tid);
    stage_rows<T>(sq, a.q, sp, t0, left, hk, tid);
    stage_cols<T>(skt, a.k, sp, t0, left, hk, tid, 512);
    stage_square<C, false>(st, a.tm + at * C * C, tid);
    stage_square<C, false>(sp_, a.pm + at * C * C, tid);
    if (tid < 3 * C) gates[tid] = a.gates[at * 5 * C + tid];
    if (a.s0)
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) a.s0[at * kHead * kHead + tile_row(t, 4 * g + r) * kHead + col] = S[t][r];
    __syncthreads();

    floatx4 X[MT], O[MT], U[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) X[mt] = O[mt] = U[mt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const Parts<3> s = split_pair(S[2 * ks], S[2 * ks + 1]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma(X[mt], staged<NP>(sk, mt * 4 + ks, l), s);
        mma(O[mt], staged<NP>(sq, mt * 4 + ks, l), s);
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = tile_row(mt, 4 * g + r);
        X[mt][r] = gates[2 * C + t] * (v[mt][r] - gates[t] * X[mt][r]);      // R
        O[mt][r] *= a.scale * gates[t];
      }
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      const Parts<3> r = split_pair(X[2 * js], X[2 * js + 1]);
#pragma unroll
      for (int mt = 2 * js; mt < MT; ++mt) mma(U[mt], staged<3>(st, mt * JS + js, l), r);
    }
    const float whole = gates[C - 1];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][r] *= whole;
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      const Parts<3> u = split_pair(U[2 * js], U[2 * js + 1]);
#pragma unroll
      for (int mt = 2 * js; mt < MT; ++mt) mma(O[mt], staged<3>(sp_, mt * JS + js, l), u);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = U[2 * js + (e >> 2)][e & 3] * gates[C + 32 * js + 8 * g + e];
      const Parts<3> ud = split3(x);
#pragma unroll
      for (int t = 0; t < 8; ++t) mma(S[t], staged<NP>(skt, t * JS + js, l), ud);
    }
    T* o = static_cast<T*>(a.o);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = tile_row(mt, 4 * g + r);
        if (t < left) o[(((int64_t)sp.b * a.s.T + sp.t0 + t0 + t) * a.Hv + h) * kHead + col] = from_f32<T>(O[mt][r]);
        if (a.u) a.u[(at * C + t) * kHead + col] = U[mt][r];
      }
  }
  if (a.state_out)
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.state_out[sn + tile_row(t, 4 * g + r) * kHead + col] = S[t][r];
}

template <typename T>
__global__ __launch_bounds__(512) void delta_scan_bwd_kernel(DeltaArgs a) {
  using L = ScanLds<T>;
  constexpr int C = L::C, NP = L::NP, MT = L::MT, JS = L::JS;
  extern __shared__ __align__(16) char lds[];
  bf16x8* sk = reinterpret_cast<bf16x8*>(lds);
  bf16x8* skt = sk + L::kRows;
  bf16x8* sqt = skt + L::kCols;
  bf16x8* st = sqt + L::kCols;
  bf16x8* sp_ = st + L::kSquare;
  float* gates = reinterpret_cast<float*>(sp_ + L::kSquare);
  const int h = blockIdx.y, hk = h / (a.Hv / a.Hk), tid = threadIdx.x, l = lane_id(), g = l >> 4;
  const int col = 16 * (tid >> 6) + (l & 15);
  const Span sp = span_of<C>(a.s, blockIdx.x);
  const int64_t sn = ((int64_t)sp.n * a.Hv + h) * kHead * kHead;

  floatx4 S[8];                                              // dS
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) S[t][r] = a.dstate_out ? a.dstate_out[sn + tile_row(t, 4 * g + r) * kHead + col] : 0.f;

  for (int c = (sp.len + C - 1) / C - 1; c >= 0; --c) {
    const int64_t t0 = (int64_t)c * C, at = (int64_t)(sp.slot0 + c) * a.Hv + h;
    const int left = sp.len - (int)t0;
    float d[MT][4];                                          // dO
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = tile_row(mt, 4 * g + r);
        d[mt][r] = t < left ? to_f32(row_at<T>(a.dout, sp, t0 + t, h)[col]) : 0.f;
      }
    __syncthreads();
    stage_rows<T>(sk, a.k, sp, t0, left, hk, tid);
    stage_cols<T>(skt, a.k, sp, t0, left, hk, tid, 512);
    stage_cols<T>(sqt, a.q, sp, t0, left, hk, tid, 512);
    stage_square<C, true>(st, a.tm + at * C * C, tid);
    stage_square<C, true>(sp_, a.pm + at * C * C, tid);
    if (tid < 3 * C) gates[tid] = a.gates[at * 5 * C + tid];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.ds1[at * kHead * kHead + tile_row(t, 4 * g + r) * kHead + col] = S[t][r];
    __syncthreads();

    floatx4 X[MT], R[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) X[mt] = R[mt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const Parts<3> s = split_pair(S[2 * ks], S[2 * ks + 1]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) mma(X[mt], staged<NP>(sk, mt * 4 + ks, l), s);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) X[mt][r] *= gates[C + tile_row(mt, 4 * g + r)];
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      const float x[8] = {d[2 * js][0], d[2 * js][1], d[2 * js][2], d[2 * js][3],
                          d[2 * js + 1][0], d[2 * js + 1][1], d[2 * js + 1][2], d[2 * js + 1][3]};
      const Parts<NP> p = parts_of<NP>(x);
#pragma unroll
      for (int mt = 0; mt < 2 * js + 2; ++mt) mma(X[mt], staged<3>(sp_, mt * JS + js, l), p);    // dU
    }
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      const Parts<3> p = split_pair(X[2 * js], X[2 * js + 1]);
#pragma unroll
      for (int mt = 0; mt < 2 * js + 2; ++mt) mma(R[mt], staged<3>(st, mt * JS + js, l), p);     // dR
    }
    T* dv = static_cast<T*>(a.dv);
    const float whole = gates[C - 1];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][r] *= whole;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = tile_row(mt, 4 * g + r);
        const float beta = gates[2 * C + t];
        a.dr[(at * C + t) * kHead + col] = R[mt][r];
        if (t < left) dv[(((int64_t)sp.b * a.s.T + sp.t0 + t0 + t) * a.Hv + h) * kHead + col] = from_f32<T>(beta * R[mt][r]);
        R[mt][r] *= -beta * gates[t];
        d[mt][r] *= a.scale * gates[t];
      }
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      const float x[8] = {d[2 * js][0], d[2 * js][1], d[2 * js][2], d[2 * js][3],
                          d[2 * js + 1][0], d[2 * js + 1][1], d[2 * js + 1][2], d[2 * js + 1][3]};
      const Parts<3> p = split3(x), r = split_pair(R[2 * js], R[2 * js + 1]);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        mma(S[t], staged<NP>(sqt, t * JS + js, l), p);
        mma(S[t], staged<NP>(skt, t * JS + js, l), r);
      }
    }
  }
  if (a.dstate_in)
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.dstate_in[sn + tile_row(t, 4 * g + r) * kHead + col] = S[t][r];
}

// ---------------------------------------------------------------------------
// dq, dk, dg, dbeta of a chunk.  With E = dO U^T, F = dR U^T (lower, strictly lower):
//   dQ = scale e^G (dO S0^T) + scale (E D) K
//   dK = scale (E D)^T Q + e^(G_C - G) (U dS1^T) - beta e^G (dR S0^T) + (B + B^T) K,  B_ij = -beta_i F_ij D_ij
//   dbeta_i = dR_i . v_i - e^G_i k_i . (dR S0^T)_i - sum_j F_ij (k_i . k_j) D_ij
//   dG: row sums less column sums of M = E P + B (K K^T), and the three products with S0 and
//       dS1, row by row, times q or k; dg is the sum of dG from the token to the chunk's end.
// 256 threads, a q/k head and the v heads that share it one after the other (so dq and dk need no
// atomics).  Products with rows of the 128 elements are computed transposed: a wave owns 32
// of them (two tiles), a lane 8 of one token.
// ---------------------------------------------------------------------------
template <typename T> struct GradLds {
  static constexpr int C = DeltaType<T>::kChunk, NP = DeltaType<T>::kParts, JS = C / 32;
  static constexpr int kLdR = kHead + 4, kLdC = C + 4;
  static constexpr int kCols = 8 * JS * NP * 64;             // 16-byte units
  static constexpr int kFloats = 2 * C * kLdR + 3 * C * kLdC + 4 * 3 * C + 5 * C + 2 * C + 8;
  static constexpr size_t kBytes = 16 * (size_t)(2 * kCols) + 4 * (size_t)kFloats + 8 * C;
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

template <typename T>
__global__ __launch_bounds__(256) void delta_grads_kernel(DeltaArgs a) {
  using L = GradLds<T>;
  constexpr int C = L::C, NP = L::NP, MT = C / 16, JS = L::JS, LR = L::kLdR, LC = L::kLdC;
  extern __shared__ __align__(16) char lds[];
  bf16x8* skt = reinterpret_cast<bf16x8*>(lds);
  bf16x8* sqt = skt + L::kCols;
  double* dsum = reinterpret_cast<double*>(sqt + L::kCols);  // [C]
  float* su = reinterpret_cast<float*>(dsum + C);            // U [C][LR]
  float* sr = su + C * LR;                                   // dR
  float* se = sr + C * LR;                                   // scale E D [C][LC]
  float* sb = se + C * LC;                                   // B + B^T
  float* sm = sb + C * LC;                                   // M
  float* red = sm + C * LC;                                  // [4 waves][3][C]
  float* gates = red + 12 * C;                               // [5][C]
  float* db = gates + 5 * C;                                 // [C]: dR . v, then + sum of F (K K^T) D
  float* fs = db + C;                                        // [C]
  float* cross = fs + C;                                     // [4]
  const int slot = blockIdx.x, hk = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, l = lane_id(), g = l >> 4, m = l & 15;
  int c;
  const Span sp = slot_of<C>(a.s, slot, c);
  if (c < 0) return;
  const int64_t t0 = (int64_t)c * C;
  const int left = sp.len - (int)t0, share = a.Hv / a.Hk;
  const int64_t tok = (int64_t)sp.b * a.s.T + sp.t0 + t0;    // row of [B * T]

  stage_cols<T>(skt, a.k, sp, t0, left, hk, tid, 256);
  stage_cols<T>(sqt, a.q, sp, t0, left, hk, tid, 256);

  floatx4 dq[2][MT], dk[2][MT];                              // [128 elements: tile 2 wave + e][tokens]
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int n = 0; n < MT; ++n) dq[e][n] = dk[e][n] = floatx4{0.f, 0.f, 0.f, 0.f};

  for (int hs = 0; hs < share; ++hs) {
    const int h = hk * share + hs;
    const int64_t at = (int64_t)slot * a.Hv + h;
    __syncthreads();
    for (int i = tid; i < C * kHead / 4; i += 256) {
      const int t = i >> 5, e = 4 * (i & 31);
      *reinterpret_cast<floatx4*>(su + t * LR + e) = *reinterpret_cast<const floatx4*>(a.u + (at * C + t) * kHead + e);
      *reinterpret_cast<floatx4*>(sr + t * LR + e) = *reinterpret_cast<const floatx4*>(a.dr + (at * C + t) * kHead + e);
    }
    for (int i = tid; i < 5 * C; i += 256) gates[i] = a.gates[at * 5 * C + i];
    __syncthreads();

    // E, F, Q K^T, K K^T by tiles of tokens
    for (int mt = wave; mt < MT; mt += 4) {
      const int i0 = 16 * mt + m;
      Parts<NP> xo[4], xk[4], xq[4];
      Parts<3> xr[4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const int e = 32 * ks + 8 * g;
        xo[ks] = operand<T>(row_at<T>(a.dout, sp, t0 + i0, h) + e, i0 < left);
        xk[ks] = operand<T>(row_at<T>(a.k, sp, t0 + i0, hk) + e, i0 < left);
        xq[ks] = operand<T>(row_at<T>(a.q, sp, t0 + i0, hk) + e, i0 < left);
        float y[8];
        load8(sr + i0 * LR + e, y);
        xr[ks] = split3(y);
      }
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      for (int nt = 0; nt < MT; ++nt) {
        floatx4 E = {0.f, 0.f, 0.f, 0.f}, F = E, QK = E, KK = E;
        const int j = 16 * nt + m;
        if (nt <= mt) {
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const int e = 32 * ks + 8 * g;
            float y[8];
            load8(su + j * LR + e, y);
            const Parts<3> u = split3(y);
            const Parts<NP> kj = operand<T>(row_at<T>(a.k, sp, t0 + j, hk) + e, j < left);
            mma(E, xo[ks], u);
            mma(F, xr[ks], u);
            mma(QK, xq[ks], kj);
            mma(KK, xk[ks], kj);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * mt + 4 * g + r;
          if (nt > mt) {
            se[i * LC + j] = sm[i * LC + j] = 0.f;
          } else {
            const float d = j <= i ? expf((gates[3 * C + i] - gates[3 * C + j]) + (gates[4 * C + i] - gates[4 * C + j])) : 0.f;
            const float ed = a.scale * E[r] * d, fd = j < i ? F[r] * d : 0.f, b = -gates[2 * C + i] * fd;
            se[i * LC + j] = ed;
            sm[i * LC + j] = j < i ? ed * QK[r] + b * KK[r] : 0.f;
            f[r] += fd * KK[r];
            if (j < i) {
              sb[i * LC + j] = b;
              sb[j * LC + i] = b;
            } else if (j == i) {
              sb[i * LC + i] = 0.f;
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f[r] = row16_sum(f[r]);
        if (m == 0) fs[16 * mt + 4 * g + r] = f[r];
      }
    }
    // dR . v: 256 / C lanes a token
    {
      constexpr int kPer = 256 / C;
      const int t = tid / kPer;
      float x = 0.f;
      if (t < left)
        for (int e = tid % kPer; e < kHead; e += kPer)
          x = __builtin_fmaf(sr[t * LR + e], to_f32(row_at<T>(a.v, sp, t0 + t, h)[e]), x);
#pragma unroll
      for (int o = 1; o < kPer; o <<= 1) x += __shfl_xor(x, o, 64);
      if (tid % kPer == 0) db[t] = x;
    }

    // dO S0^T, dR S0^T, U dS1^T, transposed
    floatx4 Z1[2][MT], Z2[2][MT], Z3[2][MT];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < MT; ++n) Z1[e][n] = Z2[e][n] = Z3[e][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    double dot = 0.;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      Parts<3> s0[2], s1[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t o = at * kHead * kHead + tile_row(2 * wave + e, m) * kHead + 32 * ks + 8 * g;
        float y[8], z[8];
        load8(a.s0 + o, y);
        load8(a.ds1 + o, z);
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x = __builtin_fmaf(y[i], z[i], x);
        dot += x;
        s0[e] = split3(y);
        s1[e] = split3(z);
      }
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const int t = 16 * n + m, e0 = 32 * ks + 8 * g;
        const Parts<NP> o = operand<T>(row_at<T>(a.dout, sp, t0 + t, h) + e0, t < left);
        float y[8];
        load8(sr + t * LR + e0, y);
        const Parts<3> r = split3(y);
        load8(su + t * LR + e0, y);
        const Parts<3> u = split3(y);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mma(Z1[e][n], s0[e], o);
          mma(Z2[e][n], s1[e], u);
          mma(Z3[e][n], s0[e], r);
        }
      }
    }
    dot = wave_sum(dot);
    if (l == 0) cross[wave] = (float)dot;
#pragma unroll
    for (int n = 0; n < MT; ++n) {
      const int t = 16 * n + m;
      const float e = gates[t], rest = gates[C + t], beta = gates[2 * C + t];
      float q[8] = {0, 0, 0, 0, 0, 0, 0, 0}, k[8] = {0, 0, 0, 0, 0, 0, 0, 0}, x1 = 0.f, x2 = 0.f, x3 = 0.f;
      if (t < left) {
        load8(row_at<T>(a.q, sp, t0 + t, hk) + 32 * wave + 8 * g, q);
        load8(row_at<T>(a.k, sp, t0 + t, hk) + 32 * wave + 8 * g, k);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z1 = a.scale * e * Z1[i >> 2][n][i & 3], z2 = rest * Z2[i >> 2][n][i & 3], z3 = e * Z3[i >> 2][n][i & 3];
        x1 = __builtin_fmaf(q[i], z1, x1);
        x2 = __builtin_fmaf(k[i], z2, x2);
        x3 = __builtin_fmaf(k[i], z3, x3);
        dq[i >> 2][n][i & 3] += z1;
        dk[i >> 2][n][i & 3] += z2 - beta * z3;
      }
      x1 += __shfl_xor(x1, 16, 64); x1 += __shfl_xor(x1, 32, 64);
      x2 += __shfl_xor(x2, 16, 64); x2 += __shfl_xor(x2, 32, 64);
      x3 += __shfl_xor(x3, 16, 64); x3 += __shfl_xor(x3, 32, 64);
      if (g == 0) {
        red[(wave * 3 + 0) * C + t] = x1;
        red[(wave * 3 + 1) * C + t] = x2;
        red[(wave * 3 + 2) * C + t] = x3;
      }
    }
    __syncthreads();

    // the products with K and Q
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      Parts<NP> kt[2], qt[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        kt[e] = staged<NP>(skt, (2 * wave + e) * JS + js, l);
        qt[e] = staged<NP>(sqt, (2 * wave + e) * JS + js, l);
      }
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const int t = 16 * n + m, j0 = 32 * js + 8 * g;
        float x[8], y[8], z[8];
        load8(se + t * LC + j0, x);
        load8(sb + t * LC + j0, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = se[(j0 + i) * LC + t];
        const Parts<3> xe = split3(x), xb = split3(y), xt = split3(z);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mma(dq[e][n], kt[e], xe);
          mma(dk[e][n], kt[e], xb);
          mma(dk[e][n], qt[e], xt);
        }
      }
    }
    // dG in 64 bits: what cancels between the rows and columns of M has to cancel exactly
    if (tid < C) {
      double s = 0.;
      for (int j = 0; j < C; ++j) s += (double)sm[tid * LC + j] - (double)sm[j * LC + tid];
      double x1 = 0., x2 = 0., x3 = 0.;
      for (int w = 0; w < 4; ++w) {
        x1 += red[(w * 3 + 0) * C + tid];
        x2 += red[(w * 3 + 1) * C + tid];
        x3 += red[(w * 3 + 2) * C + tid];
      }
      const float beta = gates[2 * C + tid];
      if (tid < left) {
        const float x = db[tid] - (float)x3 - fs[tid];
        const int64_t o = (tok + tid) * a.Hv + h;
        if (a.beta_bf16) static_cast<uint16_t*>(a.dbeta)[o] = (uint16_t)f32_to_bf16_bits(x);
        else static_cast<float*>(a.dbeta)[o] = x;
      }
      // at the end of the chunk: e^G_C <dS1, S0> and every x2
      dsum[tid] = s + x1 - x2 - beta * x3;
      red[tid] = (float)x2;
    }
    __syncthreads();
    if (wave == 0 && l < C) {
      double x2 = red[l], s = dsum[l];
      double all = x2;
#pragma unroll
      for (int o = 1; o < C; o <<= 1) all += __shfl_xor(all, o, 64);
      if (l == C - 1) s += all + (double)gates[C - 1] * ((double)cross[0] + cross[1] + cross[2] + cross[3]);
#pragma unroll
      for (int o = 1; o < C; o <<= 1) {                      // sum from l to the end
        const double y = __shfl_down(s, o, 64);
        if (l + o < C) s += y;
      }
      if (l < left) a.dg[(tok + l) * a.Hv + h] = (float)s;
    }
  }

#pragma unroll
  for (int n = 0; n < MT; ++n) {
    const int t = 16 * n + m;
    if (t < left) {
      const int64_t o = ((tok + t) * a.Hk + hk) * kHead + 32 * wave + 8 * g;
      float x[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { x[i] = dq[i >> 2][n][i & 3]; y[i] = dk[i >> 2][n][i & 3]; }
      store8(static_cast<T*>(a.dq) + o, x);
      store8(static_cast<T*>(a.dk) + o, y);
    }
  }
}

}  // namespace gsa

namespace gsa_host {
namespace {

constexpr size_t kAlign = 256;
inline size_t up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

struct DeltaSizes { int C; int64_t slots; size_t tm, gates, s0, u; };
// Sizes of one call; slots 0: out of range.
DeltaSizes delta_sizes(int B, int T, int N, int packed, int Hv, int dtype) {
  DeltaSizes z{};
  z.C = dtype == GSA_DTYPE_BF16 ? gsa::DeltaType<uint16_t>::kChunk : gsa::DeltaType<float>::kChunk;
  if (B < 1 || T < 1 || N < 1 || Hv < 1 || !dtype_size(dtype)) return z;
  z.slots = packed ? (int64_t)T / z.C + N : (int64_t)B * ((T + z.C - 1) / z.C);
  if (z.slots > 0x7fffffff) z.slots = 0;
  const size_t n = (size_t)z.slots * Hv;
  z.tm = up(n * z.C * z.C * 4);
  z.gates = up(n * 5 * z.C * 4);
  z.s0 = up(n * 128 * 128 * 4);
  z.u = up(n * z.C * 128 * 4);
  return z;
}

template <auto kKernel> int allow_lds(size_t bytes) {
  static bool done[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return GSA_ERR_SHAPE;
  if (!done[dev]) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return -static_cast<int>(e);
    done[dev] = true;
  }
  return GSA_OK;
}

template <typename T> int launch_forward(const gsa::DeltaArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(gsa::delta_chunk_kernel<T>, dim3(a.s.slots, a.Hv), dim3(256), 0, s, a);
  if (const int e = launch_status()) return e;
  constexpr size_t lds = gsa::ScanLds<T>::kFwd;
  static_assert(lds <= 160 * 1024);
  if (const int e = allow_lds<gsa::delta_scan_kernel<T>>(lds)) return e;
  hipLaunchKernelGGL(gsa::delta_scan_kernel<T>, dim3(a.s.N, a.Hv), dim3(512), lds, s, a);
  return launch_status();
}
template <typename T> int launch_backward(const gsa::DeltaArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(gsa::delta_chunk_kernel<T>, dim3(a.s.slots, a.Hv), dim3(256), 0, s, a);
  if (const int e = launch_status()) return e;
  constexpr size_t lds = gsa::ScanLds<T>::kBwd, lds_grads = gsa::GradLds<T>::kBytes;
  static_assert(lds <= 160 * 1024 && lds_grads <= 160 * 1024);
  if (const int e = allow_lds<gsa::delta_scan_bwd_kernel<T>>(lds)) return e;
  if (const int e = allow_lds<gsa::delta_grads_kernel<T>>(lds_grads)) return e;
  hipLaunchKernelGGL(gsa::delta_scan_bwd_kernel<T>, dim3(a.s.N, a.Hv), dim3(512), lds, s, a);
  if (const int e = launch_status()) return e;
  hipLaunchKernelGGL(gsa::delta_grads_kernel<T>, dim3(a.s.slots, a.Hk), dim3(256), lds_grads, s, a);
  return launch_status();
}

int delta_args(const gsa_delta_args* x, bool backward, gsa::DeltaArgs& a, DeltaSizes& z) {
  if (!x || !x->q || !x->k || !x->v || !x->g || !x->beta || !x->ws) return GSA_ERR_NULL;
  if (backward ? !x->dout || !x->dq || !x->dk || !x->dv || !x->dg || !x->dbeta || !x->saved : !x->o) return GSA_ERR_NULL;
  if (!dtype_size(x->dtype) || !dtype_size(x->beta_dtype)) return GSA_ERR_DTYPE;
  if (x->B < 1 || x->T < 1 || x->N < 1 || x->Hk < 1 || x->Hv < x->Hk || x->Hv % x->Hk || x->Hv > 65535 || x->d != 128)
    return GSA_ERR_SHAPE;
  if (x->cu_seqlens ? x->B != 1 || (x->cu_bytes != 4 && x->cu_bytes != 8) : x->N != x->B) return GSA_ERR_SHAPE;
  z = delta_sizes(x->B, x->T, x->N, x->cu_seqlens != nullptr, x->Hv, x->dtype);
  if (!z.slots) return GSA_ERR_SHAPE;
  const size_t need = 2 * z.tm + z.gates + (backward ? z.s0 + z.u : 0);
  if (x->ws_bytes < need || (x->saved && x->saved_bytes < z.s0 + z.u)) return GSA_ERR_SHAPE;
  auto vec = [&](const void* p, int64_t sb, int64_t st, int64_t sh) {
    return vec_ok(p, sb, st, x->dtype) && sh % (x->dtype == GSA_DTYPE_BF16 ? 8 : 4) == 0;
  };
  if (!vec(x->q, x->q_sb, x->q_st, x->q_sh) || !vec(x->k, x->k_sb, x->k_st, x->k_sh) || !vec(x->v, x->v_sb, x->v_st, x->v_sh) ||
      (backward && !vec(x->dout, x->do_sb, x->do_st, x->do_sh)))
    return GSA_ERR_ALIGN;
  for (const void* p : {(const void*)x->o, (const void*)x->dq, (const void*)x->dk, (const void*)x->dv, (const void*)x->state_in,
                        (const void*)x->state_out, (const void*)x->dstate_in, (const void*)x->dstate_out, (const void*)x->saved,
                        (const void*)x->ws})
    if (p && !aligned(p, 16)) return GSA_ERR_ALIGN;
  if (!aligned(x->g, 4) || !aligned(x->dg, 4) || !aligned(x->beta, dtype_size(x->beta_dtype)) ||
      !aligned(x->dbeta, dtype_size(x->beta_dtype)) || (x->cu_seqlens && !aligned(x->cu_seqlens, x->cu_bytes)))
    return GSA_ERR_ALIGN;
  a = gsa::DeltaArgs{};
  a.s = {x->cu_seqlens, x->cu_bytes == 8, x->N, x->T, (int)z.slots};
  a.q = {x->q, x->q_sb, x->q_st, x->q_sh};
  a.k = {x->k, x->k_sb, x->k_st, x->k_sh};
  a.v = {x->v, x->v_sb, x->v_st, x->v_sh};
  a.g = {x->g, x->g_sb, x->g_st, x->g_sh};
  a.beta = {x->beta, x->beta_sb, x->beta_st, x->beta_sh};
  a.beta_bf16 = x->beta_dtype == GSA_DTYPE_BF16;
  a.Hk = x->Hk;
  a.Hv = x->Hv;
  a.scale = x->scale;
  a.state_in = x->state_in;
  a.o = x->o;
  a.state_out = x->state_out;
  char* w = static_cast<char*>(x->ws);
  a.tm = reinterpret_cast<float*>(w);
  a.pm = reinterpret_cast<float*>(w + z.tm);
  a.gates = reinterpret_cast<float*>(w + 2 * z.tm);
  if (x->saved) {
    a.s0 = static_cast<float*>(x->saved);
    a.u = reinterpret_cast<float*>(static_cast<char*>(x->saved) + z.s0);
  }
  if (backward) {
    a.dout = {x->dout, x->do_sb, x->do_st, x->do_sh};
    a.dstate_out = x->dstate_out;
    a.ds1 = reinterpret_cast<float*>(w + 2 * z.tm + z.gates);
    a.dr = reinterpret_cast<float*>(w + 2 * z.tm + z.gates + z.s0);
    a.dq = x->dq;
    a.dk = x->dk;
    a.dv = x->dv;
    a.dg = x->dg;
    a.dbeta = x->dbeta;
    a.dstate_in = x->dstate_in;
  }
  return GSA_OK;
}

}  // namespace
}  // namespace gsa_host

extern "C" size_t gsa_delta_rule_workspace_bytes(int B, int T, int N, int packed, int Hv, int dtype, int backward) {
  const auto z = gsa_host::delta_sizes(B, T, N, packed, Hv, dtype);
  return z.slots ? 2 * z.tm + z.gates + (backward ? z.s0 + z.u : 0) : 0;
}
extern "C" size_t gsa_delta_rule_saved_bytes(int B, int T, int N, int packed, int Hv, int dtype) {
  const auto z = gsa_host::delta_sizes(B, T, N, packed, Hv, dtype);
  return z.slots ? z.s0 + z.u : 0;
}
extern "C" int gsa_delta_rule(const gsa_delta_args* x, void* stream) {
  gsa::DeltaArgs a;
  gsa_host::DeltaSizes z;
  if (const int e = gsa_host::delta_args(x, false, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  return x->dtype == GSA_DTYPE_BF16 ? gsa_host::launch_forward<uint16_t>(a, s) : gsa_host::launch_forward<float>(a, s);
}
extern "C" int gsa_delta_rule_backward(const gsa_delta_args* x, void* stream) {
  gsa::DeltaArgs a;
  gsa_host::DeltaSizes z;
  if (const int e = gsa_host::delta_args(x, true, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  return x->dtype == GSA_DTYPE_BF16 ? gsa_host::launch_backward<uint16_t>(a, s) : gsa_host::launch_backward<float>(a, s);
}
