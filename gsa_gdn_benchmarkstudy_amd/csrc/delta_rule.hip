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
#include "chunks.h"

namespace gsa {

struct DeltaArgs {
  Seqs s;
  Rows q, k, v, g, beta;
  int beta_bf16, Hk, Hv;
  float scale;
  const float* state_in;      // [N, Hv, 128, 128], nullable
  void* o;                    // [B, T, Hv, 128]
  float* state_out;           // nullable
  // A chunk's operands in the order in which the lanes of the scan take them, a 1 KiB unit an
  // operand part: 64 lanes' 16 bytes.
  char* tm;                   // [slots][Hv]: Tm (the backward pass: transposed)
  char* pm;                   // [slots][Hv]: P (transposed)
  float* gates;               // [slots][Hv] units: e^G, e^(G_C - G), beta [C] each
  float* sums;                // [slots][Hv][2][C]: G log2 e (upper and lower part); the backward pass only
  char *kr, *qr;              // [slots][Hk]: K, Q (fp32 inputs; bf16 rows are read from where they are)
  // The scan cut into segments of seg chunks (0: sequences in one piece), [segments][Hv][128][128] each
  int seg, units;             // units: heads of all sequences, or of all segments
  float* move;                // a segment's product of transitions
  float* add;                 // its state from a start of 0 (the first: from state_in)
  float* init;                // the state before it (backward: the gradient behind it)
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

// ---------------------------------------------------------------------------
// The operands of every chunk and v head (with kBwd those of the backward scan): 256 threads.
// 16384 tokens of 16 heads in bf16: 68 us (0.2 GB).  Bound by latency and issue: eight steps that wait
// for each other (products, the inverse by blocks), four blocks a CU (five, with a smaller A: the same);
// the VALU, mostly splits, is busy for half of the time.
// ---------------------------------------------------------------------------
// e^(G_i - G_j) from the difference of the sums in units of log2: one instruction, right to its last bit
// but one (under 2^-126 it may be 0), where expf takes 20; the difference rounds as one of G's would.
__device__ __forceinline__ float decay(float x) { return __builtin_amdgcn_exp2f(x); }
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

// Units of a chunk's operands.  P enters the output alone in the forward pass: for bf16 outputs
// two parts (2^-17 of it) do; the backward pass sums it into states.
template <typename T, bool kBwd> struct Pack {
  static constexpr int C = ChunkType<T>::kChunk, NP = ChunkType<T>::kParts;
  static constexpr int kPParts = kBwd || NP == 3 ? 3 : 2;
  static constexpr int kT = Square<C>::kFrags * 3, kP = Square<C>::kFrags * kPParts;
  static constexpr int kRows = (C / 16) * 4 * NP;
};

// [C][ld] fp32 matrix in LDS -> its operands of kN parts in global memory.
template <int C, int kN, bool kTransposed>
__device__ __forceinline__ void pack_square(char* dst, const float* x, int ld, int tid) {
  for (int u = tid; u < Square<C>::kFrags * 64; u += 256) {
    const int l = u & 63, f = u >> 6;
    const int2 w = Square<C>::of(f, kTransposed);
    const int t = tile_row(w.x, l & 15), j = 32 * w.y + 8 * (l >> 4);
    float y[8];
    if constexpr (kTransposed) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[(j + e) * ld + t];
    } else {
      load8(x + t * ld + j, y);
    }
    const Parts<3> p = split3(y);
#pragma unroll
    for (int n = 0; n < kN; ++n) *reinterpret_cast<bf16x8*>(dst + (f * kN + n) * kUnit + 16 * l) = p.p[n];
  }
}
template <typename T, bool kBwd>
__global__ __launch_bounds__(256) void delta_chunk_kernel(DeltaArgs a) {
  using K = Pack<T, kBwd>;
  constexpr int C = K::C, NP = K::NP, MT = C / 16, LD = C + 4;
  constexpr int kStage = K::kRows * kUnit, kX = C * LD * 4 > kStage ? C * LD * 4 : kStage;
  __shared__ __align__(16) float am[C][LD];                  // P, then A
  __shared__ __align__(16) char xbuf[kX];                    // K's rows, then the inverse
  __shared__ __align__(16) float ybuf[C == 32 ? 16 * LD : 1];
  __shared__ float gh[C], gl[C], bt[C];
  __shared__ int first;                                      // the first row of A that is not finite
  float (*xm)[LD] = reinterpret_cast<float (*)[LD]>(xbuf);
  bf16x8* sk = reinterpret_cast<bf16x8*>(xbuf);
  const int slot = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, share = a.Hv / a.Hk, hk = h / share, tid = threadIdx.x, wave = tid >> 6, l = lane_id();
  const int g4 = l >> 4, m = l & 15, rs = row_slot(g4, m);
  int c;
  const Span sp = slot_of(a.s, slot, C, c);
  if (c < 0) return;
  const int64_t t0 = (int64_t)c * C;
  const int left = sp.len - (int)t0;                         // tokens of the chunk (more than C: C)
  const int64_t at = (int64_t)slot * a.Hv + h, atk = (int64_t)slot * a.Hk + hk;

  stage_rows<T>(sk, a.k, sp, t0, left, hk, tid);
  if (tid == 0) first = C;
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
    const double G2 = G * 1.4426950408889634074;             // log2 e: the decays between tokens are powers of 2 (decay)
    const float hi = (float)G2, lo = (float)(G2 - (double)hi);
    if (l < C) {
      gh[l] = hi;
      gl[l] = lo;
      bt[l] = b;
      float* gates = a.gates + at * (kUnit / 4);
      gates[l] = expf((float)G);
      gates[C + l] = ok ? expf((float)(Ge - G)) : 0.f;        // (nothing comes from behind the sequence)
      gates[2 * C + l] = b;
      if (kBwd) {
        a.sums[at * 2 * C + l] = hi;
        a.sums[at * 2 * C + C + l] = lo;
      }
    }
  }
  if constexpr (NP == 3) {
    if (h % share == 0) {                                    // one of the heads that share q and k
      stage_rows<T>(reinterpret_cast<bf16x8*>(a.kr + atk * K::kRows * kUnit), a.k, sp, t0, left, hk, tid);
      stage_rows<T>(reinterpret_cast<bf16x8*>(a.qr + atk * K::kRows * kUnit), a.q, sp, t0, left, hk, tid);
    }
  }
  Parts<NP> xq[4];
  const int mt = wave % MT;                                  // rows of this wave (C = 32: waves 2, 3 take Q K^T)
  {
    const int t = tile_row(mt, m);
    const T* p = row_at<T>(a.q, sp, t0 + t, hk);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) xq[ks] = operand<T>(p + 32 * ks + 8 * g4, t < left);
  }
  __syncthreads();

  // row tile mt of Q K^T (into am, packed as P) and of K K^T (into am behind it)
  floatx4 kk[MT];
  float odd = 0.f;
#pragma unroll
  for (int nt = 0; nt < MT; ++nt) {
    if ((nt >> 1) > (mt >> 1)) continue;                     // (the upper right half is not read)
    const int j = tile_row(nt, m);
    floatx4 qk = {0.f, 0.f, 0.f, 0.f};
    kk[nt] = qk;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const Parts<NP> kj = staged<NP>(sk, nt * 4 + ks, rs);
      if (C == 64 || wave < MT) mma(kk[nt], staged<NP>(sk, mt * 4 + ks, rs), kj);
      if (C == 64 || wave >= MT) mma(qk, xq[ks], kj);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = tile_row(mt, 4 * g4 + r);
      const float d = j <= i ? decay((gh[i] - gh[j]) + (gl[i] - gl[j])) : 0.f;
      if (C == 64 || wave >= MT) am[i][j] = j <= i ? a.scale * qk[r] * d : 0.f;
      kk[nt][r] = j < i ? bt[i] * kk[nt][r] * d : 0.f;
      odd = __builtin_fmaf(kk[nt][r], 0.f, odd);
    }
  }
  if (odd != 0.f)                                            // a NaN or an infinity: the tokens before it do without
#pragma unroll
    for (int nt = 0; nt < MT; ++nt)
      if ((nt >> 1) <= (mt >> 1))
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (kk[nt][r] * 0.f != 0.f) atomicMin(&first, tile_row(mt, 4 * g4 + r));
  __syncthreads();
  const int cut = first;
  pack_square<C, K::kPParts, kBwd>(a.pm + at * K::kP * kUnit, &am[0][0], LD, tid);
  for (int i = tid; i < C / 32 * 256; i += 256)              // above the diagonal of 32 by 32: 0
    xm[32 * (i >> 8) + (i >> 4 & 15)][32 * (i >> 8) + 16 + (i & 15)] = 0.f;
  __syncthreads();
  if (C == 64 || wave < MT)
#pragma unroll
    for (int nt = 0; nt < MT; ++nt)
      if ((nt >> 1) <= (mt >> 1))
#pragma unroll
        for (int r = 0; r < 4; ++r) am[tile_row(mt, 4 * g4 + r)][tile_row(nt, m)] = tile_row(mt, 4 * g4 + r) < cut ? kk[nt][r] : 0.f;
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
      for (int k = 0; k < i; ++k) s = __builtin_fmaf(-am[16 * wave + i][16 * wave + k], x[k], s);
      x[i] = s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) xm[16 * wave + i][16 * wave + l] = x[i];
  }
  // products on the way: in the upper right of the inverse, which no operand takes (C = 32: beside it)
  float* ym = C == 32 ? ybuf : &xm[0][32];
  __syncthreads();
  if (wave < C / 32) {
    const int p = 32 * wave;
    tile_put(ym + 16 * wave * LD, LD, tile_f32(&am[p + 16][p], LD, &xm[p][p], LD, 16), 1.f);
  }
  __syncthreads();
  if (wave < C / 32) {
    const int p = 32 * wave;
    tile_put(&xm[p + 16][p], LD, tile_f32(&xm[p + 16][p + 16], LD, ym + 16 * wave * LD, LD, 16), -1.f);
  }
  __syncthreads();
  if constexpr (C == 64) {
    const int i = 16 * (wave >> 1), j = 16 * (wave & 1);
    tile_put(ym + i * LD + j, LD, tile_f32(&am[32 + i][0], LD, &xm[0][j], LD, 32), 1.f);
    __syncthreads();
    tile_put(&xm[32 + i][j], LD, tile_f32(&xm[32 + i][32], LD, ym + j, LD, 32), -1.f);
    __syncthreads();
  }
  if (cut < C) {                                             // (the same for all)
    for (int i = tid; i < C * C; i += 256)
      if (i / C >= cut && i % C <= i / C) xm[i / C][i % C] = __builtin_nanf("");
    __syncthreads();
  }
  pack_square<C, 3, kBwd>(a.tm + at * K::kT * kUnit, &xm[0][0], LD, tid);
}

// ---------------------------------------------------------------------------
// The state from chunk to chunk.  A wave owns 16 columns of one head's state in 8 tiles of 16,
// tile 2 ks + e of its registers the rows tile_row(2 ks + e, .); a block has W waves.  The chunk's
// operands come to LDS by direct loads.  Three shapes (Shape), by how many heads and sequences
// there are to fill the chip:
//   <8, one buffer>: a head a block; two blocks share a CU and cover each other's waits, each
//     buffer is refilled as soon as all waves are through with it
//   <8, two buffers> and <4, two buffers>: a head and half a head a block, one block a CU; the
//     next chunk's operands are on their way during the whole of this one's products
// Bound by the issue of instructions, the matrix ones and the splits of fp32 into bf16 parts, which
// do not overlap within a SIMD, where four waves share it (the segments' passes: three quarters of its
// cycles at 4 x 4096 tokens of 16 heads); the outputs' scan has two, and of its cycles 28 % are the matrix
// instructions', some 30 % the VALU's, the others go with waits for V, LDS and at the barriers.  A
// chunk of 64 takes 4.1 us by half heads, 5.9 by whole ones (8 on a full chip), 13 where two blocks
// share a CU.
// ---------------------------------------------------------------------------
template <int W_, bool kDouble_, int kWaves_ = 2> struct Shape {
  static constexpr int NT = 1, W = W_, kCols = 16 * NT * W_, kBlocks = kHead / kCols;     // columns of a block, blocks of a head
  static constexpr bool kDouble = kDouble_;
  static constexpr int kWaves = kWaves_;                     // of a SIMD (a head by 4 waves of 2 tiles was slower)
};

// A wave's own [C][16 NT] of a [tokens][128] matrix in LDS: token 8 a + b in row b C / 8 + a, so that a
// column's four groups of tokens lie side by side.
template <typename T, int NT> struct Slice {
  static constexpr int C = ChunkType<T>::kChunk, kRow = 16 * NT * sizeof(T), kPieces = kRow / 16, kBytes = C * kRow;
  __device__ static int token(int row) { return row % (C / 8) * 8 + row / (C / 8); }
  // bytes from the lane's place (token 8 g, column m) to token 8 g + tile_at(t, r), column 16 n + m
  static constexpr int at(int t, int r, int n) { return ((4 * (t & 1) + r) * (C / 8) + 4 * (t >> 1)) * kRow + 16 * n * (int)sizeof(T); }
  __device__ static int lane(int g, int m) { return g * kRow + m * (int)sizeof(T); }
  // p: the wave's columns of the chunk's first row (uniform), `stride` elements between rows
  __device__ static void fetch(const T* p, int64_t stride, int left, uint32_t lds, int l) {
  #pragma unroll
    for (int i = 0; i < kBytes / kUnit; ++i) {
      const int u = 64 * i + l, t = min(token(u / kPieces), left - 1);
      load_lds16(p, (uint32_t)(t * (int)stride) * (uint32_t)sizeof(T) + 16 * (u % kPieces), __builtin_amdgcn_readfirstlane(lds + i * kUnit));
    }
  }
  __device__ static void store(const char* lds, T* out, int64_t stride, int left, int l) {
#pragma unroll
    for (int i = 0; i < kBytes / kUnit; ++i) {
      const int u = 64 * i + l, t = token(u / kPieces);
      const u32x4 x = *reinterpret_cast<const u32x4*>(lds + 16 * u);
      if (t < left) *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(out + t * stride) + 16 * (u % kPieces)) = x;
    }
  }
};

template <typename T, typename Sh> struct ScanLds {
  using F = Pack<T, false>;
  using B = Pack<T, true>;
  static constexpr int kSlices = Slice<T, Sh::NT>::kBytes * Sh::W;
  // forward: K | Tm | gates | V, then O | Q | P (a pass for the state alone: without the last two)
  static constexpr int kState = (F::kRows + F::kT + 1) * kUnit + kSlices, kOne = kState + (F::kRows + F::kP) * kUnit;
  // backward: K | Q | Tm^T, then dv where it fits | P^T | gates | dv
  static constexpr bool kDvInT = kSlices <= B::kT * kUnit;
  static constexpr int kOneBwd = (2 * B::kRows + B::kT + B::kP + 1) * kUnit + (kDvInT ? 0 : kSlices);
  static constexpr size_t kFwd = (size_t)kOne * (Sh::kDouble ? 2 : 1), kBwd = (size_t)kOneBwd * (Sh::kDouble ? 2 : 1);
};

// kOut: the outputs (and what the backward pass needs).  Otherwise only what a segment does to
// the state: blockIdx.y 0 what it adds, 1 its product of transitions (V = 0 from the
// identity).
template <typename T, bool kOut, typename Sh>
__global__ __launch_bounds__(64 * Sh::W, Sh::kWaves) void delta_scan_kernel(DeltaArgs a) {
  using K = Pack<T, false>;
  using L = ScanLds<T, Sh>;
  constexpr int C = K::C, NP = K::NP, MT = C / 16, JS = C / 32, NT = Sh::NT, W = Sh::W;
  using V = Slice<T, NT>;
  extern __shared__ __align__(16) char lds[];
  int bk, bt, bg, bv, bq, bp;                                // this chunk's, bytes from lds
  const uint32_t base = lds_addr(lds);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), g = l >> 4;
  auto buffers = [&](int which) {
    bk = Sh::kDouble ? which * L::kOne : 0;
    bt = bk + K::kRows * kUnit;
    bg = bt + K::kT * kUnit;
    bv = bg + kUnit + wave * V::kBytes;
    bq = bg + kUnit + L::kSlices;
    bp = bq + K::kRows * kUnit;
  };
  buffers(0);
  const int2 unit = unit_of<Sh::kBlocks>(blockIdx.x);
  const int piece_slot = unit.x / a.Hv, h = unit.x % a.Hv, hk = h / (a.Hv / a.Hk), col0 = unit.y * Sh::kCols + 16 * NT * wave;
  if (unit.x >= a.units) return;
  int piece = 0, c0 = 0, c1;
  Span sp;
  if (a.seg) {
    sp = slot_of(a.s, piece_slot, C * a.seg, piece);
    if (piece < 0) return;
    c0 = piece * a.seg;
  } else {
    sp = span_of(a.s, piece_slot, C);
  }
  const int chunks = (sp.len + C - 1) / C;
  const bool last = !a.seg || c0 + a.seg >= chunks;
  c1 = last ? chunks : c0 + a.seg;
  const bool ident = !kOut && blockIdx.y == 1;
  if (!kOut && (last || (ident && piece == 0))) return;      // nobody asks for it
  const int slot0 = a.s.cu ? span_of(a.s, sp.n, C).slot0 : sp.n * chunks;
  const int64_t sn = ((int64_t)sp.n * a.Hv + h) * kHead * kHead, gn = ((int64_t)piece_slot * a.Hv + h) * kHead * kHead;

  floatx4 S[8][NT];
  const float* from = piece == 0 ? (a.state_in ? a.state_in + sn : nullptr) : kOut ? a.init + gn : nullptr;
  if (from) {
    tiles_load(S, from, col0, l);
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          S[t][n][r] = ident && tile_row(t, 4 * g + r) == col0 + 16 * n + (l & 15) ? 1.f : 0.f;
  }

  auto lane = [&]() { return Sh::kDouble || !kOut ? l : here(l); };   // (two blocks a CU: 128 registers)
  auto fetch_k = [&](int64_t t0, int left, int64_t atk) {
    if constexpr (NP == 1) fetch_rows<C, W>(a.k, sp, t0, left, hk, base + bk, wave, lane());
    else fetch<W>(a.kr + atk * K::kRows * kUnit, base + bk, K::kRows, wave, l);
  };
  auto fetch_q = [&](int64_t t0, int left, int64_t atk) {
    if constexpr (NP == 1) fetch_rows<C, W>(a.q, sp, t0, left, hk, base + bq, wave, lane());
    else fetch<W>(a.qr + atk * K::kRows * kUnit, base + bq, K::kRows, wave, l);
  };
  constexpr int kSome = NP == 1 ? 4 : 2;
  const int rs = row_slot(g, l & 15), place = cols_place(l);
  auto slice = [&]() { return V::lane(lane() >> 4, lane() & 15); };
  auto fetch_v = [&](int64_t t0, int left) {
    if (!ident) V::fetch(uniform(row_at<T>(a.v, sp, t0, h) + col0), a.v.st, left, base + bv, lane());
  };
  auto fetch_all = [&](int c) {
    const int64_t t0 = (int64_t)c * C, at = (int64_t)(slot0 + c) * a.Hv + h, atk = (int64_t)(slot0 + c) * a.Hk + hk;
    const int left = sp.len - (int)t0;
    fetch_k(t0, left, atk);
    fetch_v(t0, left);
    fetch<W>(a.gates + at * (kUnit / 4), base + bg, 1, wave, l);
    if (kOut) fetch_q(t0, left, atk);
    fetch<W>(a.tm + at * K::kT * kUnit, base + bt, K::kT, wave, l);
    if (kOut) fetch<W>(a.pm + at * K::kP * kUnit, base + bp, K::kP, wave, l);
  };
  if (c0 < c1) fetch_all(c0);
  for (int c = c0; c < c1; ++c) {
    const int64_t t0 = (int64_t)c * C, at = (int64_t)(slot0 + c) * a.Hv + h, atk = (int64_t)(slot0 + c) * a.Hk + hk;
    const int left = sp.len - (int)t0;
    const bool more = c + 1 < c1;
    const int64_t t1 = t0 + C;
    const int left1 = left - C;
    wait_loads();
    __syncthreads();
    if constexpr (Sh::kDouble) {
      if (more) {
        buffers((c - c0 + 1) & 1);
        fetch_all(c + 1);
      }
      buffers((c - c0) & 1);
    }
    if (kOut && a.s0) tiles_store(S, a.s0 + at * kHead * kHead, col0, l);

    const bf16x8* st = reinterpret_cast<const bf16x8*>(lds + bt);
    const bf16x8* spm = reinterpret_cast<const bf16x8*>(lds + bp);
    const float* gates = reinterpret_cast<const float*>(lds + bg);
    floatx4 X[MT][NT], O[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n) X[mt][n] = O[mt][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    Parts<3> s[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = split_pair(S[0][n], S[1][n]);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      Parts<NP> k[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) k[mt] = rows_of<NP>(lds + bk, mt, ks, rs);
      Parts<3> next[NT];
      if (ks < 3)
#pragma unroll
        for (int n = 0; n < NT; ++n) next[n] = split_pair(S[2 * ks + 2][n], S[2 * ks + 3][n]);
      mma_grid(X, k, s);
      if constexpr (kOut) {
        // for a bf16 output two parts of the state do (2^-17 of it)
        constexpr int kS = NP == 1 ? 2 : 3;
        Parts<kS> x[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < kS; ++i) x[n].p[i] = s[n].p[i];
        Parts<NP> q[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) q[mt] = rows_of<NP>(lds + bq, mt, ks, rs);
        mma_grid(O, q, x);
      }
      __builtin_amdgcn_sched_barrier(0);                     // (later steps' operands are not read ahead into registers)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n] = next[n];
    }
    if (kOut && more && !Sh::kDouble) {
      __syncthreads();                                       // Q is free
      fetch_q(t1, left1, atk + a.Hk);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const floatx4 e = *reinterpret_cast<const floatx4*>(gates + 8 * g + tile_at(mt, 0));
      const floatx4 b = *reinterpret_cast<const floatx4*>(gates + 2 * C + 8 * g + tile_at(mt, 0));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = ident ? 0.f : to_f32(*reinterpret_cast<const T*>(lds + bv + slice() + V::at(mt, r, n)));
          X[mt][n][r] = b[r] * (v - e[r] * X[mt][n][r]);     // R (behind the sequence beta is 0)
          if (kOut) O[mt][n][r] *= a.scale * e[r];
        }
    }
    // A NaN or an infinity in a column of R: the rows before it are computed without it (a product's zeros above the
    // diagonal would carry it there), the others become NaN.  The first such row waits in the place of the wave's V.
    // (The search costs 1 to 2 % of the half heads' scan, nothing by heads.)
    auto note = [&](int n) { return reinterpret_cast<int*>(lds + bv) + 64 * n + here(l); };
    auto fill = [&](floatx4 (&x)[MT][NT], float with) {
      asm volatile("" ::: "memory");
      const int g8 = here(8 * g);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int bad = *note(n);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[mt][n][r] = g8 + tile_at(mt, r) >= bad ? with : x[mt][n][r];
      }
      asm volatile("" ::: "memory");
    };
    bool any = false;
    if constexpr (kOut) {
      float odd = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) odd = __builtin_fmaf(X[mt][n][r], 0.f, odd);
      any = __builtin_amdgcn_ballot_w64(odd != 0.f) != 0;
      if (__builtin_expect(any, 0)) {
        asm volatile("" ::: "memory");
        const int g8 = here(8 * g);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          int bad = C;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (X[mt][n][r] * 0.f != 0.f) bad = min(bad, g8 + tile_at(mt, r));
          bad = min(bad, __shfl_xor(bad, 16, 64));
          *note(n) = min(bad, __shfl_xor(bad, 32, 64));
        }
        fill(X, 0.f);
      }
    }
    floatx4 U[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n) U[mt][n] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      Parts<3> r[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) r[n] = split_pair(X[2 * js][n], X[2 * js + 1][n]);
#pragma unroll
      for (int mt = 2 * js; mt < MT; mt += 2) {
        const Parts<3> x[2] = {staged<3>(st, Square<C>::at(mt, js, false), l), staged<3>(st, Square<C>::at(mt + 1, js, false), l)};
        mma_grid(U + mt, x, r);
      }
    }
    if (!Sh::kDouble) __syncthreads();                       // Tm is free
    if (more && !Sh::kDouble) fetch<W>(a.tm + (at + a.Hv) * K::kT * kUnit, base + bt, K::kT, wave, l);
    if constexpr (kOut) {
      if (__builtin_expect(any, 0)) fill(U, 0.f);
#pragma unroll
      for (int js = 0; js < JS; ++js) {
        Parts<K::kPParts> u[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const Parts<3> p = split_pair(U[2 * js][n], U[2 * js + 1][n]);
#pragma unroll
          for (int i = 0; i < K::kPParts; ++i) u[n].p[i] = p.p[i];
        }
#pragma unroll
        for (int mt = 2 * js; mt < MT; mt += 2) {
          const Parts<K::kPParts> x[2] = {staged<K::kPParts>(spm, Square<C>::at(mt, js, false), l),
                                          staged<K::kPParts>(spm, Square<C>::at(mt + 1, js, false), l)};
          mma_grid(O + mt, x, u);
        }
      }
      if (__builtin_expect(any, 0)) {
        fill(U, __builtin_nanf(""));
        fill(O, __builtin_nanf(""));
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            *reinterpret_cast<T*>(lds + bv + slice() + V::at(mt, r, n)) = from_f32<T>(O[mt][n][r]);
      if (a.u) tiles_store(U, a.u + at * C * kHead, col0, l);
      asm volatile("" ::: "memory");                         // (a wave's LDS accesses keep their order)
      V::store(lds + bv, static_cast<T*>(a.o) + (((int64_t)sp.b * a.s.T + sp.t0 + t0) * a.Hv + h) * kHead + col0, (int64_t)a.Hv * kHead,
               left, lane());
    }
    if (more && !Sh::kDouble) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the wave has read its slice
      fetch_v(t1, left1);
    }
    const float whole = gates[C - 1];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][n][r] *= whole;
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      Parts<3> u[NT];
      float d[8];
      load8(gates + C + 32 * js + 8 * g, d);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = U[2 * js + (e >> 2)][n][e & 3] * d[e];
        u[n] = split3(x);
      }
#pragma unroll
      for (int t = 0; t < 8; t += kSome) {
        Parts<NP> k[kSome];
#pragma unroll
        for (int i = 0; i < kSome; ++i) k[i] = cols_of<NP>(lds + bk, t + i, js, place);
        mma_grid(S + t, k, u);
      }
    }
    if (!Sh::kDouble) __syncthreads();                       // all buffers but Q, Tm and V are free
    if (more && !Sh::kDouble) {
      fetch_k(t1, left1, atk + a.Hk);
      if (kOut) fetch<W>(a.pm + (at + a.Hv) * K::kP * kUnit, base + bp, K::kP, wave, l);
      fetch<W>(a.gates + (at + a.Hv) * (kUnit / 4), base + bg, 1, wave, l);
    }
  }
  if (kOut ? last && a.state_out != nullptr : true)
    tiles_store(S, kOut ? a.state_out + sn : (ident ? a.move : a.add) + gn, col0, l);
}

// kOut: dv, and the gradients of the states behind the chunks and of R that the last kernel reads.
// Otherwise what a segment adds to the gradient of the state before it.
template <typename T, bool kOut, typename Sh>
__global__ __launch_bounds__(64 * Sh::W, Sh::kWaves) void delta_scan_bwd_kernel(DeltaArgs a) {
  using K = Pack<T, true>;
  using L = ScanLds<T, Sh>;
  constexpr int C = K::C, NP = K::NP, MT = C / 16, JS = C / 32, NT = Sh::NT, W = Sh::W;
  extern __shared__ __align__(16) char lds[];
  using V = Slice<T, NT>;
  int bk, bq, bt, bp, bg, bv;                                // this chunk's, bytes from lds
  const uint32_t base = lds_addr(lds);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), g = l >> 4;
  auto buffers = [&](int which) {
    bk = Sh::kDouble ? which * L::kOneBwd : 0;
    bq = bk + K::kRows * kUnit;
    bt = bq + K::kRows * kUnit;
    bp = bt + K::kT * kUnit;
    bg = bp + K::kP * kUnit;
    bv = (L::kDvInT ? bt : bg + kUnit) + wave * V::kBytes;
  };
  buffers(0);
  const int2 unit = unit_of<Sh::kBlocks>(blockIdx.x);
  const int piece_slot = unit.x / a.Hv, h = unit.x % a.Hv, hk = h / (a.Hv / a.Hk), col0 = unit.y * Sh::kCols + 16 * NT * wave;
  if (unit.x >= a.units) return;
  int piece = 0, c0 = 0;
  Span sp;
  if (a.seg) {
    sp = slot_of(a.s, piece_slot, C * a.seg, piece);
    if (piece < 0) return;
    c0 = piece * a.seg;
  } else {
    sp = span_of(a.s, piece_slot, C);
  }
  const int chunks = (sp.len + C - 1) / C;
  const bool last = !a.seg || c0 + a.seg >= chunks;
  const int c1 = last ? chunks : c0 + a.seg;
  if (!kOut && piece == 0) return;                           // nobody asks for it
  const int slot0 = a.s.cu ? span_of(a.s, sp.n, C).slot0 : sp.n * chunks;
  const int64_t sn = ((int64_t)sp.n * a.Hv + h) * kHead * kHead, gn = ((int64_t)piece_slot * a.Hv + h) * kHead * kHead;

  floatx4 S[8][NT];                                           // dS
  const float* from = last ? (a.dstate_out ? a.dstate_out + sn : nullptr) : kOut ? a.init + gn : nullptr;
  if (from) {
    tiles_load(S, from, col0, l);
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) S[t][n] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  T d[MT][NT][4];                                            // dO as it is (turned to fp32 where it is used)
  auto load_do = [&](int64_t t0, int left) {
    const T* p = uniform(row_at<T>(a.dout, sp, t0, h) + col0);
    const uint32_t off = 8 * g * (uint32_t)a.dout.st + (l & 15);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          d[mt][n][r] = 8 * g + tile_at(mt, r) < left ? (p + tile_at(mt, r) * a.dout.st + 16 * n)[off] : T(0);
  };
  auto lane = [&]() { return Sh::kDouble || !kOut ? l : here(l); };   // (two blocks a CU: 128 registers)
  auto fetch_k = [&](int64_t t0, int left, int64_t atk) {
    if constexpr (NP == 1) fetch_rows<C, W>(a.k, sp, t0, left, hk, base + bk, wave, lane());
    else fetch<W>(a.kr + atk * K::kRows * kUnit, base + bk, K::kRows, wave, l);
  };
  auto fetch_q = [&](int64_t t0, int left, int64_t atk) {
    if constexpr (NP == 1) fetch_rows<C, W>(a.q, sp, t0, left, hk, base + bq, wave, lane());
    else fetch<W>(a.qr + atk * K::kRows * kUnit, base + bq, K::kRows, wave, l);
  };
  constexpr int kSome = NP == 1 ? 4 : 2;
  const int rs = row_slot(g, l & 15), place = cols_place(l);
  auto slice = [&]() { return V::lane(lane() >> 4, lane() & 15); };
  auto fetch_all = [&](int c) {
    const int64_t t0 = (int64_t)c * C, at = (int64_t)(slot0 + c) * a.Hv + h, atk = (int64_t)(slot0 + c) * a.Hk + hk;
    const int left = sp.len - (int)t0;
    fetch_k(t0, left, atk);
    fetch<W>(a.gates + at * (kUnit / 4), base + bg, 1, wave, l);
    fetch<W>(a.pm + at * K::kP * kUnit, base + bp, K::kP, wave, l);
    fetch<W>(a.tm + at * K::kT * kUnit, base + bt, K::kT, wave, l);
    fetch_q(t0, left, atk);
  };
  if (c0 < c1) {
    load_do((int64_t)(c1 - 1) * C, sp.len - (c1 - 1) * C);
    fetch_all(c1 - 1);
  }
  for (int c = c1 - 1; c >= c0; --c) {
    const int64_t t0 = (int64_t)c * C, at = (int64_t)(slot0 + c) * a.Hv + h, atk = (int64_t)(slot0 + c) * a.Hk + hk;
    const int left = sp.len - (int)t0;
    const bool more = c > c0;
    wait_loads();
    __syncthreads();
    if constexpr (Sh::kDouble) {
      if (more) {
        buffers((c1 - c) & 1);
        fetch_all(c - 1);
      }
      buffers((c1 - 1 - c) & 1);
    }
    if (kOut) tiles_store(S, a.ds1 + at * kHead * kHead, col0, l);

    const bf16x8* st = reinterpret_cast<const bf16x8*>(lds + bt);
    const bf16x8* spm = reinterpret_cast<const bf16x8*>(lds + bp);
    const float* gates = reinterpret_cast<const float*>(lds + bg);
    floatx4 X[MT][NT], R[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NT; ++n) X[mt][n] = R[mt][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    Parts<3> s[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = split_pair(S[0][n], S[1][n]);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      Parts<NP> k[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) k[mt] = rows_of<NP>(lds + bk, mt, ks, rs);
      Parts<3> next[NT];
      if (ks < 3)
#pragma unroll
        for (int n = 0; n < NT; ++n) next[n] = split_pair(S[2 * ks + 2][n], S[2 * ks + 3][n]);
      mma_grid(X, k, s);
      __builtin_amdgcn_sched_barrier(0);                     // (later steps' operands are not read ahead into registers)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n] = next[n];
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const floatx4 e = *reinterpret_cast<const floatx4*>(gates + C + 8 * g + tile_at(mt, 0));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) X[mt][n][r] *= e[r];
    }
    // dS <- e^G_C dS + Q^T (scale e^G dO), then dU <- dU + P^T dO: dO's registers are free behind it
    const float whole = gates[C - 1];
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][n][r] *= whole;
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      Parts<NP> p[NT];
      Parts<3> ps[NT];
      float e[8];
      load8(gates + 32 * js + 8 * g, e);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(d[2 * js + (i >> 2)][n][i & 3]);
        p[n] = parts_of<NP>(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= a.scale * e[i];
        ps[n] = split3(x);
      }
#pragma unroll
      for (int mt = 0; mt < 2 * js + 2; mt += 2) {           // dU
        const Parts<3> x[2] = {staged<3>(spm, Square<C>::at(mt, js, true), l), staged<3>(spm, Square<C>::at(mt + 1, js, true), l)};
        mma_grid(X + mt, x, p);
      }
#pragma unroll
      for (int t = 0; t < 8; t += kSome) {
        Parts<NP> x[kSome];
#pragma unroll
        for (int i = 0; i < kSome; ++i) x[i] = cols_of<NP>(lds + bq, t + i, js, place);
        mma_grid(S + t, x, ps);
      }
    }
    load_do(more ? t0 - C : t0, more ? left + C : left);     // (no condition: it would be waited for here)
    if (!Sh::kDouble) __syncthreads();                       // Q and P^T are free
    if (more && !Sh::kDouble) {
      fetch<W>(a.pm + (at - a.Hv) * K::kP * kUnit, base + bp, K::kP, wave, l);
      fetch_q(t0 - C, left + C, atk - a.Hk);
    }
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      Parts<3> p[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) p[n] = split_pair(X[2 * js][n], X[2 * js + 1][n]);
#pragma unroll
      for (int mt = 0; mt < 2 * js + 2; mt += 2) {           // dR
        const Parts<3> x[2] = {staged<3>(st, Square<C>::at(mt, js, true), l), staged<3>(st, Square<C>::at(mt + 1, js, true), l)};
        mma_grid(R + mt, x, p);
      }
    }
    __syncthreads();                                         // Tm^T is read by all: dv goes through its place
    if (kOut) tiles_store(R, a.dr + at * C * kHead, col0, l);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const floatx4 e = *reinterpret_cast<const floatx4*>(gates + 8 * g + tile_at(mt, 0));
      const floatx4 b = *reinterpret_cast<const floatx4*>(gates + 2 * C + 8 * g + tile_at(mt, 0));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (kOut) *reinterpret_cast<T*>(lds + bv + slice() + V::at(mt, r, n)) = from_f32<T>(b[r] * R[mt][n][r]);
          R[mt][n][r] *= -b[r] * e[r];
        }
    }
    if constexpr (kOut) {
      asm volatile("" ::: "memory");                         // (a wave's LDS accesses keep their order)
      V::store(lds + bv, static_cast<T*>(a.dv) + (((int64_t)sp.b * a.s.T + sp.t0 + t0) * a.Hv + h) * kHead + col0, (int64_t)a.Hv * kHead,
               left, lane());
    }
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      Parts<3> q[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) q[n] = split_pair(R[2 * js][n], R[2 * js + 1][n]);
#pragma unroll
      for (int t = 0; t < 8; t += kSome) {
        Parts<NP> x[kSome];
#pragma unroll
        for (int i = 0; i < kSome; ++i) x[i] = cols_of<NP>(lds + bk, t + i, js, place);
        mma_grid(S + t, x, q);
      }
    }
    if (!Sh::kDouble) __syncthreads();                       // K, the gates and dv's place are free
    if (more && !Sh::kDouble) {
      fetch<W>(a.tm + (at - a.Hv) * K::kT * kUnit, base + bt, K::kT, wave, l);
      fetch_k(t0 - C, left + C, atk - a.Hk);
      fetch<W>(a.gates + (at - a.Hv) * (kUnit / 4), base + bg, 1, wave, l);
    }
  }
  if (kOut ? piece == 0 && a.dstate_in != nullptr : true) tiles_store(S, kOut ? a.dstate_in + sn : a.add + gn, col0, l);
}

// The states before the segments (kBwd: the gradients behind them) from what each adds and its
// product of transitions: S <- move S + add (dS <- move^T dS + add), segment after segment.  512
// threads and 16 columns a block: a wave owns the rows tile_row(wave, .), the state goes round
// through LDS.  A wave's rows of move and add come by direct loads, two segments ahead, to places of
// its own (loads to registers that far ahead were waited for at each turn of the loop).  1.9 to 2.4 us a
// segment, most of it the parts of move's rows, which only 16 columns share.
constexpr int kJoinWave = 9 * kUnit;                         // 8 of move, 1 of add
constexpr size_t kJoinLds = 2 * 8 * kJoinWave + 12 * kUnit;
template <bool kBwd>
__global__ __launch_bounds__(512) void delta_join_kernel(DeltaArgs a, int chunk) {
  extern __shared__ __align__(16) char lds[];
  bf16x8* buf = reinterpret_cast<bf16x8*>(lds + 2 * 8 * kJoinWave);          // the state's operands
  const int2 unit = unit_of<8>(blockIdx.x);                  // a head of a sequence, 16 columns
  if (unit.x >= a.s.N * a.Hv) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), g = l >> 4, m = l & 15;
  const int h = unit.x % a.Hv, col = 16 * unit.y + m;
  const Span sp = span_of(a.s, unit.x / a.Hv, chunk * a.seg);
  const int pieces = (sp.len + chunk * a.seg - 1) / (chunk * a.seg);
  if (pieces == 0) {                                         // no token: no segment to hand the state on
    const float* from = kBwd ? a.dstate_out : a.state_in;
    float* to = kBwd ? a.dstate_in : a.state_out;
    if (to)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t o = (((int64_t)sp.n * a.Hv + h) * kHead + tile_row(wave, 4 * g + r)) * kHead + col;
        to[o] = from ? from[o] : 0.f;
      }
  }
  if (pieces < 2) return;
  const int first = kBwd ? pieces - 1 : 0, step = kBwd ? -1 : 1;
  auto at = [&](int i) { return ((int64_t)(sp.slot0 + first + i * step) * a.Hv + h) * kHead * kHead; };   // the i-th segment's matrix
  char* const mine = lds + wave * kJoinWave;
  const uint32_t mine_lds = lds_addr(lds) + wave * kJoinWave;
  // (behind the last segment that is asked for that one again: the waits count on all loads)
  auto fetch = [&](int i) {
    const int64_t o = at(max(min(i, pieces - 2), 1));
    const float* mv = uniform(a.move + o);
    const float* ad = uniform(a.add + o);
    const uint32_t to = mine_lds + (i & 1) * 8 * kJoinWave;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      uint32_t off;
      if constexpr (kBwd) {                                  // 16 columns, row 8 a + b at b 16 + a: so rows 8 apart lie side by side
        off = 4 * ((8 * (l >> 2) + u) * kHead + tile_row(wave, 4 * (l & 3)));
      } else {                                               // rows, two a unit; a piece's place turns with the row
        const int r = 2 * u + (l >> 5);
        off = 4 * tile_row(wave, r) * kHead + 16 * ((l & 31) ^ r);
      }
      load_lds16(mv, off, __builtin_amdgcn_readfirstlane(to + u * kUnit));
    }
    load_lds16(ad, 4 * (tile_row(wave, l >> 2) * kHead + 16 * unit.y + 4 * (l & 3)), __builtin_amdgcn_readfirstlane(to + 8 * kUnit));
  };
  floatx4 S;
  auto keep = [&](int i) {                                   // 4 stores, no more and no fewer: the waits count them
    const float* init = uniform(a.init + at(i));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t off = 4 * (tile_row(wave, 4 * g + r) * kHead + col);
      const float x = S[r];
      asm volatile("global_store_dword %0, %1, %2" ::"v"(off), "v"(x), "s"(init) : "memory");
    }
  };
  {
    const float* x = a.add + at(0);                          // the first one's start is in it
#pragma unroll
    for (int r = 0; r < 4; ++r) S[r] = x[tile_row(wave, 4 * g + r) * kHead + col];
  }
  if (pieces > 2) {
    fetch(1);
    fetch(2);
  }
  keep(1);
  for (int i = 1; i + 1 < pieces; ++i) {
    asm volatile("s_waitcnt vmcnt(13)" ::: "memory");        // all but the next segment's 9 loads and 4 stores
    const char* p = mine + (i & 1) * 8 * kJoinWave;
    Parts<3> k[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      float x[8];
      if constexpr (kBwd) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = reinterpret_cast<const float*>(p)[(16 * e + 4 * ks + g) * 16 + m];
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const floatx4 y = *reinterpret_cast<const floatx4*>(p + 512 * m + 16 * ((8 * ks + 2 * g + e) ^ m));
#pragma unroll
          for (int n = 0; n < 4; ++n) x[4 * e + n] = y[n];
        }
      }
      k[ks] = split3(x);
    }
    floatx4 ad;
#pragma unroll
    for (int r = 0; r < 4; ++r) ad[r] = reinterpret_cast<const float*>(p + 8 * kUnit)[(4 * g + r) * 16 + m];
    const float x[8] = {S[0], S[1], S[2], S[3], 0.f, 0.f, 0.f, 0.f};
    const Parts<3> s = split3(x);
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      const u32x4 w = __builtin_bit_cast(u32x4, s.p[n]);
      *reinterpret_cast<uint2*>(reinterpret_cast<char*>(&buf[((wave >> 1) * 3 + n) * 64 + l]) + 8 * (wave & 1)) = uint2{w[0], w[1]};
    }
    __syncthreads();                                         // (this wave's reads are done as well)
    fetch(i + 2);
    floatx4 sum[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      sum[ks] = floatx4{0.f, 0.f, 0.f, 0.f};
      mma(sum[ks], k[ks], staged<3>(buf, ks, l));
    }
    S = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ad;
    keep(i + 1);
    __syncthreads();                                         // the state's operands are read
  }
  wait_loads();                                              // nothing on its way to LDS when the block ends
}

// ---------------------------------------------------------------------------
// dq, dk, dg, dbeta of a chunk.  With E = dO U^T, F = dR U^T (lower, strictly lower):
//   dQ = scale e^G (dO S0^T) + scale (E D) K
//   dK = scale (E D)^T Q + e^(G_C - G) (U dS1^T) - beta e^G (dR S0^T) + (B + B^T) K,  B_ij = -beta_i F_ij D_ij
//   dbeta_i = dR_i . v_i - e^G_i k_i . (dR S0^T)_i - sum_j F_ij (k_i . k_j) D_ij
//   dG: row sums less column sums of M = E P + B (K K^T), and the three products with S0 and
//       dS1, row by row, times q or k; dg is the sum of dG from the token to the chunk's end.
// 256 threads a chunk and v head.  First everything summed over the 128 elements of v, 32 at a
// time through LDS; then the products summed over tokens.  Those with rows of the 128 elements of
// k are computed transposed: a wave owns 32 of them (two tiles), a lane 8 of one token.  Where v
// heads share a q/k head, each leaves its part of dq and dk in fp32 where its dS1 was, and
// delta_shared_kernel adds them in the heads' order (no atomics).
// 4 x 4096 tokens of 16 heads in bf16: 337 us, 1.07 GB (3.2 TB/s).  Bound by issue: the splits and
// products take three quarters of a block's cycles, at a clock that falls to 1.7 GHz under them; with
// everything in the caches it would be 290.  (Slices of S0, dS1, U and dR laid out end to end: the
// same.  512 threads, 128 registers: spills, 859 us.)
// ---------------------------------------------------------------------------
template <typename T> struct GradLds {
  static constexpr int C = ChunkType<T>::kChunk, NP = ChunkType<T>::kParts, MT = C / 16, JS = C / 32, kLd = C + 4;
  // what enters dq and dk alone: for bf16 two parts do (2^-17 of it)
  static constexpr int kIn = NP == 1 ? 2 : 3;
  static constexpr int kStage = MT * (NP + 3 + 3) * kUnit;   // dO, U, dR: 32 elements of every token
  static constexpr int kRows = MT * 4 * NP * kUnit;          // K, Q
  static constexpr int kStates = 4 * 2 * 4 * kUnit;          // 32 elements of the 32 rows of S0 and dS1 of each wave, then K, Q
  static constexpr int kKind = MT * JS * kIn * kUnit;        // a [C][C] operand
  static constexpr int kLate = 3 * kKind + C * kLd * 4;
  static constexpr int kEarly = kStage + (2 * kRows > kStates ? 2 * kRows : kStates);
  static constexpr int kBig = kEarly > kLate ? kEarly : kLate;
  static constexpr size_t kBytes = kBig + 4 * (12 * C + 5 * C + C + MT * C + 4) + 8 * C;
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

template <typename T>
__global__ __launch_bounds__(256, 2) void delta_grads_kernel(DeltaArgs a) {
  using L = GradLds<T>;
  constexpr int C = L::C, NP = L::NP, MT = L::MT, JS = L::JS, kIn = L::kIn, LD = L::kLd;
  constexpr int kTiles = MT * (MT + 1) / 2, kMine = (kTiles + 3) / 4;
  extern __shared__ __align__(16) char lds[];
  bf16x8* stage = reinterpret_cast<bf16x8*>(lds);            // dO | U | dR
  char* bk = lds + L::kStage;
  char* bq = bk + L::kRows;
  char* xe = lds;                                            // scale E D, then its transpose, then B + B^T
  char* xt = xe + L::kKind;
  char* xb = xt + L::kKind;
  float* sm = reinterpret_cast<float*>(xb + L::kKind);       // M [C][LD]
  float* red = reinterpret_cast<float*>(lds + L::kBig);      // [4 waves][3][C]
  float* gates = red + 12 * C;                               // [5][C]
  float* db = gates + 5 * C;                                 // [C]: dR . v
  float* fs = db + C;                                        // [MT][C]: sums of F (K K^T) D by tiles
  float* cross = fs + MT * C;                                     // [4]
  double* dsum = reinterpret_cast<double*>(cross + 4);       // [C]
  const int slot = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, share = a.Hv / a.Hk, hk = h / share, tid = threadIdx.x, l = lane_id(), g = l >> 4;
  const int m = l & 15, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int c;
  const Span sp = slot_of(a.s, slot, C, c);
  if (c < 0) return;
  const int64_t t0 = (int64_t)c * C;
  const int left = sp.len - (int)t0;
  const int64_t tok = (int64_t)sp.b * a.s.T + sp.t0 + t0;    // row of [B * T]
  const int64_t at = (int64_t)slot * a.Hv + h, atk = (int64_t)slot * a.Hk + hk;

  auto fetch_kq = [&]() {
    if constexpr (NP == 1) {
      const int l_ = here(l);
      fetch_rows<C, 4>(a.k, sp, t0, left, hk, lds_addr(bk), wave, l_);
      fetch_rows<C, 4>(a.q, sp, t0, left, hk, lds_addr(bq), wave, l_);
    } else {
      fetch<4>(a.kr + atk * L::kRows, lds_addr(bk), L::kRows / kUnit, wave, l);
      fetch<4>(a.qr + atk * L::kRows, lds_addr(bq), L::kRows / kUnit, wave, l);
    }
  };
  // The wave's rows of S0 and dS1, 32 elements each, by direct loads into a place of its own:
  // piece p (16 bytes) of row r at p ^ turn(r), so that the 16 rows of an operand meet 16 banks.
  const float* s0p = uniform(a.s0 + at * kHead * kHead + 32 * wave * kHead);
  const float* s1p = uniform(a.ds1 + at * kHead * kHead + 32 * wave * kHead);
  char* bs = bk + wave * 8 * kUnit;
  auto turn = [](int r) { return (r >> 1 & 1) | (r >> 3 & 1) << 1 | (r >> 4 & 1) << 2; };
  auto fetch_states = [&](int ks) {
    const int l_ = here(l);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 8 * u + (l_ >> 3);
      const uint32_t o = 4 * (r * kHead + 32 * ks) + 16 * ((l_ & 7) ^ turn(r));
      load_lds16(s0p, o, __builtin_amdgcn_readfirstlane(lds_addr(bs) + u * kUnit));
      load_lds16(s1p, o, __builtin_amdgcn_readfirstlane(lds_addr(bs) + (4 + u) * kUnit));
    }
  };
  fetch_states(0);
  {
    // a thread's 8 elements of each 32: token tid / 4
    const int st = tid >> 2, so = tid & 3;
    const bool mine = 4 * C == 256 || st < C, there = st < left;
    // uniform rows and one offset a thread (whole addresses were spilled, and what reads them back waits for every
    // load in flight); rows that are not there: the last one
    const char* up = reinterpret_cast<const char*>(uniform(a.u + at * C * kHead));
    const char* rp = reinterpret_cast<const char*>(uniform(a.dr + at * C * kHead));
    const char* op = reinterpret_cast<const char*>(uniform(row_at<T>(a.dout, sp, t0, h)));
    const char* vp = reinterpret_cast<const char*>(uniform(row_at<T>(a.v, sp, t0, h)));
    const int last = min(st, left - 1);
    const uint32_t uo = 4 * (min(st, C - 1) * kHead + 8 * so);
    const uint32_t oo = sizeof(T) * ((uint32_t)last * (uint32_t)a.dout.st + 8 * so);
    const uint32_t vo = sizeof(T) * ((uint32_t)last * (uint32_t)a.v.st + 8 * so);
    float dot_v = 0.f;
    u32x4 xu[2], xr[2], xo[sizeof(T) / 2], xv[sizeof(T) / 2];   // 8 elements as they are
    auto load = [&](int ks) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        xu[i] = *reinterpret_cast<const u32x4*>(up + 128 * ks + 16 * i + uo);
        xr[i] = *reinterpret_cast<const u32x4*>(rp + 128 * ks + 16 * i + uo);
      }
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        xo[i] = *reinterpret_cast<const u32x4*>(op + 32 * sizeof(T) * ks + 16 * i + oo);
        xv[i] = *reinterpret_cast<const u32x4*>(vp + 32 * sizeof(T) * ks + 16 * i + vo);
      }
    };
    auto floats = [](const u32x4* x, float (&y)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = sizeof(T) == 2 ? x[0][i >> 1] : x[i >> 2][i & 3];
        y[i] = sizeof(T) == 4 ? __uint_as_float(w) : i & 1 ? bf16hi(w) : bf16lo(w);
      }
    };
    auto put = [&]() {
      if (!mine) return;
      bf16x8* to = stage + 16 * so + (st & 15);
      const int tile = st >> 4;
      float fo[8], fv[8], fu[8], fr[8];
      floats(xo, fo);
      floats(xv, fv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        fo[i] = there ? fo[i] : 0.f;
        fu[i] = __uint_as_float(xu[i >> 2][i & 3]);
        fr[i] = __uint_as_float(xr[i >> 2][i & 3]);
      }
      const Parts<NP> o = parts_of<NP>(fo);
      const Parts<3> u = split3(fu), r = split3(fr);
#pragma unroll
      for (int i = 0; i < NP; ++i) to[(tile * NP + i) * 64] = o.p[i];
#pragma unroll
      for (int i = 0; i < 3; ++i) to[(MT * NP + tile * 3 + i) * 64] = u.p[i];
#pragma unroll
      for (int i = 0; i < 3; ++i) to[(MT * (NP + 3) + tile * 3 + i) * 64] = r.p[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) dot_v = __builtin_fmaf(fr[i], fv[i], dot_v);
    };
    load(0);
    if (tid < 3 * C / 4) load_lds16(uniform(a.gates + at * 256), 16u * l, lds_addr(gates));
    if (tid < 2 * C / 4) load_lds16(uniform(a.sums + at * 2 * C), 16u * l, lds_addr(gates + 3 * C));

    // dO S0^T, U dS1^T, dR S0^T (transposed), E and F by tiles of tokens
    floatx4 Z1[2][MT], Z2[2][MT], Z3[2][MT], E[kMine], F[kMine];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < MT; ++n) Z1[e][n] = Z2[e][n] = Z3[e][n] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kMine; ++i) E[i] = F[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    double dot = 0.;
#pragma unroll 1
    for (int ks = 0; ks < 4; ++ks) {
      float y[2][8], z[2][8];
      wait_loads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * (m >> 2) + 4 * e + (m & 3), o = 128 * r;
        const floatx4* p = reinterpret_cast<const floatx4*>(bs + o);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const floatx4 u = p[(2 * g + i) ^ turn(r)], w = p[((2 * g + i) ^ turn(r)) + 4 * kUnit / 16];
#pragma unroll
          for (int k = 0; k < 4; ++k) { y[e][4 * i + k] = u[k]; z[e][4 * i + k] = w[k]; }
        }
      }
      __syncthreads();                                       // the last elements' operands are read
      put();
      if (ks < 3) fetch_states(ks + 1); else fetch_kq();
      __syncthreads();
      const bf16x8* so_ = stage;
      const bf16x8* su_ = so_ + MT * NP * 64;
      const bf16x8* sr_ = su_ + MT * 3 * 64;
      Parts<3> sx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x = __builtin_fmaf(y[e][i], z[e][i], x);
        dot += x;
        sx[e] = split3(y[e]);
      }
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const Parts<NP> o = staged<NP>(so_, n, l);
        const Parts<3> r = staged<3>(sr_, n, l);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mma(Z1[e][n], sx[e], o);
          mma(Z3[e][n], sx[e], r);
        }
      }
      __builtin_amdgcn_sched_barrier(0);                     // (fewer operands in registers at a time)
      load(ks < 3 ? ks + 1 : 3);                             // (a load under a condition would be waited for at its end)
#pragma unroll
      for (int e = 0; e < 2; ++e) sx[e] = split3(z[e]);
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const Parts<3> u = staged<3>(su_, n, l);
#pragma unroll
        for (int e = 0; e < 2; ++e) mma(Z2[e][n], sx[e], u);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int t = wave + 4 * i;
        if (t < kTiles) {
          const int mt = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, nt = t - mt * (mt + 1) / 2;
          const Parts<3> u = staged<3>(su_, nt, l);
          mma(E[i], staged<NP>(so_, mt, l), u);
          mma(F[i], staged<3>(sr_, mt, l), u);
        }
      }
    }
    dot_v += __shfl_xor(dot_v, 1, 64);
    dot_v += __shfl_xor(dot_v, 2, 64);
    if (mine && so == 0) db[st] = dot_v;
    dot = wave_sum(dot);
    if (l == 0) cross[wave] = (float)dot;
    // rows 16 tile + m of the tokens: where tile_row has them
    auto natural = [&](const char* src, int tile, int ks) {
      const int tk = 16 * tile + m, x = 2 * (tk >> 5) + ((tk >> 2) & 1), y = 4 * ((tk >> 3) & 3) + (tk & 3);
      return staged<NP>(reinterpret_cast<const bf16x8*>(src), x * 4 + ks, row_slot(g, y));
    };
    wait_loads();
    __syncthreads();                                         // K and Q are there
    floatx4 dq[2][MT], dk[2][MT];                            // [128 elements: tile 2 wave + e][tokens]
#pragma unroll
    for (int n = 0; n < MT; ++n) {
      const int t = 16 * n + m;
      const float e = gates[t], rest = gates[C + t], beta = gates[2 * C + t];
      float q[8], k[8], x1 = 0.f, x2 = 0.f, x3 = 0.f;
      const Parts<NP> qp = natural(bq, n, wave), kp = natural(bk, n, wave);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[i] = k[i] = 0.f;
#pragma unroll
        for (int j = NP - 1; j >= 0; --j) {                  // (the parts' sum: exactly the element)
          q[i] += (float)qp.p[j][i];
          k[i] += (float)kp.p[j][i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z1 = a.scale * e * Z1[i >> 2][n][i & 3], z2 = rest * Z2[i >> 2][n][i & 3], z3 = e * Z3[i >> 2][n][i & 3];
        x1 = __builtin_fmaf(q[i], z1, x1);
        x2 = __builtin_fmaf(k[i], z2, x2);
        x3 = __builtin_fmaf(k[i], z3, x3);
        dq[i >> 2][n][i & 3] = z1;
        dk[i >> 2][n][i & 3] = z2 - beta * z3;
      }
      x1 += __shfl_xor(x1, 16, 64); x1 += __shfl_xor(x1, 32, 64);
      x2 += __shfl_xor(x2, 16, 64); x2 += __shfl_xor(x2, 32, 64);
      x3 += __shfl_xor(x3, 16, 64); x3 += __shfl_xor(x3, 32, 64);
      if (g == 0) {
        red[(wave * 3 + 0) * C + t] = t < left ? x1 : 0.f;
        red[(wave * 3 + 1) * C + t] = t < left ? x2 : 0.f;
        red[(wave * 3 + 2) * C + t] = t < left ? x3 : 0.f;
      }
    }
    for (int i = tid; i < MT * C; i += 256) fs[i] = 0.f;
    floatx4 QK[kMine], KK[kMine];
    const int place = cols_place(l);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int t = wave + 4 * i;
      QK[i] = KK[i] = floatx4{0.f, 0.f, 0.f, 0.f};
      if (t < kTiles) {
        const int mt = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, nt = t - mt * (mt + 1) / 2;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const Parts<NP> kj = natural(bk, nt, ks);
          mma(QK[i], natural(bq, mt, ks), kj);
          mma(KK[i], natural(bk, mt, ks), kj);
        }
      }
    }
    Parts<NP> kt[JS][2], qt[JS][2];                          // this wave's rows of K^T and Q^T
#pragma unroll
    for (int js = 0; js < JS; ++js)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        kt[js][e] = cols_of<NP>(bk, 2 * wave + e, js, place);
        qt[js][e] = cols_of<NP>(bq, 2 * wave + e, js, place);
      }
    __syncthreads();                                         // all operands are read
    // of the triangular operands' tiles beside the diagonal's, those that are read and 0 everywhere
    if (tid < MT * kIn * 32) {
      const int pair = tid >> 6, n = pair % kIn, t = 2 * (pair / kIn);
      char* to = l < 32 ? xe + ((t * JS + t / 2) * kIn + n) * kUnit + 512 : xt + (((t + 1) * JS + t / 2) * kIn + n) * kUnit;
      reinterpret_cast<u32x4*>(to)[l & 31] = u32x4{0, 0, 0, 0};
    }

    // E and F become the operands of the products over tokens
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int t = wave + 4 * i;
      if (t < kTiles) {
        const int mt = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, nt = t - mt * (mt + 1) / 2;
        const int j = 16 * nt + m;
        float ed[4], bb[4], f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ii = 16 * mt + 4 * g + r;
          const float d = j <= ii ? decay((gates[3 * C + ii] - gates[3 * C + j]) + (gates[4 * C + ii] - gates[4 * C + j])) : 0.f;
          const float fd = j < ii ? F[i][r] * d : 0.f;
          ed[r] = a.scale * E[i][r] * d;
          bb[r] = -gates[2 * C + ii] * fd;
          f[r] = row16_sum(fd * KK[i][r]);
          sm[ii * LD + j] = j < ii ? ed[r] * QK[i][r] + bb[r] * KK[i][r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m == 0) fs[nt * C + 16 * mt + 4 * g + r] = f[r];
        // (row, summed over) = (i, j): elements apart; (j, i): 4 neighbours
        const int ij = ((mt * JS + (j >> 5)) * kIn * 64 + 16 * ((j >> 3) & 3) + 4 * g) * 16 + 2 * (j & 7);
        const int i0 = 16 * mt + 4 * g;
        const int ji = ((nt * JS + (i0 >> 5)) * kIn * 64 + 16 * ((i0 >> 3) & 3) + m) * 16 + 2 * (i0 & 7);
        __bf16 pe[kIn][4], pb[kIn][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = ed[r], y = bb[r];
#pragma unroll
          for (int n = 0; n < kIn; ++n) {
            pe[n][r] = (__bf16)x;
            pb[n][r] = (__bf16)y;
            x -= (float)pe[n][r];
            y -= (float)pb[n][r];
          }
        }
#pragma unroll
        for (int n = 0; n < kIn; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            *reinterpret_cast<uint16_t*>(xe + ij + n * kUnit + 16 * r) = __builtin_bit_cast(uint16_t, pe[n][r]);
            if (j <= i0 + r) *reinterpret_cast<uint16_t*>(xb + ij + n * kUnit + 16 * r) = __builtin_bit_cast(uint16_t, pb[n][r]);
          }
          uint32_t w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) w[r] = __builtin_bit_cast(uint16_t, pe[n][r]);
          *reinterpret_cast<uint2*>(xt + ji + n * kUnit) = uint2{w[0] | w[1] << 16, w[2] | w[3] << 16};
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (j < i0 + r) *reinterpret_cast<uint16_t*>(xb + ji + n * kUnit + 2 * r) = __builtin_bit_cast(uint16_t, pb[n][r]);
        }
      }
    }
    __syncthreads();

    // the products with K and Q
#pragma unroll
    for (int js = 0; js < JS; ++js) {
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const Parts<kIn> b = staged<kIn>(reinterpret_cast<const bf16x8*>(xb), n * JS + js, l);
#pragma unroll
        for (int e = 0; e < 2; ++e) mma(dk[e][n], kt[js][e], b);
        if (js <= n / 2) {
          const Parts<kIn> x = staged<kIn>(reinterpret_cast<const bf16x8*>(xe), n * JS + js, l);
#pragma unroll
          for (int e = 0; e < 2; ++e) mma(dq[e][n], kt[js][e], x);
        }
        if (js >= n / 2) {
          const Parts<kIn> x = staged<kIn>(reinterpret_cast<const bf16x8*>(xt), n * JS + js, l);
#pragma unroll
          for (int e = 0; e < 2; ++e) mma(dk[e][n], qt[js][e], x);
        }
      }
    }
    // dG in 64 bits: what cancels between the rows and columns of M has to cancel exactly
    if (mine) {
      double s = 0.;
      for (int j = so; j < C; j += 4) s += (double)(j < st ? sm[st * LD + j] : 0.f) - (double)(j > st ? sm[j * LD + st] : 0.f);
      s += __shfl_xor(s, 1, 64);
      s += __shfl_xor(s, 2, 64);
      if (so == 0) {
        double x1 = 0., x2 = 0., x3 = 0.;
        for (int w = 0; w < 4; ++w) {
          x1 += red[(w * 3 + 0) * C + st];
          x2 += red[(w * 3 + 1) * C + st];
          x3 += red[(w * 3 + 2) * C + st];
        }
        const float beta = gates[2 * C + st];
        if (st < left) {
          float x = db[st] - (float)x3;
          for (int n = 0; n < MT; ++n) x -= fs[n * C + st];
          const int64_t o = (tok + st) * a.Hv + h;
          if (a.beta_bf16) static_cast<uint16_t*>(a.dbeta)[o] = (uint16_t)f32_to_bf16_bits(x);
          else static_cast<float*>(a.dbeta)[o] = x;
        }
        // at the end of the chunk: e^G_C <dS1, S0> and every x2, the same fp32 numbers that their rows lose
        const float f2 = (float)x2;
        dsum[st] = s + x1 - (double)f2 - beta * x3;
        red[st] = f2;
      }
    }
    __syncthreads();
    if (wave == 0 && l < C) {
      const double x2 = red[l];
      double s = dsum[l], all = x2;
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
#pragma unroll
    for (int n = 0; n < MT; ++n) {
      const int t = 16 * n + m;
      float x[8], y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { x[i] = dq[i >> 2][n][i & 3]; y[i] = dk[i >> 2][n][i & 3]; }
      if (share > 1) {                                       // (every wave is through with dS1)
        float* part = a.ds1 + at * kHead * kHead + t * kHead + 32 * wave + 8 * g;
        store8(part, x);
        store8(part + C * kHead, y);
      } else if (t < left) {
        const int64_t o = ((tok + t) * a.Hk + hk) * kHead + 32 * wave + 8 * g;
        store8(static_cast<T*>(a.dq) + o, x);
        store8(static_cast<T*>(a.dk) + o, y);
      }
    }
  }
}

// dq and dk of a q/k head from the parts of the v heads that share it.
template <typename T>
__global__ __launch_bounds__(256) void delta_shared_kernel(DeltaArgs a) {
  constexpr int C = ChunkType<T>::kChunk;
  const int slot = blockIdx.x / a.Hk, hk = blockIdx.x % a.Hk, share = a.Hv / a.Hk;
  int c;
  const Span sp = slot_of(a.s, slot, C, c);
  if (c < 0) return;
  const int left = sp.len - c * C;
  const int64_t tok = (int64_t)sp.b * a.s.T + sp.t0 + (int64_t)c * C;
  for (int u = threadIdx.x; u < 2 * C * 16; u += 256) {
    const int t = (u >> 4) % C, e = 8 * (u & 15);
    if (t >= left) continue;
    const float* part = a.ds1 + ((int64_t)slot * a.Hv + hk * share) * kHead * kHead + (u >> 4) * kHead + e;
    float x[8];
    load8(part, x);
    for (int i = 1; i < share; ++i) {
      float y[8];
      load8(part + (int64_t)i * kHead * kHead, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] += y[k];
    }
    store8(static_cast<T*>((u >> 4) < C ? a.dq : a.dk) + ((tok + t) * a.Hk + hk) * kHead + e, x);
  }
}

}  // namespace gsa

namespace gsa_host {
namespace {

// Blocks of the scans that give the outputs: half a head, a head with the CU to itself, or with another one beside it.
enum { kHalf = 1, kAlone = 2, kTwo = 3 };

// What one call lays out, from its sizes alone (so a backward pass finds what its forward kept).
struct DeltaSizes {
  int C, seg, shape;          // tokens of a chunk; chunks of a segment, 0: none; of the scans that give the outputs (kHalf, ..)
  int64_t slots, segs;        // 0 slots: out of range
  size_t tm, pm, gates, sums, kr, states, s0, u;
  size_t workspace(bool backward) const {
    return tm + pm + gates + sums + 2 * kr + (backward ? 2 * states + s0 + u : 3 * states);
  }
  size_t saved() const { return s0 + u + states; }
};
template <typename T, bool kBwd> void pack_sizes(DeltaSizes& z, size_t n, size_t nk) {
  using K = gsa::Pack<T, kBwd>;
  z.tm = n * K::kT * gsa::kUnit;
  z.pm = n * K::kP * gsa::kUnit;
  z.gates = n * gsa::kUnit;
  if (kBwd) z.sums = up(n * 2 * K::C * 4);
  if (K::NP == 3) z.kr = nk * K::kRows * gsa::kUnit;
}
DeltaSizes delta_sizes(int B, int T, int N, int packed, int Hk, int Hv, int dtype, bool backward) {
  DeltaSizes z{};
  z.C = dtype == GSA_DTYPE_BF16 ? gsa::ChunkType<uint16_t>::kChunk : gsa::ChunkType<float>::kChunk;
  if (B < 1 || T < 1 || N < 1 || Hk < 1 || Hv < Hk || Hv % Hk || !dtype_size(dtype)) return z;
  const int64_t nc = ((int64_t)T + z.C - 1) / z.C;
  z.slots = packed ? (int64_t)T / z.C + N : B * nc;
  // grids of 256 threads a chunk and head and of 512 a sequence and head: a launch has less than 2^32
  if (z.slots > (1 << 23) / Hv || (int64_t)N * Hv >= 1 << 23) {
    z.slots = 0;
    return z;
  }
  // Half heads while the longest chain of chunks decides, whole ones when the chip is full.  Measured for the whole call,
  // bf16 (fp32: the same order but where said), 12288 tokens, forward / forward and backward, us, by halves, by heads
  // alone, by two heads on a CU:
  //   equal rows of a batch: 128 heads 179 / 768, 216 / 885, 270 / 1004; 144: 261 / 995, 204 / 839, 238 / 854;
  //     256: 177 / 738, 146 / 654, 168 / 657; 272: 227 / 889, 218 / 844, 210 / 795; 768: 191 / 740, 156 / 679, 154 / 661
  // Packed sequences have lengths that only the device knows:
  //   one of half of the tokens, the others alike: 144 heads 530 / 1738, 639 / 1971, 785 / 2066; 512: 553 / 1788, 677 / 2098,
  //     827 / 2163; 1024: 578 / 1828, 700 / 2151, 850 / 2226
  //   random: 160 heads 350 / 1242, 430 / 1446, 529 / 1489; 224: 281 / 1013, 300 / 1081, 359 / 1118; 368: 221 / 880, 222 / 860,
  //     239 / 886; 512: 235 / 916, 226 / 874, 214 / 808 (fp32 424 / 1541, 422 / 1523, 396 / 1425); 1024: 246 / 925, 217 / 853, 216 / 825
  //   all alike: as the rows of a batch
  // Halves, the best for unequal lengths up to some 250 heads and within 6 % up to 512, cost at most 28 % (all alike);
  // above, heads alone gain 7 to 20 % but for one long sequence (23 % lost); two on a CU gain nothing on them and lose 50 % there.
  const int64_t heads = (int64_t)N * Hv;
  z.shape = heads <= (packed ? 512 : 128) ? kHalf : packed || heads <= 256 ? kAlone : kTwo;
  const int64_t length = packed ? nc / N : nc;               // of one sequence
  // Segments cost two passes over them and the join, and pay for few heads and long sequences:
  //   16 heads of 512 tokens 46 / 143 in one piece, 60 / 175 by segments; 768: 62 / 187 and 64 / 185; 1024: 78 / 231 and 69 / 195
  //   64 heads of 1024 tokens 88 / 312 and 100 / 330; 2048: 169 / 627 and 165 / 586; 80 heads of 4096: 377 / 1460 and 406 / 1418
  if (heads <= 64 && length >= std::max<int64_t>(12, heads / 2 - 4)) {
    // a block a CU, of at least 4 chunks (16384 tokens of 16 heads: 16 segments 323 us, 32 356); joining costs some 2 us a
    // segment and the two passes 16 us a chunk of one: more than sqrt(8 chunks) segments lose
    int64_t pieces = 256 / heads;
    while (pieces > 3 && pieces * pieces > 8 * length) --pieces;
    const int64_t seg = std::max<int64_t>(4, (length + pieces - 1) / pieces);
    z.seg = (int)seg;
    z.segs = packed ? (int64_t)T / (z.C * seg) + N : B * ((nc + seg - 1) / seg);
    z.shape = z.segs * Hv <= 256 ? kAlone : kTwo;
  }
  const size_t n = (size_t)z.slots * Hv, nk = (size_t)z.slots * Hk;
  if (dtype == GSA_DTYPE_BF16) backward ? pack_sizes<uint16_t, true>(z, n, nk) : pack_sizes<uint16_t, false>(z, n, nk);
  else backward ? pack_sizes<float, true>(z, n, nk) : pack_sizes<float, false>(z, n, nk);
  z.states = (size_t)z.segs * Hv * 128 * 128 * 4;
  z.s0 = n * 128 * 128 * 4;
  z.u = n * z.C * 128 * 4;
  return z;
}

using Heads = gsa::Shape<8, false, 4>;
using HeadsAlone = gsa::Shape<8, true>;
using Columns64 = gsa::Shape<4, true>;

template <typename T, bool kOut, typename Sh> int launch_scan(const gsa::DeltaArgs& a, int passes, hipStream_t s) {
  using L = gsa::ScanLds<T, Sh>;
  constexpr size_t lds = kOut ? L::kFwd : L::kState;
  static_assert(lds * (Sh::kDouble ? 1 : 2) <= 160 * 1024);
  if (const int e = allow_lds<gsa::delta_scan_kernel<T, kOut, Sh>>(lds)) return e;
  hipLaunchKernelGGL((gsa::delta_scan_kernel<T, kOut, Sh>), dim3(gsa::blocks_for(a.units, Sh::kBlocks), passes), dim3(64 * Sh::W), lds, s, a);
  return launch_status();
}
template <typename T, bool kOut, typename Sh> int launch_scan_bwd(const gsa::DeltaArgs& a, hipStream_t s) {
  constexpr size_t lds = gsa::ScanLds<T, Sh>::kBwd;
  static_assert(lds * (Sh::kDouble ? 1 : 2) <= 160 * 1024);
  if (const int e = allow_lds<gsa::delta_scan_bwd_kernel<T, kOut, Sh>>(lds)) return e;
  hipLaunchKernelGGL((gsa::delta_scan_bwd_kernel<T, kOut, Sh>), dim3(gsa::blocks_for(a.units, Sh::kBlocks)), dim3(64 * Sh::W), lds, s, a);
  return launch_status();
}
template <typename T, bool kBwd> int launch_chunks(const gsa::DeltaArgs& a, const DeltaSizes& z, hipStream_t s) {
  hipLaunchKernelGGL((gsa::delta_chunk_kernel<T, kBwd>), dim3(z.slots * a.Hv), dim3(256), 0, s, a);
  return launch_status();
}
template <bool kBwd> int launch_join(const gsa::DeltaArgs& a, const DeltaSizes& z, hipStream_t s) {
  if (const int e = allow_lds<gsa::delta_join_kernel<kBwd>>(gsa::kJoinLds)) return e;
  hipLaunchKernelGGL(gsa::delta_join_kernel<kBwd>, dim3(gsa::blocks_for((int64_t)a.s.N * a.Hv, 8)), dim3(512), gsa::kJoinLds, s, a, z.C);
  return launch_status();
}
// Rows outside every packed sequence: o, or the gradients (two arrays of Hk heads, one of Hv, dg, dbeta).
int launch_outside(const gsa::DeltaArgs& a, int dtype, bool backward, hipStream_t s) {
  if (!a.s.cu) return GSA_OK;
  const int64_t row = 128 * (int64_t)dtype_size(dtype), gate = a.beta_bf16 ? 2 : 4;
  const gsa::Outside x = backward ? gsa::Outside{a.s, {(char*)a.dq, (char*)a.dk, (char*)a.dv, (char*)a.dg, (char*)a.dbeta},
                                                 {a.Hk * row, a.Hk * row, a.Hv * row, a.Hv * (int64_t)4, a.Hv * gate}}
                                  : gsa::Outside{a.s, {(char*)a.o}, {a.Hv * row}};
  hipLaunchKernelGGL(gsa::outside_kernel, dim3(256), dim3(256), 0, s, x);
  return launch_status();
}
template <typename T> int launch_forward(const gsa::DeltaArgs& a, const DeltaSizes& z, hipStream_t s) {
  if (const int e = launch_outside(a, sizeof(T) == 2 ? GSA_DTYPE_BF16 : GSA_DTYPE_F32, false, s)) return e;
  if (const int e = launch_chunks<T, false>(a, z, s)) return e;
  if (a.seg) {
    if (const int e = launch_scan<T, false, Heads>(a, 2, s)) return e;
    if (const int e = launch_join<false>(a, z, s)) return e;
  }
  return z.shape == kHalf ? launch_scan<T, true, Columns64>(a, 1, s)
       : z.shape == kAlone ? launch_scan<T, true, HeadsAlone>(a, 1, s) : launch_scan<T, true, Heads>(a, 1, s);
}
template <typename T> int launch_backward(const gsa::DeltaArgs& a, const DeltaSizes& z, hipStream_t s) {
  if (const int e = launch_outside(a, sizeof(T) == 2 ? GSA_DTYPE_BF16 : GSA_DTYPE_F32, true, s)) return e;
  if (const int e = launch_chunks<T, true>(a, z, s)) return e;
  int e;
  if (a.seg) {
    if ((e = launch_scan_bwd<T, false, Heads>(a, s))) return e;
    if ((e = launch_join<true>(a, z, s))) return e;
  }
  e = z.shape == kHalf ? launch_scan_bwd<T, true, Columns64>(a, s)
    : z.shape == kAlone ? launch_scan_bwd<T, true, HeadsAlone>(a, s) : launch_scan_bwd<T, true, Heads>(a, s);
  if (e) return e;
  constexpr size_t lds = gsa::GradLds<T>::kBytes;
  static_assert(2 * lds <= 160 * 1024, "two blocks a CU");
  if ((e = allow_lds<gsa::delta_grads_kernel<T>>(lds))) return e;
  hipLaunchKernelGGL(gsa::delta_grads_kernel<T>, dim3(z.slots * a.Hv), dim3(256), lds, s, a);
  if ((e = launch_status()) || a.Hv == a.Hk) return e;
  hipLaunchKernelGGL(gsa::delta_shared_kernel<T>, dim3(z.slots * a.Hk), dim3(256), 0, s, a);
  return launch_status();
}

int delta_args(const gsa_delta_args* x, bool backward, gsa::DeltaArgs& a, DeltaSizes& z) {
  if (!x || !x->q || !x->k || !x->v || !x->g || !x->beta || !x->ws) return GSA_ERR_NULL;
  if (backward ? !x->dout || !x->dq || !x->dk || !x->dv || !x->dg || !x->dbeta || !x->saved : !x->o) return GSA_ERR_NULL;
  if (!dtype_size(x->dtype) || !dtype_size(x->beta_dtype)) return GSA_ERR_DTYPE;
  if (x->B < 1 || x->T < 1 || x->N < 1 || x->Hk < 1 || x->Hv < x->Hk || x->Hv % x->Hk || x->Hv > 65535 || x->d != 128)
    return GSA_ERR_SHAPE;
  if (x->cu_seqlens ? x->B != 1 || (x->cu_bytes != 4 && x->cu_bytes != 8) : x->N != x->B) return GSA_ERR_SHAPE;
  z = delta_sizes(x->B, x->T, x->N, x->cu_seqlens != nullptr, x->Hk, x->Hv, x->dtype, backward);
  if (!z.slots || x->ws_bytes < z.workspace(backward) || (x->saved && x->saved_bytes < z.saved())) return GSA_ERR_SHAPE;
  // a chunk's rows are addressed by 32-bit offsets
  for (int64_t st : {x->q_st, x->k_st, x->v_st, backward ? x->do_st : (int64_t)0})
    if (st < 0 || st * 64 * dtype_size(x->dtype) >= (int64_t)1 << 31) return GSA_ERR_SHAPE;
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
  a.s = {x->cu_seqlens, x->cu_bytes == 8, x->N, x->T};
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
  auto take = [&](size_t n) {
    char* p = w;
    w += n;
    return p;
  };
  a.tm = take(z.tm);
  a.pm = take(z.pm);
  a.gates = reinterpret_cast<float*>(take(z.gates));
  a.sums = reinterpret_cast<float*>(take(z.sums));
  a.kr = take(z.kr);
  a.qr = take(z.kr);
  a.seg = z.seg;
  a.units = (int)((z.seg ? z.segs : x->N) * x->Hv);
  a.add = reinterpret_cast<float*>(take(z.states));
  a.init = reinterpret_cast<float*>(take(z.states));
  if (x->saved) {
    char* p = static_cast<char*>(x->saved);
    a.s0 = reinterpret_cast<float*>(p);
    a.u = reinterpret_cast<float*>(p + z.s0);
    a.move = reinterpret_cast<float*>(p + z.s0 + z.u);
  } else {
    a.move = reinterpret_cast<float*>(take(z.states));
  }
  if (backward) {
    a.ds1 = reinterpret_cast<float*>(take(z.s0));
    a.dr = reinterpret_cast<float*>(take(z.u));
    a.dout = {x->dout, x->do_sb, x->do_st, x->do_sh};
    a.dstate_out = x->dstate_out;
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

extern "C" size_t gsa_delta_rule_workspace_bytes(int B, int T, int N, int packed, int Hk, int Hv, int dtype, int backward) {
  const auto z = gsa_host::delta_sizes(B, T, N, packed, Hk, Hv, dtype, backward != 0);
  return z.slots ? z.workspace(backward != 0) : 0;
}
extern "C" size_t gsa_delta_rule_saved_bytes(int B, int T, int N, int packed, int Hk, int Hv, int dtype) {
  const auto z = gsa_host::delta_sizes(B, T, N, packed, Hk, Hv, dtype, false);
  return z.slots ? z.saved() : 0;
}
extern "C" int gsa_delta_rule_shape(int B, int T, int N, int packed, int Hk, int Hv, int dtype) {
  const auto z = gsa_host::delta_sizes(B, T, N, packed, Hk, Hv, dtype, false);
  return z.slots ? z.shape + (z.seg ? 4 : 0) : 0;
}
extern "C" int gsa_delta_rule(const gsa_delta_args* x, void* stream) {
  gsa::DeltaArgs a;
  gsa_host::DeltaSizes z;
  if (const int e = gsa_host::delta_args(x, false, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  return x->dtype == GSA_DTYPE_BF16 ? gsa_host::launch_forward<uint16_t>(a, z, s) : gsa_host::launch_forward<float>(a, z, s);
}
extern "C" int gsa_delta_rule_backward(const gsa_delta_args* x, void* stream) {
  gsa::DeltaArgs a;
  gsa_host::DeltaSizes z;
  if (const int e = gsa_host::delta_args(x, true, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  return x->dtype == GSA_DTYPE_BF16 ? gsa_host::launch_backward<uint16_t>(a, z, s) : gsa_host::launch_backward<float>(a, z, s);
}
