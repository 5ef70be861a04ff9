// Linear attention with a decay for each head over whole sequences, forward and backward, in chunks of C tokens.
//
//   S_t = a S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   a = e^g          (S [128 x 128], fp32)
//
// In a chunk, with X the state before it and D_ij = a^(i-j) (j <= i):
//   O = scale a^(i+1) Q X + (scale Q K^T * D) V       X' = a^C X + sum_j a^(C-1-j) k_j v_j^T
// The gradients are the same sum with other operands, two of them from the last token to the first:
//   dq: rows dO, keys V, values K, X = S^T
//   dk: rows V, keys dO, values Q, X = D^T, backwards;   dv: rows K, keys Q, values dO, X = D, backwards
// (D_t = a D_{t+1} + scale q_t do_t^T from the gradient of the final state).  So one kernel (linear_scan_kernel) does all
// four: a Pass names its operands, its direction and where scale goes.  dg = sum_t <D_t, a S_{t-1}> counts the decays
// between each query i and key j, i - j of them, by positive terms alone (differences of sums over the sequence would cancel).
// dq's pass does it, with X2, the state with each term times the tokens since its key (or since the segment's start):
//   inside a chunk          sum_ij (i - j) P_ij (do_i . v_j)
//   from earlier ones       q_i . ((i + 1) dq_i's part of X + the same of X2)
//   to later segments       <D, X2> at the segment's end
//
// Long sequences of few heads are cut into segments: what each adds to the state from 0 (a pass of the same kernel without
// outputs), the states between them (linear_join_kernel), all segments' outputs at once.
//
// A block takes a head: 8 waves of 16 columns of the state each, which stays in registers from chunk to chunk (tile_row: a
// product's result is the next one's operand in the same lanes).  4 x 4096 tokens of 16 heads in bf16: state pass 39-45 us (0.1
// GB, 2.5 TB/s; its loads alone, two blocks a CU, 28), join 7, outputs 86-91 (0.27 GB, 3.1 TB/s); with gradients besides dk and dv
// 136-143 (0.54 GB, 3.9 TB/s) and dq with dg 156-169 (0.34 GB).  Of the outputs' cycles a quarter is MFMA and a quarter VALU
// (98 MFMA, 400 VALU a wave and chunk: the splits in parts), a third each for dk and dv, which do not overlap within a SIMD; the rest
// waits for loads and at the chunk's two barriers.  dq with dg: 216 MFMA and 1160 VALU, three quarters of its cycles.
// Measured and not taken (us of the outputs' pass, two blocks a CU, now 76): one block a CU with all of the next chunk ahead 98
// where V and the outputs' stage in one buffer gave 88; outputs through LDS, three barriers a chunk 85; operands read from LDS
// several products ahead (schedule groups) the same within 1 %, as two parts of the values in X for three.
//
// Precision: as the gated delta rule's (mma): fp32 operands enter products as sums of three bf16 parts.  Where only a bf16
// output depends on them two parts do, 2^-17 of a term under a rounding of 2^-9: X in Q X and P in P V (not where dg is
// summed from the product).
#include "chunks.h"

namespace gsa {

constexpr int kWaves = 8;                                    // of a block: 16 columns of the state each

// One sum over the tokens of every sequence.  Heads of q and k (shared) or of v.
struct Pass {
  Rows a, b, v, dot;                                         // rows, keys, values; dot: q (dq) or k (dk), for dg
  int a_shared, b_shared, v_shared;                          // whose rows are those of a q/k head
  int back, turn;                                            // from the last token to the first; X transposed in memory
  float in_p, in_x, in_o;                                    // scale of P, of what enters X, of A X
  const float* first;                                        // [N, Hv, 128, 128]: X before the first token, nullable
  const float* init;                                         // [segments, Hv, 128, 128]: X before the others' segments
  const float *far_first, *far;                              // dq: the same of D, for dg
  void* out;                                                 // [B, T, Hv, 128]; parts: fp32
  int out_parts;
  float* last;                                               // [N, Hv, 128, 128]: X behind the last token (back: times a), nullable
  float* add;                                                // without outputs: X behind a segment from 0
};
struct LinearArgs {
  Seqs s;
  int Hk, Hv, units, seg;                                    // units: heads of all sequences, or of all segments of seg chunks
  const float* g; int64_t g_sh;
  float* dg_parts;                                           // [units]
  Outside outside;                                           // by the kOutside blocks behind the units (packed sequences)
  Pass pass[3];
};
constexpr int kOutside = 64;

// e^-128 is 0 in fp32: a lower g (down to -inf, a reset) gives the same without inf * 0.
struct Decay { float g, hi, lo; };                           // hi + lo: g in units of log2
__device__ __forceinline__ Decay decay_of(const float* p) {
  const float x = *p, g = x < -128.f ? -128.f : x, hi = g * kLog2e;
  return {g, hi, __builtin_fmaf(g, 1.9259629911e-8f, __builtin_fmaf(g, kLog2e, -hi))};       // (log2 e less its fp32 value)
}
// e^(g n), one exp2's error whatever n: what the exponent's rounding left comes in by its first term.
__device__ __forceinline__ float power(const Decay& d, int n) {
  const float t = d.hi * (float)n, rest = __builtin_fmaf(d.hi, (float)n, -t) + d.lo * (float)n, y = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(y, rest * 0.69314718f, y);
}
// e^(g n) in two floats, a factor that a state is multiplied with again and again: its rounding would come in once for each chunk
// that a term passes (fp32, 2050 chunks in one piece, g = -2e-5: 2.9e-5 of the state; so 5e-7).  So what rounding a factor leaves
// goes into the next one, and the product of any number of them in a row is off by one rounding.
struct Whole { float hi, lo; };
__device__ __forceinline__ Whole whole_power(const Decay& d, int n) {
  const double y = exp((double)d.g * n);
  const float hi = (float)y;
  return {hi, hi < __builtin_inff() ? (float)(y - hi) : 0.f};
}
struct Factors { Whole w; float left[kWaves]; };             // a^C of whole chunks; in LDS, as registers are short
__device__ __forceinline__ float next_factor(const Whole& w, float& left) {
  const float t = w.lo + left, y = w.hi + t;
  left = t - (y - w.hi);
  return y;
}

// The matrix cores cut what they add to an accumulator below its last bit, always downwards.  So the products of smaller
// parts are summed apart, where that is less, and sums over many chunks (X) take each chunk's sum by an fma.
template <int M, int NA, int NB>
__device__ __forceinline__ void mma_apart(floatx4 (&hi)[M][1], floatx4 (&lo)[M][1], const Parts<NA> (&a)[M], const Parts<NB>& b) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == o)
#pragma unroll
          for (int t = 0; t < M; ++t) {
            floatx4& acc = o ? lo[t][0] : hi[t][0];
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t].p[i], b.p[j], acc, 0, 0, 0);
          }
}

// acc[t] += x rows[t]: the result's rows are x's index, its columns the rows' (a lane has 4 neighbours of one row).
template <int M, int NA, int NB>
__device__ __forceinline__ void mma_rows(floatx4 (&acc)[M], const Parts<NA>& x, const Parts<NB>* rows) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == o)
#pragma unroll
          for (int t = 0; t < M; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], rows[t].p[j], acc[t], 0, 0, 0);
}
template <int M, int NA, int NB>
__device__ __forceinline__ void mma_rows_apart(floatx4 (&hi)[M], floatx4 (&lo)[M], const Parts<NA>& x, const Parts<NB>* rows) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == o)
#pragma unroll
          for (int t = 0; t < M; ++t) {
            floatx4& acc = o ? lo[t] : hi[t];
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], rows[t].p[j], acc, 0, 0, 0);
          }
}

// What of the next chunk is on its way beside a chunk's products (direct loads: bf16): nothing, its keys, all of it
enum Ahead { kNothing, kKeys, kAll };

// P enters a product with bf16 outputs in two parts
template <typename T, bool kDg, Ahead kAhead> struct LinearSizes {
  static constexpr int C = ChunkType<T>::kChunk, NP = ChunkType<T>::kParts;
  static constexpr int kPParts = NP == 1 ? 2 : 3, kXParts = NP == 1 && !kDg ? 2 : 3;
  static constexpr int kRows = (C / 16) * 4 * NP * kUnit, kP = Square<C>::kFrags * kPParts * kUnit;
  // keys, values and dot (what goes ahead twice, kGroup apart); rows, P
  static constexpr int kB = 0, kV = (kAhead == kKeys ? 2 : 1) * kRows, kDot = 2 * kRows, kGroup = (kAhead == kKeys ? 1 : kDg ? 3 : 2) * kRows;
  static constexpr int kA = kAhead == kKeys ? kV + kRows : (kAhead == kAll ? 2 : 1) * kGroup, kAtP = kA + kRows;
  // powers of the decay: in_x a^(C-1-t), in_o a^(t+1); the chunks' factors
  static constexpr int kToEnd = kAtP + kP, kFromX = kToEnd + 4 * C;
  static constexpr size_t kBytes = kFromX + 4 * C + sizeof(Factors), kState = kA + 4 * C + sizeof(Factors);
};

template <int N> __device__ __forceinline__ float element(const Parts<N>& x, int e) {
  float s = (float)x.p[0][e];
#pragma unroll
  for (int n = 1; n < N; ++n) s += (float)x.p[n][e];
  return s;
}

// A state [128][128] in memory -> the lane's part: rows tile_row(t, 4 g + r), column `col`
__device__ __forceinline__ void state_load(floatx4 (&S)[8][1], const float* p, int turn, int g, int col) {
  p = uniform(p);
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int row = 8 * g + tile_at(t, 0);
    if (turn) {
      S[t][0] = *reinterpret_cast<const floatx4*>(p + (uint32_t)(col * kHead + row));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][0][r] = p[(uint32_t)((row + r) * kHead + col)];
    }
  }
}
__device__ __forceinline__ void state_store(const floatx4 (&S)[8][1], float* p, float f, int g, int col) {
  p = const_cast<float*>(uniform(p));
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) p[(uint32_t)((8 * g + tile_at(t, r)) * kHead + col)] = S[t][0][r] * f;
}

// kOut: the outputs; otherwise what a segment adds to X.  kDg: dq's pass, with dg.
template <typename T, bool kOut, bool kDg, Ahead kAhead>
__device__ __forceinline__ void linear_scan(const LinearArgs& a, const Pass& x, char* lds, float* dg_part) {
  using Z = LinearSizes<T, kDg, kAhead>;
  constexpr int C = Z::C, NP = Z::NP, MT = C / 16, JS = C / 32, kToEnd = kOut ? Z::kToEnd : Z::kA;
  const uint32_t base = lds_addr(lds);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane_id(), g = l >> 4, m = l & 15;
  const int slot = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, hk = h / (a.Hv / a.Hk);
  int piece = 0, c0 = 0;
  Span sp;
  if (a.seg) {
    sp = slot_of(a.s, slot, C * a.seg, piece);
    if (piece < 0) {
      if (kDg && tid == 0) *dg_part = 0.f;
      return;
    }
    c0 = piece * a.seg;
  } else {
    sp = span_of(a.s, slot, C);
  }
  const int chunks = (sp.len + C - 1) / C;
  const bool last = !a.seg || c0 + a.seg >= chunks;
  const int c1 = last ? chunks : c0 + a.seg;
  const bool begins = x.back ? last : piece == 0, ends = x.back ? piece == 0 : last;    // the pass's first and last segment
  if (!kOut && ends) return;                                 // nobody asks for it
  const int64_t sn = ((int64_t)sp.n * a.Hv + h) * kHead * kHead, gn = ((int64_t)slot * a.Hv + h) * kHead * kHead;
  const Decay g2 = decay_of(a.g + h * a.g_sh);
  const int col = tile_row(wave, m);                         // this lane's column of the state and the outputs

  floatx4 X[8][1], X2[kDg ? 8 : 1];
#pragma unroll
  for (int t = 0; t < 8; ++t) X[t][0] = floatx4{0.f, 0.f, 0.f, 0.f};
  if constexpr (kDg)
#pragma unroll
    for (int t = 0; t < 8; ++t) X2[t] = floatx4{0.f, 0.f, 0.f, 0.f};
  if (kOut) {
    const float* from = begins ? (x.first ? x.first + sn : nullptr) : x.init + gn;
    if (from) state_load(X, from, x.turn, g, col);
  }

  // token i of the pass in chunk c is token at(i) of the chunk's rows
  const int rs = row_slot(g, m), place = cols_place(l);
  // bf16 rows go to LDS by direct loads, a lane 16 bytes of rows t and t + 32; `lane` is its place in the first 32 rows of a
  // whole chunk, in bytes.
  auto lane_of = [&](const Rows& r) {
    const int t = tile_row(wave >> 2, (l - 4 * g) & 15);     // (row_slot)
    return (uint32_t)((x.back ? 31 - t : t) * (int)r.st + 32 * (wave & 3) + 8 * g) * 2u;
  };
  auto fetch = [&](const Rows& r, int shared, int c, int to, uint32_t lane) {
    const int left = min(C, sp.len - c * C), hh = shared ? hk : h;
    const T* p = uniform(row_at<T>(r, sp, (int64_t)c * C, hh));
    if constexpr (NP == 1) {
      static_assert(kWaves == 8 && C == 64);
      const uint32_t at = __builtin_amdgcn_readfirstlane(base + to + wave * kUnit);
      if (left == C) {
        const T* q = p + 32 * r.st;
        load_lds16(x.back ? q : p, lane, at);
        load_lds16(x.back ? p : q, lane, at + 8 * kUnit);
      } else {
        const int lh = here(l), t0 = tile_row(wave >> 2, (lh - 4 * (lh >> 4)) & 15);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = min(t0 + 32 * i, left - 1);
          load_lds16(p, (uint32_t)((x.back ? left - 1 - t : t) * (int)r.st + 32 * (wave & 3) + 8 * (lh >> 4)) * 2u, at + 8 * kUnit * i);
        }
      }
    } else {
      bf16x8* dst = reinterpret_cast<bf16x8*>(lds + to);
      for (int u = tid; u < C * 16; u += 64 * kWaves) {
        const int d8 = u & 15, i = u >> 4, t = min(i, left - 1);
        const int tile = 2 * (i >> 5) + ((i >> 2) & 1), mm = 4 * ((i >> 3) & 3) + (i & 3);
        const Parts<NP> y = operand<T>(p + (int64_t)(x.back ? left - 1 - t : t) * r.st + 8 * d8, true);
#pragma unroll
        for (int n = 0; n < NP; ++n) dst[((tile * 4 + (d8 >> 2)) * NP + n) * 64 + row_slot(d8 & 3, mm)] = y.p[n];
      }
    }
  };
  const uint32_t lane_a = lane_of(x.a), lane_b = lane_of(x.b), lane_v = lane_of(x.v), lane_dot = kDg ? lane_of(x.dot) : 0;
  float* to_end = reinterpret_cast<float*>(lds + kToEnd);
  if (tid < C) {
    to_end[tid] = x.in_x * power(g2, C - 1 - tid);
    if (kOut) to_end[C + tid] = x.in_o * power(g2, tid + 1);
  }
  Factors* const a_whole = reinterpret_cast<Factors*>(to_end + (kOut ? 2 * C : C));
  if (tid == 0) a_whole->w = whole_power(g2, C);
  a_whole->left[wave] = 0.f;
  // P: row tile pt of it by the waves pt, pt + MT, ..; this wave's columns are tile part or tiles 2 part, 2 part + 1
  const int pt = wave % MT, part = wave / MT;
  constexpr int kTiles = C == 64 ? 2 : 1;
  float pd[kTiles][4];                                       // in_p a^(i-j)
  auto tile_of = [&](int k) { return C == 64 && pt >= 2 ? 2 * part + k : part; };
  if constexpr (kOut)
#pragma unroll
    for (int k = 0; k < kTiles; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) pd[k][r] = x.in_p * power(g2, max(0, tile_row(pt, m) - tile_row(tile_of(k), 4 * g + r)));
  const int step = x.back ? -1 : 1;
  float dg = 0.f;
  int c = x.back ? c1 - 1 : c0;
  auto fetch_group = [&](int c, int to) {
    fetch(x.b, x.b_shared, c, to + Z::kB, lane_b);
    fetch(x.v, x.v_shared, c, to + Z::kV, lane_v);
    if (kDg) fetch(x.dot, 1, c, to + Z::kDot, lane_dot);
  };
  int group = 0;                                             // this chunk's keys (kAll: and values), bytes from lds
  if (c0 < c1) {
    if (kOut) fetch(x.a, x.a_shared, c, Z::kA, lane_a);
    if (kAhead == kKeys) fetch(x.b, x.b_shared, c, Z::kB, lane_b);
    else fetch_group(c, 0);
  }
  for (int n = c0; n < c1; ++n, c += step) {
    const bool more = n + 1 < c1;
    const int left = min(C, sp.len - c * C);
    // steps of decay from X to the chunk's first token: 1, or (the gradient of the final state) 0
    const int lead = x.back && c == chunks - 1 ? 0 : 1;
    wait_loads();
    __syncthreads();
    const int vals = (kAhead == kKeys ? 0 : group) + Z::kV;
    if (kAhead == kKeys) fetch(x.v, x.v_shared, c, Z::kV, lane_v);         // needed behind P and A X
    if (kAhead == kKeys && more) fetch(x.b, x.b_shared, c + step, Z::kGroup - group, lane_b);
    if (kAhead == kAll && more) fetch_group(c + step, Z::kGroup - group);

    floatx4 O[MT];                                           // O[i][r]: token tile_row(i, m), element col4 + r
    const int col4 = 32 * (wave >> 1) + 4 * (wave & 1);      // (and 8 g)
    if constexpr (kOut) {
      char* pm = lds + Z::kAtP;
#pragma unroll
      for (int k = 0; k < kTiles; ++k) {
        const int nt = tile_of(k);
        if (nt >= MT || (k == 1 && pt < 2)) continue;
        auto product = [&](int rows, int columns) {          // lane: row tile_row(pt, m), columns tile_row(nt, 4 g + r)
          floatx4 hi[1] = {floatx4{0.f, 0.f, 0.f, 0.f}}, lo[1] = {hi[0]};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const Parts<NP> y[1] = {rows_of<NP>(lds + rows, pt, ks, rs)};
            mma_rows_apart(hi, lo, rows_of<NP>(lds + columns, nt, ks, rs), y);
          }
          return NP == 1 ? hi[0] : hi[0] + lo[0];
        };
        floatx4 p = product(Z::kA, group + Z::kB), kv;
        if constexpr (kDg) kv = product(group + Z::kDot, vals);
        const int lh = here(l), i = tile_row(pt, lh & 15), j = 32 * (nt >> 1) + 4 * (nt & 1) + 8 * (lh >> 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = j + r <= i ? p[r] * pd[k][r] : 0.f;
          if constexpr (kDg)
            if (i < left) dg = __builtin_fmaf(p[r] * (float)(i - j - r), j + r < i ? kv[r] : 0.f, dg);
        }
        char* to = pm + Square<C>::at(pt, nt >> 1, false) * Z::kPParts * kUnit + 16 * lh + 8 * (nt & 1);
#pragma unroll
        for (int e = 0; e < Z::kPParts; ++e) {
          float a0 = p[0], a1 = p[1], a2 = p[2], a3 = p[3];
          const uint2 y = {take_part(a0, a1), take_part(a2, a3)};
          p = floatx4{a0, a1, a2, a3};
          *reinterpret_cast<uint2*>(to + e * kUnit) = y;
        }
      }
      // A X
      floatx4 O2[MT], lo[MT], lo2[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) O[i] = O2[i] = lo[i] = lo2[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        Parts<NP> r[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) r[i] = rows_of<NP>(lds + Z::kA, i, ks, rs);
        auto pair = [&](const floatx4& u, const floatx4& v, floatx4 (&to)[MT], floatx4 (&low)[MT]) {
          const float y[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
          const Parts<Z::kXParts> p = parts_of<Z::kXParts>(y);
          if constexpr (Z::kXParts == 3) mma_rows_apart(to, low, p, r);
          else mma_rows(to, p, r);
        };
        pair(X[2 * ks][0], X[2 * ks + 1][0], O, lo);
        if constexpr (kDg) pair(X2[2 * ks], X2[2 * ks + 1], O2, lo2);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int t = 8 * (m >> 2) + (m & 3) + tile_at(i, 0);
        float e = to_end[C + t];
        if (!lead) e = x.in_o * power(g2, t);
        float y[4];
        if constexpr (kDg) {                                // q of the lane's outputs
          const char* at = lds + group + Z::kDot + (i * 4 + (wave >> 1)) * NP * kUnit + 16 * rs + 8 * (wave & 1);
#pragma unroll
          for (int r = 0; r < 4; ++r) y[r] = 0.f;
#pragma unroll
          for (int n2 = 0; n2 < NP; ++n2) {
            const uint2 w = *reinterpret_cast<const uint2*>(at + n2 * kUnit);
            y[0] += bf16lo(w.x);
            y[1] += bf16hi(w.x);
            y[2] += bf16lo(w.y);
            y[3] += bf16hi(w.y);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (Z::kXParts == 3) O[i][r] += lo[i][r];
          if constexpr (kDg) O2[i][r] += lo2[i][r];
          O[i][r] *= e;
          if constexpr (kDg) {
            if (t < left) dg = __builtin_fmaf(y[r], __builtin_fmaf(O[i][r], (float)(t + 1), O2[i][r] * e), dg);
          }
        }
      }
      if (kAhead == kKeys && more) wait_loads<2>();          // (the next keys' two)
      else if (kAhead == kKeys) wait_loads();
      __syncthreads();                                       // P is there; A is free
      if (more) fetch(x.a, x.a_shared, c + step, Z::kA, lane_a);
    }

    if constexpr (kOut) {
      // A NaN or an infinity in a column of V: the rows before it do without it (the zeros above P's diagonal would carry it
      // there), the others become NaN.
      Parts<NP> v[JS];
      float odd = 0.f;
#pragma unroll
      for (int js = 0; js < JS; ++js) {
        v[js] = cols_of<NP>(lds + vals, wave, js, place);
        // (times 0, added: v_dot2c_f32_bf16; the first part of an fp32 value is not finite where the value is not)
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          odd = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[js].p[0][e], v[js].p[0][e + 1]}, bf16x2{(__bf16)0.f, (__bf16)0.f}, odd, false);
      }
      int bad = C;
      const bool any = __builtin_amdgcn_ballot_w64(odd != 0.f) != 0;
      if (__builtin_expect(any, 0)) {
#pragma unroll
        for (int js = 0; js < JS; ++js)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (element(v[js], e) * 0.f != 0.f) bad = min(bad, 32 * js + 8 * (here(l) >> 4) + e);
        bad = min(bad, __shfl_xor(bad, 16, 64));
        bad = min(bad, __shfl_xor(bad, 32, 64));
#pragma unroll
        for (int js = 0; js < JS; ++js)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (32 * js + 8 * (here(l) >> 4) + e >= bad)
#pragma unroll
              for (int n2 = 0; n2 < NP; ++n2) v[js].p[n2][e] = (__bf16)0.f;
      }
      const bf16x8* pm = reinterpret_cast<const bf16x8*>(lds + Z::kAtP);
#pragma unroll
      for (int js = 0; js < JS; ++js)
#pragma unroll
        for (int i = 2 * js; i < MT; i += 2) {
          const Parts<Z::kPParts> p[2] = {staged<Z::kPParts>(pm, Square<C>::at(i, js, false), l),
                                          staged<Z::kPParts>(pm, Square<C>::at(i + 1, js, false), l)};
          mma_rows(reinterpret_cast<floatx4 (&)[2]>(O[i]), v[js], p);
        }
      if (__builtin_expect(any, 0))
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int lh = here(l), b = __shfl(bad, 4 * (lh >> 4) + r, 64), t = 8 * (lh >> 2 & 3) + (lh & 3);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            if (t + tile_at(i, 0) >= b) O[i][r] = __builtin_nanf("");
        }
      const int lh = here(l), t = 8 * (lh >> 2 & 3) + (lh & 3), e = col4 + 8 * (lh >> 4);
      if (x.out_parts) {
        const int64_t row0 = (int64_t)sp.b * a.s.T + sp.t0 + (int64_t)c * C;
        float* to = const_cast<float*>(uniform(static_cast<float*>(x.out) + (row0 * a.Hv + h) * kHead));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int at = t + tile_at(i, 0);
          if (at < left) *reinterpret_cast<floatx4*>(to + (int64_t)(x.back ? left - 1 - at : at) * a.Hv * kHead + e) = O[i];
        }
      } else {
        const int64_t row0 = (int64_t)sp.b * a.s.T + sp.t0 + (int64_t)c * C, st = (int64_t)a.Hv * kHead;
        T* to = const_cast<T*>(uniform(static_cast<T*>(x.out) + (row0 * a.Hv + h) * kHead));
        auto store = [&](T* at, int i) {
          if constexpr (NP == 1) *reinterpret_cast<uint2*>(at) = uint2{pack_bf16(O[i][0], O[i][1]), pack_bf16(O[i][2], O[i][3])};
          else *reinterpret_cast<floatx4*>(at) = O[i];
        };
        if (left == C) {
          const uint32_t lane = (uint32_t)(x.back ? 31 - t : t) * (uint32_t)st + e;
#pragma unroll
          for (int i = 0; i < MT; ++i) store(to + (x.back ? C - 32 - tile_at(i, 0) : tile_at(i, 0)) * st + lane, i);
        } else {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int at = t + tile_at(i, 0);
            if (at < left) store(to + (x.back ? left - 1 - at : at) * st + e, i);
          }
        }
      }
    }

    // the values times the decay to the chunk's end
    asm volatile("" ::: "memory");                           // (read again: kept over P V they would cost registers)
    float whole;
    if (c == chunks - 1) {
      whole = power(g2, left - 1 + lead);
    } else {
      float rest = a_whole->left[wave];
      whole = next_factor(a_whole->w, rest);
      a_whole->left[wave] = rest;
    }
    Parts<3> vd[JS], vd2[kDg ? JS : 1];
#pragma unroll
    for (int js = 0; js < JS; ++js) {
      const Parts<NP> v = cols_of<NP>(lds + vals, wave, js, place);
      float y[8];
      if (left == C) {
        load8(to_end + 32 * js + 8 * g, y);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = 32 * js + 8 * g + e;
          y[e] = t < left ? to_end[t + C - left] : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= element(v, e);
      vd[js] = split3(y);
      if constexpr (kDg) {                                   // and that times the tokens to there
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= (float)max(0, left - 1 - (32 * js + 8 * g + e));
        vd2[js] = split3(y);
      }
    }

    // X
    constexpr int kSome = 2;
    constexpr bool kApart = NP == 3 || kDg;
#pragma unroll
    for (int t = 0; t < 8; t += kSome) {
      floatx4 hi[kSome][1], lo[kSome][1], hi2[kSome][1], lo2[kSome][1];
#pragma unroll
      for (int i = 0; i < kSome; ++i) hi[i][0] = lo[i][0] = hi2[i][0] = lo2[i][0] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int js = 0; js < JS; ++js) {
        Parts<NP> k[kSome];
#pragma unroll
        for (int i = 0; i < kSome; ++i) k[i] = cols_of<NP>(lds + group + Z::kB, t + i, js, place);
        mma_apart(hi, kApart ? lo : hi, k, vd[js]);
        if constexpr (kDg) mma_apart(hi2, lo2, k, vd2[js]);
      }
#pragma unroll
      for (int i = 0; i < kSome; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (kDg) X2[t + i][r] = __builtin_fmaf(__builtin_fmaf(X[t + i][0][r], (float)left, X2[t + i][r]), whole, hi2[i][0][r] + lo2[i][0][r]);
          X[t + i][0][r] = __builtin_fmaf(X[t + i][0][r], whole, kApart ? hi[i][0][r] + lo[i][0][r] : hi[i][0][r]);
        }
#pragma unroll
      for (int i = 0; i < kSome; ++i) {                      // here, not where X is used next: the sums would be kept until then
        asm volatile("" : "+v"(X[t + i][0]));
        if constexpr (kDg) asm volatile("" : "+v"(X2[t + i]));
      }
    }
    if constexpr (kAhead != kNothing) {
      group = Z::kGroup - group;
    } else {
      __syncthreads();                                       // B, V, dot and P are free
      if (more) fetch_group(c + step, 0);
    }
  }
  if constexpr (!kOut) {
    state_store(X, x.add + gn, 1.f, g, col);
  } else {
    if (ends && x.last) state_store(X, x.last + sn, x.back ? power(g2, chunks ? 1 : 0) : 1.f, g, col);
    if constexpr (kDg) {
      const float* far = last ? (x.far_first ? x.far_first + sn : nullptr) : x.far + gn;
      if (far) {
        state_load(X, far, x.turn, g, col);
        const float f = power(g2, last ? 0 : 1);             // D is the next token's, the final state's gradient this one's
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) dg = __builtin_fmaf(X[t][0][r] * f, X2[t][r], dg);
      }
    }
    if constexpr (kDg) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) dg += __shfl_xor(dg, o, 64);
      __syncthreads();
      float* red = reinterpret_cast<float*>(lds);
      if (l == 0) red[wave] = dg;
      __syncthreads();
      if (tid == 0) {
        float s = 0.f;
        for (int w = 0; w < kWaves; ++w) s += red[w];
        *dg_part = s;
      }
    }
  }
}

// Two blocks share a CU (kPerSimd 4) and cover each other's waits (fp32, 16384 tokens of 16 heads forward: 323 -> 287 us); dq with dg
// is alone, for its registers.  bf16: all of the next chunk ahead where LDS has room for it.
template <typename T, bool kOut, bool kDg> constexpr int kPerSimd = !kDg ? 4 : 2;
template <typename T, bool kOut, bool kDg> constexpr Ahead kAheadOf = sizeof(T) == 4 ? kNothing : kOut && !kDg ? kKeys : kAll;

template <typename T, bool kOut, bool kDg>
__global__ __launch_bounds__(64 * kWaves, (kPerSimd<T, kOut, kDg>)) void linear_scan_kernel(LinearArgs a) {
  extern __shared__ __align__(16) char lds[];
  const int which = blockIdx.y;
  if ((int)blockIdx.x >= a.units) {
    if (which == 0) clear_outside(a.outside, blockIdx.x - a.units, kOutside);
    return;
  }
  linear_scan<T, kOut, kDg, kAheadOf<T, kOut, kDg>>(a, a.pass[which], lds, kDg ? a.dg_parts + blockIdx.x : nullptr);
}

// X before each segment but the pass's first from what the segments add: 256 threads, 1024 elements of a head's state.  Bound by
// latency: 33 MB in 6-8 us where 16 heads have 16 segments or 64 heads 4.
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a, int C) {
  const Pass& x = a.pass[0];
  const int n = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, e = blockIdx.y * 1024 + 4 * threadIdx.x;
  const int tokens = C * a.seg;
  const Span sp = span_of(a.s, n, tokens);
  const int segs = (sp.len + tokens - 1) / tokens;
  const int64_t sn = ((int64_t)n * a.Hv + h) * kHead * kHead + e;
  if (segs == 0 && x.last)                                   // an empty sequence: no block has it
    *reinterpret_cast<floatx4*>(x.last + sn) = x.first ? *reinterpret_cast<const floatx4*>(x.first + sn) : floatx4{0.f, 0.f, 0.f, 0.f};
  if (segs < 2) return;
  const Decay g2 = decay_of(a.g + h * a.g_sh);
  floatx4 X = {0.f, 0.f, 0.f, 0.f};
  if (x.first) X = *reinterpret_cast<const floatx4*>(x.first + sn);
  // the last tokens' segment may be short, and no decay lies before the gradient of the final state
  const Whole whole = whole_power(g2, tokens);
  float left = 0.f;
  auto at = [&](int i) { return ((int64_t)(sp.slot0 + (x.back ? segs - 1 - i : i)) * a.Hv + h) * kHead * kHead + e; };
  constexpr int kSome = 8;                                   // loads on their way at once (32 segments of 16 heads: 12 us, one by one 14)
  for (int i0 = 0; i0 + 1 < segs; i0 += kSome) {
    floatx4 add[kSome];
#pragma unroll
    for (int k = 0; k < kSome; ++k) add[k] = *reinterpret_cast<const floatx4*>(x.add + at(min(i0 + k, segs - 2)));
#pragma unroll
    for (int k = 0; k < kSome; ++k) {
      const int i = i0 + k;
      if (i + 1 >= segs) break;
      const float f = x.back && i == 0 ? power(g2, sp.len - (segs - 1) * tokens - 1) : next_factor(whole, left);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[r] = __builtin_fmaf(X[r], f, add[k][r]);
      *reinterpret_cast<floatx4*>(const_cast<float*>(x.init) + at(i + 1)) = X;
    }
  }
}

// dg of a head: the parts of its blocks, in their order (4-5 us: a launch).
__global__ __launch_bounds__(256) void linear_dg_kernel(const float* parts, int units, int Hv, float* dg) {
  __shared__ double red[256];
  const int h = blockIdx.x;
  double s = 0.;
  for (int i = threadIdx.x; i < units / Hv; i += 256) s += parts[(int64_t)i * Hv + h];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) dg[h] = (float)red[0];
}

// dq (blockIdx.y 0) and dk of the q/k heads from the parts of the v heads that share them: a thread 8 elements.  Bound by HBM: 4
// bytes an element and v head read, sizeof(T) an element and q/k head written.
template <typename T>
__global__ __launch_bounds__(256) void linear_shared_kernel(const float* dq_parts, const float* dk_parts, int64_t rows, int Hk, int share,
                                                            T* dq, T* dk) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, row = u / 16;          // row: token and q/k head
  if (row >= rows * Hk) return;
  const float* p = (blockIdx.y ? dk_parts : dq_parts) + row * share * kHead + 8 * (u & 15);
  float x[8];
  load8(p, x);
  for (int i = 1; i < share; ++i) {
    float y[8];
    load8(p + i * kHead, y);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] += y[k];
  }
  store8((blockIdx.y ? dk : dq) + row * kHead + 8 * (u & 15), x);
}

}  // namespace gsa

namespace gsa_host {
namespace {

// What one call lays out, from its sizes alone (so a backward pass finds what its forward kept).
struct LinearPlan {
  int C, seg;                 // tokens of a chunk; chunks of a segment, 0: none
  int64_t units, segs;        // heads of all sequences or segments (0: out of range); segments
  size_t states, dg, parts;   // bytes: a state of every segment; dg's parts; dq and dk by v heads
  size_t workspace(bool backward) const { return 2 * states + (backward ? dg + 2 * parts : 0); }
};
LinearPlan linear_plan(int B, int T, int N, int packed, int Hk, int Hv, int dtype) {
  LinearPlan z{};
  z.C = dtype == GSA_DTYPE_BF16 ? gsa::ChunkType<uint16_t>::kChunk : gsa::ChunkType<float>::kChunk;
  if (B < 1 || T < 1 || N < 1 || Hk < 1 || Hv < Hk || Hv % Hk || !dtype_size(dtype)) return z;
  const int64_t nc = ((int64_t)T + z.C - 1) / z.C, heads = (int64_t)N * Hv;
  // a grid of 512 threads a unit: a launch has less than 2^32 of them; rows are counted in 32 bits
  if ((packed ? (int64_t)T / z.C + N : B * nc) > (1 << 23) / Hv || heads >= 1 << 23) return z;
  const int64_t length = packed ? (nc + N - 1) / N : nc;
  z.segs = 0;
  // A head is one chain of chunks; cut into segments it is passed over twice, once for the state alone (about half the work), so
  // where the heads fill most of the card that costs more.  Few heads: a block a CU, 256 / heads segments (fewer states to join, and
  // dq's pass has a CU's block at a time anyhow); more of them, packed ones, whose lengths differ, and fp32: two a CU, 512 / heads.
  // Measured in us, segments of n chunks of 64 (0: none), 16 heads a row of the batch, bf16 forward:
  //   T = 512:   0: 37    1: 22 (taken)  2: 25  4: 35        B = 6, T = 4096:   0: 270   8: 191  13: 169 (taken)  16: 184
  //   T = 2048:  0: 134   1: 43  2: 36 (taken)  4: 41        B = 10, T = 4096:  0: 273   16: 296  22: 268 (taken)
  //   T = 4096:  2: 54  4: 48 (taken)  8: 64                 B = 12, T = 4096:  0: 276 (taken)  16: 327  22: 346
  //   T = 16384: 0: 1020  4: 149  8: 121  16: 121 (taken)    B = 16, T = 4096:  0: 312 (taken)  16: 416  32: 378
  //   packed, 23 sequences, 12289 tokens: 0: 101 (taken)  4: 125  8: 118;  4 sequences, 16384: 8: 140 (taken)  16: 170
  // With gradients, T = 16384  4: 564  8: 482  16: 439 (taken)  32: 669; B = 4, T = 4096  0: 1024  8: 455  16: 431 (taken);
  // B = 16, T = 4096  0: 1401 (taken)  16: 1694.  fp32 (chunks of 32), T = 16384  8: 291  16: 266 (taken)  32: 333.
  // One chunk a segment pays where the join then has few to go through: T = 1000  1: 29  2: 30.
  if (heads <= 160 && length >= 4) {
    const int64_t pieces = (dtype == GSA_DTYPE_BF16 && !packed && heads <= 64 ? 256 : 512) / heads;
    const int64_t seg = std::max<int64_t>(length <= 16 ? 1 : 2, (length + pieces - 1) / pieces);
    if (seg < length) {
      z.seg = (int)seg;
      z.segs = packed ? (int64_t)T / (z.C * seg) + N : B * ((nc + seg - 1) / seg);
    }
  }
  z.units = z.seg ? z.segs * Hv : heads;
  z.states = (size_t)z.segs * Hv * 128 * 128 * 4;
  z.dg = up(z.units * 4);
  z.parts = Hv > Hk ? (size_t)B * T * Hv * 128 * 4 : 0;
  return z;
}

template <typename T, bool kOut, bool kDg> int launch_linear(const gsa::LinearArgs& a, int passes, hipStream_t s) {
  using Z = gsa::LinearSizes<T, kDg, gsa::kAheadOf<T, kOut, kDg>>;
  constexpr size_t lds = kOut ? Z::kBytes : Z::kState;
  static_assert(lds * (gsa::kPerSimd<T, kOut, kDg> / 2) <= 160 * 1024);
  if (const int e = allow_lds<gsa::linear_scan_kernel<T, kOut, kDg>>(lds)) return e;
  hipLaunchKernelGGL((gsa::linear_scan_kernel<T, kOut, kDg>), dim3(a.units + (kOut && a.outside.s.cu ? gsa::kOutside : 0), passes), dim3(64 * gsa::kWaves), lds, s, a);
  return launch_status();
}
// X between the segments of a.pass[0]: what each adds, then their join.
template <typename T> int launch_segments(const gsa::LinearArgs& a, const LinearPlan& z, hipStream_t s) {
  if (!z.seg) return GSA_OK;
  if (const int e = launch_linear<T, false, false>(a, 1, s)) return e;
  hipLaunchKernelGGL(gsa::linear_join_kernel, dim3(a.s.N * a.Hv, 16), dim3(256), 0, s, a, z.C);
  return launch_status();
}

int linear_args(const gsa_linear_args* x, bool backward, gsa::LinearArgs& a, LinearPlan& z) {
  if (!x || !x->q || !x->k || !x->v || !x->g) return GSA_ERR_NULL;
  if (backward ? !x->dout || !x->dq || !x->dk || !x->dv : !x->o) return GSA_ERR_NULL;
  if (!dtype_size(x->dtype)) return GSA_ERR_DTYPE;
  if (x->B < 1 || x->T < 1 || x->N < 1 || x->Hk < 1 || x->Hv < x->Hk || x->Hv % x->Hk || x->Hv > 65535 || x->d != 128)
    return GSA_ERR_SHAPE;
  if (x->cu_seqlens ? x->B != 1 || (x->cu_bytes != 4 && x->cu_bytes != 8) : x->N != x->B) return GSA_ERR_SHAPE;
  z = linear_plan(x->B, x->T, x->N, x->cu_seqlens != nullptr, x->Hk, x->Hv, x->dtype);
  if (!z.units) return GSA_ERR_SHAPE;
  if (z.workspace(backward) && !x->ws) return GSA_ERR_NULL;
  if (backward && z.seg && !x->saved) return GSA_ERR_NULL;
  if (x->ws_bytes < z.workspace(backward) || (x->saved && x->saved_bytes < z.states)) return GSA_ERR_SHAPE;
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
  if (!aligned(x->g, 4) || !aligned(x->dg, 4) || (x->cu_seqlens && !aligned(x->cu_seqlens, x->cu_bytes))) return GSA_ERR_ALIGN;
  a = gsa::LinearArgs{};
  a.s = {x->cu_seqlens, x->cu_bytes == 8, x->N, x->T};
  a.Hk = x->Hk;
  a.Hv = x->Hv;
  a.units = (int)z.units;
  a.seg = z.seg;
  a.g = x->g;
  a.g_sh = x->g_sh;
  return GSA_OK;
}
template <typename T> int linear_forward(const gsa_linear_args* x, gsa::LinearArgs& a, const LinearPlan& z, hipStream_t s) {
  float* add = static_cast<float*>(x->ws);
  gsa::Pass& p = a.pass[0];
  p.a = {x->q, x->q_sb, x->q_st, x->q_sh};
  p.b = {x->k, x->k_sb, x->k_st, x->k_sh};
  p.v = {x->v, x->v_sb, x->v_st, x->v_sh};
  p.a_shared = p.b_shared = 1;
  p.in_p = p.in_o = x->scale;
  p.in_x = 1.f;
  p.first = x->state_in;
  p.init = x->saved && z.seg ? static_cast<float*>(x->saved) : add + z.states / 4;
  p.add = add;
  p.out = x->o;
  p.last = x->state_out;
  if (const int e = launch_segments<T>(a, z, s)) return e;
  a.outside = {a.s, {(char*)x->o}, {a.Hv * 128 * (int64_t)sizeof(T)}};
  return launch_linear<T, true, false>(a, 1, s);
}

template <typename T> int linear_backward(const gsa_linear_args* x, gsa::LinearArgs& a, const LinearPlan& z, hipStream_t s) {
  char* w = static_cast<char*>(x->ws);
  float *add = reinterpret_cast<float*>(w), *init = reinterpret_cast<float*>(w + z.states);
  float *dqp = reinterpret_cast<float*>(w + 2 * z.states + z.dg), *dkp = dqp + z.parts / 4;
  const bool parts = a.Hv > a.Hk;
  const gsa::Rows q{x->q, x->q_sb, x->q_st, x->q_sh}, k{x->k, x->k_sb, x->k_st, x->k_sh}, v{x->v, x->v_sb, x->v_st, x->v_sh},
      dout{x->dout, x->do_sb, x->do_st, x->do_sh};
  a.dg_parts = reinterpret_cast<float*>(w + 2 * z.states);
  gsa::Pass dq{}, dk{}, dv{};
  dq.a = dout; dq.b = v; dq.v = k; dq.dot = q;
  dq.v_shared = dq.turn = 1;
  dq.in_p = dq.in_o = x->scale;
  dq.in_x = 1.f;
  dq.first = x->state_in;
  dq.init = static_cast<const float*>(x->saved);
  dq.far_first = x->dstate_out;
  dq.far = init;
  dq.out = parts ? (void*)dqp : x->dq;
  dq.out_parts = parts;
  dk.a = v; dk.b = dout; dk.v = q;
  dk.v_shared = dk.turn = dk.back = 1;
  dk.in_p = dk.in_x = x->scale;
  dk.in_o = 1.f;
  dk.first = x->dstate_out;
  dk.init = init;
  dk.out = parts ? (void*)dkp : x->dk;
  dk.out_parts = parts;
  dv.a = k; dv.b = q; dv.v = dout;
  dv.a_shared = dv.b_shared = dv.back = 1;
  dv.in_p = dv.in_x = x->scale;
  dv.in_o = 1.f;
  dv.first = x->dstate_out;
  dv.init = init;
  dv.out = x->dv;
  dv.last = x->dstate_in;
  dv.add = add;
  a.pass[0] = dv;
  if (const int e = launch_segments<T>(a, z, s)) return e;
  a.pass[0] = dk;
  a.pass[1] = dv;
  a.pass[2] = dq;
  const int64_t row = 128 * (int64_t)(parts ? 4 * a.Hv : sizeof(T) * a.Hk);
  a.outside = {a.s, {(char*)dq.out, (char*)dk.out, (char*)x->dv}, {row, row, a.Hv * 128 * (int64_t)sizeof(T)}};
  int e = launch_linear<T, true, false>(a, x->dg ? 2 : 3, s);
  if (e) return e;
  if (x->dg) {                                               // dq by itself: more registers, so one block a CU
    a.pass[0] = dq;
    a.outside = gsa::Outside{};
    e = launch_linear<T, true, true>(a, 1, s);
  }
  if (e) return e;
  if (x->dg) {
    hipLaunchKernelGGL(gsa::linear_dg_kernel, dim3(a.Hv), dim3(256), 0, s, a.dg_parts, a.units, a.Hv, x->dg);
    if ((e = launch_status())) return e;
  }
  if (parts) {
    const int64_t rows = (int64_t)x->B * x->T;
    hipLaunchKernelGGL(gsa::linear_shared_kernel<T>, dim3((rows * a.Hk * 16 + 255) / 256, 2), dim3(256), 0, s, dqp, dkp, rows, a.Hk,
                       a.Hv / a.Hk, static_cast<T*>(x->dq), static_cast<T*>(x->dk));
    if ((e = launch_status())) return e;
  }
  return GSA_OK;
}

}  // namespace
}  // namespace gsa_host

extern "C" size_t gsa_linear_attn_workspace_bytes(int B, int T, int N, int packed, int Hk, int Hv, int dtype, int backward) {
  const auto z = gsa_host::linear_plan(B, T, N, packed, Hk, Hv, dtype);
  return z.units ? z.workspace(backward != 0) : (size_t)-1;
}
extern "C" size_t gsa_linear_attn_saved_bytes(int B, int T, int N, int packed, int Hk, int Hv, int dtype) {
  return gsa_host::linear_plan(B, T, N, packed, Hk, Hv, dtype).states;
}
extern "C" int gsa_linear_attn(const gsa_linear_args* x, void* stream) {
  gsa::LinearArgs a;
  gsa_host::LinearPlan z;
  if (const int e = gsa_host::linear_args(x, false, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  return x->dtype == GSA_DTYPE_BF16 ? gsa_host::linear_forward<uint16_t>(x, a, z, s) : gsa_host::linear_forward<float>(x, a, z, s);
}
extern "C" int gsa_linear_attn_backward(const gsa_linear_args* x, void* stream) {
  gsa::LinearArgs a;
  gsa_host::LinearPlan z;
  if (const int e = gsa_host::linear_args(x, true, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  return x->dtype == GSA_DTYPE_BF16 ? gsa_host::linear_backward<uint16_t>(x, a, z, s) : gsa_host::linear_backward<float>(x, a, z, s);
}
