// Attention in a sliding window with a few first tokens that stay visible, forward and backward.
//
//   key j is visible to query i:  j <= i  and  (j > i - W  or  j < S)
//   o_i = sum_j P_ij v_j,  P_ij = 2^(c q_i . k_j - L_i),  c = scale log2 e,  L_i = log2 sum_j 2^(c q_i . k_j)
// and backwards, with D_i = do_i . o_i:
//   dS_ij = P_ij (do_i . v_j - D_i)    dq_i = scale sum_j dS_ij k_j    dk_j = scale sum_i dS_ij q_i    dv_j = sum_i P_ij do_i
//
// Forward: a block of 4 waves takes 128 queries of a head, walks the tiles of keys that hold a visible one (the first
// tokens' tiles, then the window's) and keeps the running maximum and sum of each row's softmax.  Both products are taken
// transposed (v_mfma_f32_32x32x16_bf16): S^T = K Q^T, O^T = V^T P^T, so that lanes l and l ^ 32 hold query l % 32, its
// softmax state lives in them and P enters the second product from the registers in which it was computed.
// dq (window_dq_kernel) goes the same way; dk and dv (window_dkv_kernel): a block takes 128 keys of a key head and walks the
// queries of all heads on it that see them, so that no two blocks write one gradient: no atomics, the same bits on every
// run.  The first tokens are seen by all later queries; those past the window's are cut into parts of
// queries, whose sums are added in their order (window_join_kernel).
//
// Bound by issue: a wave's 32 queries and 32 keys take 16 MFMA (512 cycles), 16 exponentials and some 90 further VALU (about as
// many cycles), which do not overlap within a SIMD; three waves a SIMD hide most of what else there is.  Forward, 16384
// tokens, window 4096, 16 heads on 4, bf16: 480-500 us, 0.98 PFLOP/s in the pairs that are seen (a large library product: 1.33).
// 4 x 4096 tokens, window 1024, with gradients: forward 153-163 us, dq 227-236, dk and dv 265-285, far queries 29-31 (134 MB of
// q and do read once more: 28), their join 10.
// Measured and not taken: a swizzle under which transposed reads meet in no bank (conflicts a third of LDS's cycles now,
// 0 then): 505 us for 494 forward, 687 for 668 with gradients, for what the addresses cost; tiles of 64 keys forward and two
// blocks a CU: slower throughout; dk and dv by one wave a SIMD: 857 for 707.
//
// Precision: sums, softmax statistics and D are fp32, D from o with what its rounding to bf16 left (with the rounded o alone the
// gradients' error is 1.7 times a rounding of theirs where 4 keys are visible, for 1.4).  P and dS enter the second products in
// bf16 (2^-9 of a term, as the inputs themselves were rounded; in two parts where a query sees few keys: kFine), or, for fp32, as
// three bf16 parts each, as all fp32 operands do (chunks.h).
#include "chunks.h"

#include <algorithm>
#include <climits>

namespace gsa {

// Where something is kept of blocks of sequences' first tokens.  Only sequences longer than the window have such blocks, so the
// places are bounded by the tokens and not by the sequences: of a sequence from token t on, block b is in place t / div * mult + b,
// with div the least tokens of such a sequence and mult the blocks of one, or, where that is fewer, div the keys of a
// block (each block holds that many tokens of its own) and mult 1; div 0: sequence n's blocks from n * mult on.  The parts of far queries
// behind a sequence's first part go by the same rule, as blocks of as many tokens as they have queries.
struct FirstPlaces {
  int div, mult;
  __device__ int at(int n, int start, int b) const { return (div ? start / div : n) * mult + b; }
};

struct WindowArgs {
  Seqs s;
  Rows q, k, v, dout;
  int B, H, Hkv, W, S;
  float scale, scale_l2;      // scale log2 e (forward: of |scale|, and above 0)
  void *o, *low;              // [B, T, H, 128]; bf16: what o's rounding left, in bf16 (nullable)
  float* lse;                 // [H][B * T]: L (forward: nullable)
  float* D;                   // [H][B * T]
  void *dq, *dk, *dv;
  // dk and dv: blocks of near_keys keys; the far queries of first tokens in parts of far_rows queries of a head, far_keys keys a block
  int near_keys, near_first, far_keys, far_first, far_rows;            // first: blocks of a sequence's first tokens
  int near_split;             // parts that a block's queries are cut into
  FirstPlaces near_at;
  float* near_parts;          // [near_at's places][Hkv][2][near_keys][128]; near_split > 1: [slots of keys][Hkv][near_split][2][..
  // the first far_rows far queries of a block are in far_at's places, the further ones behind those: more_at's places, far_first each
  FirstPlaces far_at, more_at;
  int far_places, more;       // more: further parts of a sequence, at most
  float* far_parts;           // [places][H][2][far_keys][128]
};

template <int N> struct Number { static constexpr int value = N; };

// Three parts of any finite value: those that round to an infinity of bf16 have its largest value as their first part.
__device__ __forceinline__ Parts<3> split_wide(const float (&x)[8]) {
  constexpr float kMost = 0x1.fep127f;
  float c[8], rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = __builtin_fabsf(x[e]) < __builtin_inff() ? fminf(fmaxf(x[e], -kMost), kMost) : x[e];
  const bf16x8 first = parts_of<1>(c).p[0];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = x[e] - (float)first[e];
  const Parts<2> more = parts_of<2>(rest);
  return {first, more.p[0], more.p[1]};
}

template <typename T> struct WindowType;
template <> struct WindowType<uint16_t> { static constexpr int NP = 1, kTile = 64, kBuffers = 2; };
template <> struct WindowType<float> { static constexpr int NP = 3, kTile = 32, kBuffers = 1; };

// ---------------------------------------------------------------------------
// Tiles of kTile rows of 128 elements in LDS: for each bf16 part (plane) rows of 16 units of 16 bytes, unit u of row t in
// place u ^ swizzle(t), so that 16 rows' reads of one unit meet in no bank (transposed reads of 32 lanes do, two by two).
// ---------------------------------------------------------------------------
__device__ __forceinline__ int swizzle(int t) { return (t & 7) << 1 | (t >> 3 & 1); }
// Row m of a 32-row product stands for row perm(m): an accumulator's 8 rows r = 8 s .. + 7 are then 16 s + 8 (l / 32) .. + 7,
// the 8 that the lane has to hold as an operand of the next product.
__device__ __forceinline__ int perm(int m) { return (m & ~12) | (m & 4) << 1 | (m & 8) >> 1; }

template <typename T, int kN = WindowType<T>::kTile> struct Tile {
  static constexpr int NP = WindowType<T>::NP, N = kN, kPlane = N * 256, kBytes = NP * kPlane;
  // Both readers hold addresses in LDS with the base (a multiple of 256 bytes) in them: what is left is the instruction's
  // offset.  tile: the tile's place behind the base.
  // Operand with rows t0 + perm(l % 32): elements 16 ks + 8 (l / 32) .. + 7
  struct RowReader {
    uint32_t at;
    __device__ RowReader(uint32_t base, int l) {
      const int t = perm(l & 31);
      at = base + t * 256 + 16 * (swizzle(t) ^ (l >> 5));
      asm("" : "+v"(at));                                    // (else the base is taken out again, and added for each read)
    }
    __device__ Parts<NP> read(uint32_t tile, int t0, int ks) const {
      Parts<NP> r;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        r.p[i] = *(const __attribute__((address_space(3))) bf16x8*)(uintptr_t)((at ^ 32u * ks) + (tile + i * kPlane + t0 * 256));
      return r;
    }
  };
  // Operand with rows of elements 32 dt + l % 32: rows t0 + 8 (l / 32) .. + 7 of the tile summed over (ds_read_b64_tr_b16: of
  // 16 lanes, lane i names row i / 4, elements 4 (i % 4) .. + 3 of 16, and gets element i of the four rows)
  struct ColReader {
    uint32_t at[2];
    __device__ ColReader(uint32_t base, int l) {
      const int i = l & 15, z = (2 * (l >> 4 & 1) + ((i & 3) >> 1)) ^ (2 * (i >> 2) + (l >> 5));
      const uint32_t row = base + (8 * (l >> 5) + (i >> 2)) * 256 + 8 * (i & 1);
      at[0] = row + 16 * z;
      at[1] = row + 16 * (z ^ 4);
      asm("" : "+v"(at[0]), "+v"(at[1]));
    }
    __device__ Parts<NP> read(uint32_t tile, int t0, int dt) const {
      Parts<NP> r;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        s16x4 x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)(
              at[dt & 1] + (tile + n * kPlane + t0 * 256 + 1024 * e + 16 * ((dt & 2 ? 8 : 0) ^ (8 * e)))));
        r.p[n] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
      }
      return r;
    }
  };
  // Rows t0 .. of one head (uniform pointer p to row t0, `stride` elements apart) to LDS, `left` of them: rows behind are the
  // last one again (they are masked).  256 threads; bf16 by direct loads, fp32 by registers (load, then store).
  struct Loader {
    static constexpr int kUnits = N * 16 / 256;              // a thread's units
    floatx4 x[NP == 3 ? 2 * kUnits : 1];
    uint32_t lane;                                           // bf16: a lane's place in the first 16 rows, in bytes
    __device__ Loader(int64_t stride, int wave, int l) {
      const int t = 4 * wave + (l >> 4);
      lane = ((uint32_t)t * (uint32_t)stride + 8 * ((l & 15) ^ swizzle(t))) * 2u;
    }
    __device__ void load(const T* p, int64_t stride, int left, uint32_t lds, int wave, int l) {
      p = uniform(p);
      if constexpr (NP == 1) {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds + wave * 1024);
        if (left >= N) {
#pragma unroll
          for (int j = 0; j < kUnits; ++j) load_lds16(p + 16 * j * stride, lane, to + j * 4096);
        } else {
          const int lh = here(l);
#pragma unroll
          for (int j = 0; j < kUnits; ++j) {
            const int t = 16 * j + 4 * wave + (lh >> 4), u = (lh & 15) ^ swizzle(t);
            load_lds16(p, ((uint32_t)min(t, left - 1) * (uint32_t)stride + 8 * u) * 2u, to + j * 4096);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
          const int t = 16 * j + 4 * wave + (l >> 4);
          const T* at = p + ((uint32_t)min(t, left - 1) * (uint32_t)stride + 8 * (l & 15));
          x[2 * j] = *reinterpret_cast<const floatx4*>(at);
          x[2 * j + 1] = *reinterpret_cast<const floatx4*>(at + 4);
        }
      }
    }
    template <bool kWide = false> __device__ void store(char* tile, int wave, int l) {
      if constexpr (NP == 3) {
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
          const int t = 16 * j + 4 * wave + (l >> 4), u = (l & 15) ^ swizzle(t);
          const floatx4 &y = x[2 * j], &z = x[2 * j + 1];
          const float all[8] = {y[0], y[1], y[2], y[3], z[0], z[1], z[2], z[3]};
          const Parts<3> p = kWide ? split_wide(all) : split3(all);
#pragma unroll
          for (int n = 0; n < 3; ++n) *reinterpret_cast<bf16x8*>(tile + n * kPlane + t * 256 + 16 * u) = p.p[n];
        }
      }
    }
  };
};

template <int NA, int NB> __device__ __forceinline__ void mma32(floatx16& acc, const Parts<NA>& a, const Parts<NB>& b) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == o) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
}
// Visible keys up to which P and dS of bf16 take two parts: the rounding of few terms does not average (two visible keys' are one and
// the same error over a whole row).  Windows with first tokens of at most so many have kernels of their own (kP = 2): the further products
// cost little there.  us by one part / two: B = 4, T = 4096 with gradients, 68 keys 277 / 298, 128 310 / 338, 256 361 / 411, 512 467 / 563,
// 1028 670 / 861; T = 16384 forward, 128 66 / 65, 256 82 / 82, 512 110 / 122, 4100 476 / 628.  Under longer windows the queries that see
// few keys are the first ones of a sequence: blocks of them, and tiles of them in dk and dv, go through a loop of two parts.  Errors in
// the norm, in roundings of the result: one part 1.41 (few keys: up to 1.5), two 1.00.
constexpr int kFine = 128;
// All queries before i of a sequence see few keys, whatever the window
__device__ __forceinline__ bool few_visible(int i, const Span& sp) { return min(i, sp.len) <= kFine; }
// The schedule of a product of kMany instructions (bf16), each with an operand from LDS: kAhead reads on their way before each
// (the compiler's own is one, and waits for it).
template <int kAhead, int kMany> __device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
  for (int i = kAhead; i < kMany; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}
// By halves, so that a long row's sum is rounded once a tile: one after the other, 8192 keys' fp32 dq was off by 1.7 times what plain
// fp32 sums give where v and dO have a mean (the error of a row's sum is common to all of its outputs, and so adds up in do . o).
__device__ __forceinline__ float sum16(const floatx16& x) {
  return (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]))) + (((x[8] + x[9]) + (x[10] + x[11])) + ((x[12] + x[13]) + (x[14] + x[15])));
}
__device__ __forceinline__ void zero(floatx16& x) {
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = 0.f;
}
// Registers 8 s .. + 7 of an accumulator as an operand
template <int N> __device__ __forceinline__ Parts<N> parts_at(const floatx16& x, int s) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = x[8 * s + e];
  return parts_of<N>(y);
}
// Operand with columns of one row of memory each: elements 16 ks + 8 (l / 32) .. + 7
template <typename T> __device__ __forceinline__ void row_operand(Parts<WindowType<T>::NP> (&x)[8], const T* p, int l) {
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) x[ks] = operand<T>(p + 16 * ks + 8 * (l >> 5), true);
}

// The transpose of a wave's [128 elements][32 rows] in 4 accumulators to rows of memory: through 32 x 128 elements of LDS of the
// wave's own.  row: of the wave's rows the i-th, `left` of them are written.
template <typename T>
__device__ __forceinline__ void store_rows(const floatx16 (&x)[4], float f, char* lds, T* p, int64_t stride, int left, int l) {
  const int i = l & 31, h = l >> 5;
  constexpr int kRowBytes = 128 * sizeof(T);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int at = 32 * dt + 2 * r + 4 * h;               // element of x[dt][r]
      char* to = lds + i * kRowBytes;
      if constexpr (sizeof(T) == 2) {
        const uint2 y = {pack_bf16(x[dt][r] * f, x[dt][r + 1] * f), pack_bf16(x[dt][r + 2] * f, x[dt][r + 3] * f)};
        *reinterpret_cast<uint2*>(to + (((at >> 3) ^ (i & 15)) << 4) + 2 * (at & 7)) = y;
      } else {
        const floatx4 y = {x[dt][r] * f, x[dt][r + 1] * f, x[dt][r + 2] * f, x[dt][r + 3] * f};
        *reinterpret_cast<floatx4*>(to + (((at >> 2) ^ i) << 4)) = y;
      }
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // (a wave's LDS accesses keep their order)
  constexpr int kPieces = kRowBytes / 16, kPer = 64 / kPieces;
#pragma unroll
  for (int j = 0; j < 32 / kPer; ++j) {
    const int t = kPer * j + l / kPieces, u = l % kPieces;
    const u32x4 y = *reinterpret_cast<const u32x4*>(lds + t * kRowBytes + ((u ^ (sizeof(T) == 2 ? t & 15 : t)) << 4));
    if (t < left) *reinterpret_cast<u32x4*>(p + t * stride + 16 / sizeof(T) * u) = y;
  }
}

// What of a tile of N keys from j0 a wave's queries r0 .. r0 + 31 see: 0 nothing, 1 something, 2 everything.
template <int N> __device__ __forceinline__ int seen(const WindowArgs& a, int r0, int j0) {
  if (j0 > r0 + 31 || (j0 + N <= r0 - a.W + 1 && j0 >= a.S)) return 0;
  return j0 + N - 1 <= r0 && (j0 > r0 + 31 - a.W || j0 + N <= a.S) ? 2 : 1;
}
__device__ __forceinline__ bool visible(const WindowArgs& a, int i, int j) { return j <= i && (i - j < a.W || j < a.S); }

// The tiles of keys that queries q0 .. q0 + n - 1 of a sequence of len tokens see
template <int N> struct KeyTiles {
  int first, from, count;                                    // tiles of first tokens; the window's first tile; of both
  __device__ KeyTiles(const WindowArgs& a, int q0, int n, int len) {
    from = max(0, q0 - a.W + 1) / N;
    first = min((min(a.S, len) + N - 1) / N, from);
    count = first + (min(len, q0 + n) + N - 1) / N - from;
  }
  __device__ int at(int t) const { return (t < first ? t : from + t - first) * N; }
};

// 0 for what is not finite, or (kNot) for what is
template <bool kNot> __device__ __forceinline__ bf16x8 finite(const bf16x8& x) {
  u32x4 y = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t odd = ((y[i] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((y[i] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    y[i] &= kNot ? odd : ~odd;
  }
  return __builtin_bit_cast(bf16x8, y);
}
template <int N> __device__ __forceinline__ Parts<N> finite(Parts<N> x) {
#pragma unroll
  for (int n = 0; n < N; ++n) x.p[n] = finite<false>(x.p[n]);
  return x;
}
// What the values that are not finite do to the outputs (made without them) of the 32 queries from r0 on that see them: NaN, or where
// all that a query sees in a column are infinities of one sign that one.  A wave: lane l looks at elements 2 l, 2 l + 1 of each key
// and keeps the queries that see such a one, a bit each; the masks go through 384 words of LDS to the lanes that hold the outputs.
template <typename T>
__device__ __forceinline__ void spoil(const WindowArgs& a, const T* vbase, int r0, int len, floatx16 (&o)[4], uint32_t* lds, int l) {
  const int from = max(0, r0 - a.W + 1), first = min(a.S, from), count = first + min(r0 + 31, len - 1) - from + 1;
  uint32_t nan[2] = {0u, 0u}, inf[2][2] = {{0u, 0u}, {0u, 0u}};
#pragma unroll 8
  for (int e = 0; e < count; ++e) {
    const int j = e < first ? e : from + e - first;
    const T* v = vbase + j * a.v.st + 2 * l;
    const int hi = j < a.S ? 31 : (int)min((int64_t)31, (int64_t)j - r0 + a.W - 1);
    const uint32_t rows = ~0u << max(0, j - r0) & ~0u >> (31 - hi);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float x = to_f32(v[c]);
      nan[c] |= x != x ? rows : 0u;
      inf[c][0] |= x == __builtin_inff() ? rows : 0u;
      inf[c][1] |= x == -__builtin_inff() ? rows : 0u;
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    lds[2 * l + c] = nan[c] | (inf[c][0] & inf[c][1]);
    lds[kHead + 2 * l + c] = inf[c][0];
    lds[2 * kHead + 2 * l + c] = inf[c][1];
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const uint32_t row = 1u << (l & 31);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const uint32_t* at = lds + 32 * dt + 2 * r + 4 * (l >> 5);         // element of o[dt][r]
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y = o[dt][r + i];
        y = at[2 * kHead + i] & row ? -__builtin_inff() : y;
        y = at[kHead + i] & row ? __builtin_inff() : y;
        o[dt][r + i] = at[i] & row ? __builtin_nanf("") : y;
      }
    }
}

// Tiles of rows for kGroups groups of 32 rows that a block's 4 waves hold: at least 32 for each wave of a group, and kLeast
template <typename T, int kGroups, int kLeast> struct WindowTiles {
  static constexpr int kSplit = 4 / kGroups;
  using L = Tile<T, 32 * (kSplit > kLeast ? kSplit : kLeast)>;
  static constexpr int NP_ = L::NP, kBuffers = WindowType<T>::kBuffers, kTiles = kBuffers * 2 * L::kBytes;
};
// Queries: 32 kGroups of a block.  LDS also holds the rows on the way out and what the waves of a group hand over.
template <typename T, int kGroups> struct WindowQueries : WindowTiles<T, kGroups, 1> {
  using Base = WindowTiles<T, kGroups, 1>;
  static constexpr int kOut = kGroups * 32 * kHead * (int)sizeof(T), kHand = Base::kSplit > 1 ? kGroups * 66 * 256 : 0;
  static constexpr size_t kBytes = std::max({Base::kTiles, kOut, kHand});
  // waves of a SIMD: bf16 three blocks a CU (registers and LDS allow it with tiles of 32 keys), with two waves a group two
  static constexpr int kWaves = Base::NP_ == 1 ? (kGroups == 4 ? 3 : 2) : kGroups == 4 ? 2 : 1;
};

// A wave of a group: 32 kGroups queries a block, the wave's every kSplit-th 32 keys.
// kP: parts of P (and dS) in the second products; 1: but for queries that see few keys
template <typename T, int kGroups, int kP>
__global__ __launch_bounds__(256, (WindowQueries<T, kGroups>::kWaves)) void window_fwd_kernel(WindowArgs a) {
  using Z = WindowQueries<T, kGroups>;
  using L = typename Z::L;
  constexpr int NP = L::NP, N = L::N, kBuffers = Z::kBuffers, kBuffer = 2 * L::kBytes, kQueries = 32 * kGroups, kSplit = Z::kSplit;
  constexpr int kMine = N / 32 / kSplit;                     // products of 32 keys a tile and wave
  extern __shared__ __align__(1024) char lds[];
  const uint32_t base = lds_addr(lds);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), group = wave % kGroups, split = kSplit > 1 ? wave / kGroups : 0;
  const int slot = gridDim.x / a.H - 1 - blockIdx.x / a.H, h = blockIdx.x % a.H, hk = h / (a.H / a.Hkv);
  int c;
  const Span sp = slot_of(a.s, slot, kQueries, c);
  if (c < 0) return;
  const int q0 = c * kQueries, r0 = q0 + 32 * group, row = r0 + (l & 31), rowc = min(row, sp.len - 1);
  const T *kbase = uniform(row_at<T>(a.k, sp, 0, hk)), *vbase = uniform(row_at<T>(a.v, sp, 0, hk));
  const KeyTiles<N> tiles(a, q0, kQueries, sp.len);
  typename L::Loader lk(a.k.st, wave, l), lv(a.v.st, wave, l);
  auto load = [&](int t, int buffer) {
    const int j0 = tiles.at(t), left = sp.len - j0;
    lk.load(kbase + j0 * a.k.st, a.k.st, left, base + buffer * kBuffer, wave, l);
    lv.load(vbase + j0 * a.v.st, a.v.st, left, base + buffer * kBuffer + L::kBytes, wave, l);
  };
  load(0, 0);
  Parts<NP> q[8];
  auto query = [&](bool wide) __attribute__((always_inline)) {
    const T* p = row_at<T>(a.q, sp, rowc, h);
    row_operand<T>(q, p, l);
    if constexpr (NP == 3) {
      if (wide) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          float x[8];
          load8(p + 16 * ks + 8 * (l >> 5), x);
          q[ks] = split_wide(x);
        }
      }
    }
    if (a.scale < 0.f)                                       // (the largest score is then the largest product)
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int n = 0; n < NP; ++n) q[ks].p[n] = -q[ks].p[n];
  };
  query(false);
  floatx16 o[4];
  const typename L::RowReader rows(base, l);
  const typename L::ColReader cols(base, l);
  // softmax state of the lane's row, log2 domain: the reference m moves only when a tile's maximum exceeds it by more than
  // kLazy (the sums then stay below 2^8 times what they are, far from fp32's range)
  constexpr float kLazy = 8.f;
  float m, limit, minus, sum;
  // clean: without the values that are not finite (of keys those give the score that they have: -infinity, or one that makes a row NaN)
  auto step = [&](int t, auto which, auto parts, auto clean) __attribute__((always_inline)) {   // the buffer's place in LDS is a constant
    constexpr int buffer = kBuffers == 2 ? decltype(which)::value : 0;
    constexpr uint32_t K = buffer * kBuffer, V = K + L::kBytes;
    if constexpr (NP == 3) {
      if (t) __syncthreads();                                // every wave is through with the last tile
      lk.template store<decltype(clean)::value != 0>(lds + K, wave, l);
      lv.template store<decltype(clean)::value != 0>(lds + V, wave, l);
    }
    wait_loads();
    __syncthreads();
    if (t + 1 < tiles.count) load(t + 1, buffer ^ 1);
    if (r0 >= sp.len) return;
#pragma unroll
    for (int mine = 0; mine < kMine; ++mine) {
      const int n = split * kMine + mine, j0 = tiles.at(t) + 32 * n, see = seen<32>(a, r0, j0);
      if (!see) continue;
      floatx16 s;
      zero(s);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const Parts<NP> k = rows.read(K, 32 * n, ks);
        if constexpr (NP == 3 && decltype(clean)::value) {   // an infinity's other parts are NaN: it goes by itself, times q's first part
          mma32(s, finite(k), q[ks]);
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(finite<true>(k.p[0]), q[ks].p[0], s, 0, 0, 0);
        } else {
          mma32(s, k, q[ks]);
        }
      }
      if constexpr (NP == 1) reads_ahead<4, 8>();
      if (see == 1) {
        const int lh = here(l), j = j0 + 8 * (lh >> 5);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = visible(a, row, j + 16 * (r >> 3) + (r & 7)) ? s[r] : -__builtin_inff();
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
      mx = max_halves(mx) * a.scale_l2;
      if (ballot64(mx > limit)) {                            // some row's reference moves
        const bool bump = mx > limit;
        const float f = bump ? __builtin_amdgcn_exp2f(m - mx) : 1.f;         // m = -inf: 0
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= f;
        sum *= f;
        m = bump ? mx : m;
        limit = m + kLazy;
        minus = m == -__builtin_inff() ? 0.f : -m;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.scale_l2, minus));
      sum += sum16(s);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const auto p = parts_at<decltype(parts)::value>(s, k);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const Parts<NP> v = cols.read(V, 32 * n + 16 * k, dt);
          mma32(o[dt], decltype(clean)::value ? finite(v) : v, p);
        }
      }
    }
  };
  auto walk = [&](auto parts, auto clean) __attribute__((always_inline)) {
    for (int t = 0; t < tiles.count; t += 2) {
      step(t, Number<0>{}, parts, clean);
      if (t + 1 < tiles.count) step(t + 1, Number<1>{}, parts, clean);
    }
  };
  auto attend = [&](auto clean) __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) zero(o[dt]);
    m = limit = -__builtin_inff();
    minus = sum = 0.f;
    if (kP == 1 && few_visible(q0 + kQueries, sp)) walk(Number<2>{}, clean);
    else walk(Number<kP>{}, clean);
    sum = sum_halves(sum);
    __syncthreads();                                         // the tiles are free
    // the waves of a group join one after the other: sums, maximum and sum of the softmax through LDS
    float* hand = reinterpret_cast<float*>(lds) + group * 66 * 64 + l;
#pragma unroll 1
    for (int w = 1; w < kSplit; ++w) {
      if (split == w) {
#pragma unroll
        for (int r = 0; r < 64; ++r) hand[64 * r] = o[r >> 4][r & 15];
        hand[64 * 64] = m;
        hand[64 * 65] = sum;
      }
      __syncthreads();
      if (split == 0) {
        const float mw = hand[64 * 64], top = mw > m ? mw : m;
        const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top), fw = mw == top ? 1.f : __builtin_amdgcn_exp2f(mw - top);
        m = top;
        sum = sum * f + hand[64 * 65] * fw;
#pragma unroll
        for (int r = 0; r < 64; ++r) o[r >> 4][r & 15] = __builtin_fmaf(o[r >> 4][r & 15], f, hand[64 * r] * fw);
      }
      __syncthreads();
    }
  };
  attend(Number<0>{});
  // Something that is not finite in a row's tiles may have reached it without being seen (0 * NaN).  Then the block goes through them
  // once more without such values, and what they do to the queries that see them is put in by itself: the others' outputs are
  // the same bits as if finite values stood there.  2 x 6000 tokens, window 4096, 8 heads on 2, bf16: 170 us, with NaN behind one row's
  // tokens 750, where all queries see one 975 (each such query by itself, key by key: 2200 and 61000).
  const bool mine = split == 0 && r0 < sp.len;
  float odd = sum * 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = __builtin_fmaf(o[dt][r], 0.f, odd);
  const bool again = __syncthreads_or(mine && !(odd == 0.f));
  if (__builtin_expect(again, 0)) {
    load(0, 0);
    if constexpr (NP == 3) query(true);
    attend(Number<1>{});
  }
  if (!mine) return;
  if (__builtin_expect(again, 0)) spoil<T>(a, vbase, r0, sp.len, o, reinterpret_cast<uint32_t*>(lds + group * 32 * kHead * sizeof(T)), l);
  const int left = sp.len - r0;
  const int64_t to = (((int64_t)sp.b * a.s.T + sp.t0 + r0) * a.H + h) * kHead;
  T *out = static_cast<T*>(a.o) + to, *low = a.low ? static_cast<T*>(a.low) + to : nullptr;
  store_rows<T>(o, 1.f / sum, lds + group * 32 * kHead * sizeof(T), out, (int64_t)a.H * kHead, left, l);
  if constexpr (NP == 1)
    if (low) {
      const float f = 1.f / sum;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        asm volatile("" : "+v"(o[dt]));                      // (else the rounded rows above are kept in registers for this)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          o[dt][r] *= f;
          o[dt][r + 1] *= f;
          float x = o[dt][r], y = o[dt][r + 1];
          take_part(x, y);
          o[dt][r] = x;
          o[dt][r + 1] = y;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the rows have been read back
      store_rows<T>(o, 1.f, lds + group * 32 * kHead * sizeof(T), low, (int64_t)a.H * kHead, left, l);
    }
  float* lse = a.lse ? a.lse + (int64_t)h * a.B * a.s.T + (int64_t)sp.b * a.s.T + sp.t0 : nullptr;
  if (lse && row < sp.len && l < 32) lse[row] = m + __builtin_amdgcn_logf(sum);
}

// The accumulators of the waves that share their rows, summed in their order into the first wave's through LDS.
template <int kGroups, int kSplit, int kMany>
__device__ __forceinline__ void join_waves(floatx16 (*const (&x)[kMany])[4], char* lds, int group, int split, int l) {
  float* hand = reinterpret_cast<float*>(lds) + group * 64 * 64 + l;
#pragma unroll 1
  for (int w = 1; w < kSplit; ++w)
#pragma unroll
    for (int n = 0; n < kMany; ++n) {
      floatx16 (&y)[4] = *x[n];
      if (split == w)
#pragma unroll
        for (int r = 0; r < 64; ++r) hand[64 * r] = y[r >> 4][r & 15];
      __syncthreads();
      if (split == 0)
#pragma unroll
        for (int r = 0; r < 64; ++r) y[r >> 4][r & 15] += hand[64 * r];
      __syncthreads();
    }
}

// dq and D: a block's queries against the tiles of keys, as forwards.
template <typename T, int kGroups, int kP>
__global__ __launch_bounds__(256, (WindowType<T>::NP == 1 ? 2 : 1)) void window_dq_kernel(WindowArgs a) {
  using Z = WindowQueries<T, kGroups>;
  using L = typename Z::L;
  constexpr int NP = L::NP, N = L::N, kBuffers = Z::kBuffers, kBuffer = 2 * L::kBytes, kQueries = 32 * kGroups, kSplit = Z::kSplit;
  constexpr int kMine = N / 32 / kSplit;
  extern __shared__ __align__(1024) char lds[];
  const uint32_t base = lds_addr(lds);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), group = wave % kGroups, split = kSplit > 1 ? wave / kGroups : 0;
  const int slot = gridDim.x / a.H - 1 - blockIdx.x / a.H, h = blockIdx.x % a.H, hk = h / (a.H / a.Hkv);
  int c;
  const Span sp = slot_of(a.s, slot, kQueries, c);
  if (c < 0) return;
  const int q0 = c * kQueries, r0 = q0 + 32 * group, row = r0 + (l & 31), rowc = min(row, sp.len - 1);
  const T *kbase = uniform(row_at<T>(a.k, sp, 0, hk)), *vbase = uniform(row_at<T>(a.v, sp, 0, hk));
  const KeyTiles<N> tiles(a, q0, kQueries, sp.len);
  typename L::Loader lk(a.k.st, wave, l), lv(a.v.st, wave, l);
  auto load = [&](int t, int buffer) {
    const int j0 = tiles.at(t), left = sp.len - j0;
    lk.load(kbase + j0 * a.k.st, a.k.st, left, base + buffer * kBuffer, wave, l);
    lv.load(vbase + j0 * a.v.st, a.v.st, left, base + buffer * kBuffer + L::kBytes, wave, l);
  };
  load(0, 0);
  Parts<NP> q[8], d[8];
  row_operand<T>(q, row_at<T>(a.q, sp, rowc, h), l);
  const T* dout = row_at<T>(a.dout, sp, rowc, h);
  row_operand<T>(d, dout, l);
  const int64_t first = (int64_t)sp.b * a.s.T + sp.t0;
  float D = 0.f;
  {
    const T* o = static_cast<const T*>(a.o) + ((first + rowc) * a.H + h) * kHead;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      float x[8], y[8];
      load8(o + 16 * ks + 8 * (l >> 5), x);
      load8(dout + 16 * ks + 8 * (l >> 5), y);
      if (a.low) {
        float z[8];
        load8(static_cast<const T*>(a.low) + ((first + rowc) * a.H + h) * kHead + 16 * ks + 8 * (l >> 5), z);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += z[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) D = __builtin_fmaf(x[e], y[e], D);
    }
    D = sum_halves(D);
  }
  const int64_t at = (int64_t)h * a.B * a.s.T + first + rowc;
  const float lse = a.lse[at];
  if (split == 0 && row < sp.len && l < 32) a.D[at] = D;
  floatx16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) zero(acc[dt]);
  const typename L::RowReader rows(base, l);
  const typename L::ColReader cols(base, l);
  auto step = [&](int t, auto which, auto parts) __attribute__((always_inline)) {   // the buffer's place in LDS is a constant
    constexpr int buffer = kBuffers == 2 ? decltype(which)::value : 0;
    constexpr uint32_t K = buffer * kBuffer, V = K + L::kBytes;
    if constexpr (NP == 3) {
      if (t) __syncthreads();
      lk.store(lds + K, wave, l);
      lv.store(lds + V, wave, l);
    }
    wait_loads();
    __syncthreads();
    if (t + 1 < tiles.count) load(t + 1, buffer ^ 1);
    if (r0 >= sp.len) return;
#pragma unroll 1
    for (int mine = 0; mine < kMine; ++mine) {
      const int n = split * kMine + mine, j0 = tiles.at(t) + 32 * n, see = seen<32>(a, r0, j0);
      if (!see) continue;
      floatx16 s, p;
      zero(s);
      zero(p);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        mma32(s, rows.read(K, 32 * n, ks), q[ks]);
        mma32(p, rows.read(V, 32 * n, ks), d[ks]);
      }
      if constexpr (NP == 1) reads_ahead<6, 16>();
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.scale_l2, -lse)) * (p[r] - D);
      if (see == 1) {
        const int lh = here(l), j = j0 + 8 * (lh >> 5);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = visible(a, row, j + 16 * (r >> 3) + (r & 7)) ? s[r] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const auto ds = parts_at<decltype(parts)::value>(s, k);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) mma32(acc[dt], cols.read(K, 32 * n + 16 * k, dt), ds);
      }
    }
  };
  auto walk = [&](auto parts) __attribute__((always_inline)) {
    for (int t = 0; t < tiles.count; t += 2) {
      step(t, Number<0>{}, parts);
      if (t + 1 < tiles.count) step(t + 1, Number<1>{}, parts);
    }
  };
  if (kP == 1 && few_visible(q0 + kQueries, sp)) walk(Number<2>{});
  else walk(Number<kP>{});
  __syncthreads();                                           // the tiles are free
  if constexpr (kSplit > 1) {
    join_waves<kGroups, kSplit, 1>({&acc}, lds, group, split, l);
    if (split) return;
  }
  if (r0 >= sp.len) return;
  store_rows<T>(acc, a.scale, lds + group * 32 * kHead * sizeof(T), static_cast<T*>(a.dq) + ((first + r0) * a.H + h) * kHead,
                (int64_t)a.H * kHead, sp.len - r0, l);
}

// Keys: 32 kGroups of a block, tiles of queries (far queries: one buffer, so that two blocks share a CU)
template <typename T, int kGroups, bool kFarPart> struct WindowKeys : WindowTiles<T, kGroups, WindowType<T>::kTile / 32> {
  using Base = WindowTiles<T, kGroups, WindowType<T>::kTile / 32>;
  static constexpr int kBuffers = kFarPart ? 1 : Base::kBuffers, kTiles = kBuffers * 2 * Base::L::kBytes;
  static constexpr int kStats = std::max(kTiles, kGroups * 64 * 256);        // (rows on the way out: as much as the waves' sums)
  static constexpr size_t kBytes = kStats + 2 * 2 * std::max(64, Base::L::N) * 4;
};

// A sequence's first token, counted over all rows of a batch; the sequence that holds a token (len 0: none does).
__device__ __forceinline__ int start_of(const Seqs& s, const Span& sp) { return s.cu ? sp.t0 : sp.n * s.T; }
__device__ __forceinline__ Span holder(const Seqs& s, int token) {
  int lo = 0;
  if (!s.cu) {
    lo = token / s.T;
  } else {
    for (int hi = s.N - 1; lo < hi;) {                       // the last sequence that does not begin behind it
      const int m = (lo + hi + 1) / 2;
      if (__builtin_amdgcn_readfirstlane((int)s.at(m)) <= token) lo = m; else hi = m - 1;
    }
  }
  Span sp = span_of(s, lo, 1);
  const int t = token - start_of(s, sp);
  if (t < 0 || t >= sp.len) sp.len = 0;
  return sp;
}
// The sequence and block of a place; len 0: none.
__device__ __forceinline__ Span holder(const Seqs& s, const FirstPlaces& p, int place, int blocks, int& b) {
  if (!p.div) {
    b = place % p.mult;
    return span_of(s, place / p.mult, 1);
  }
  Span sp = holder(s, (int)min((int64_t)INT_MAX, (int64_t)(place / p.mult + 1) * p.div - 1));
  b = place - start_of(s, sp) / p.div * p.mult;
  if (b < 0 || b >= blocks) sp.len = 0;
  return sp;
}

// dk and dv of 32 kGroups keys of a key head.  A wave has 32 of them, and of the tiles' queries each 4 / kGroups-th 32.
// kFarPart: a part of the far queries of first tokens; otherwise the queries near the keys: all that see them, but for those.
template <typename T, int kGroups, bool kFarPart, int kP>
__device__ __forceinline__ void window_dkv(const WindowArgs& a, char* lds, int index) {
  using Z = WindowKeys<T, kGroups, kFarPart>;
  using L = typename Z::L;
  constexpr int NP = L::NP, N = L::N, kBuffers = Z::kBuffers, kBuffer = 2 * L::kBytes, kKeys = 32 * kGroups, kSplit = Z::kSplit;
  const uint32_t base = lds_addr(lds);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), share = a.H / a.Hkv;
  int unit, hk, h0, heads, c, i0, i1, k0, part = 0;
  float* parts = nullptr;
  Span sp;
  if constexpr (!kFarPart) {
    part = index % a.near_split;
    unit = index / a.near_split;
    hk = unit % a.Hkv;
    h0 = hk * share;
    heads = share;
    unit /= a.Hkv;
    sp = slot_of(a.s, unit, kKeys, c);
    if (c < 0) return;
    k0 = c * kKeys;
    i0 = k0;
    const int64_t end = (int64_t)k0 + kKeys - 1 + a.W;
    i1 = (int)min((int64_t)sp.len, end);
    if (a.near_split > 1) parts = a.near_parts + (int64_t)index * 2 * kKeys * kHead;
    else if (k0 < a.S && end < sp.len) parts = a.near_parts + ((int64_t)a.near_at.at(sp.n, start_of(a.s, sp), c) * a.Hkv + hk) * 2 * kKeys * kHead;
  } else {
    h0 = index % a.H;
    hk = h0 / share;
    heads = 1;
    unit = index / a.H;
    int block;
    if (unit < a.far_places) {
      sp = holder(a.s, a.far_at, unit, a.far_first, block);
      c = 0;
    } else {
      block = (unit - a.far_places) % a.far_first;
      sp = holder(a.s, a.more_at, (unit - a.far_places) / a.far_first, a.more, c);
      ++c;
    }
    k0 = block * kKeys;
    const int64_t from = (int64_t)k0 / a.near_keys * a.near_keys + a.near_keys - 1 + a.W + (int64_t)c * a.far_rows;
    if (k0 >= a.S || from >= sp.len) return;
    i0 = (int)from;
    i1 = (int)min((int64_t)sp.len, from + a.far_rows);
    parts = a.far_parts + ((int64_t)unit * a.H + h0) * 2 * kKeys * kHead;
  }
  const int group = wave % kGroups, split = kSplit > 1 ? wave / kGroups : 0;
  const int j0 = k0 + 32 * group, key = j0 + (l & 31), keyc = min(key, sp.len - 1);
  const int tiles = (i1 - i0 + N - 1) / N, all = tiles * heads;
  const int first = kFarPart ? 0 : (int)((int64_t)all * part / a.near_split), count = kFarPart ? all : (int)((int64_t)all * (part + 1) / a.near_split);
  const T *q0 = uniform(row_at<T>(a.q, sp, i0, h0)), *d0 = uniform(row_at<T>(a.dout, sp, i0, h0));
  const int64_t stat0 = (int64_t)h0 * a.B * a.s.T + (int64_t)sp.b * a.s.T + sp.t0 + i0;
  typename L::Loader lq(a.q.st, wave, l), ld(a.dout.st, wave, l);
  constexpr int kStatRow = N < 64 ? 64 : N;                  // L of a tile's queries, then D, each a wave's 64 or two
  auto load = [&](int t, int buffer) {
    const int h = t / tiles, r = t % tiles * N, left = i1 - i0 - r;
    lq.load(q0 + r * a.q.st + h * a.q.sh, a.q.st, left, base + buffer * kBuffer, wave, l);
    ld.load(d0 + r * a.dout.st + h * a.dout.sh, a.dout.st, left, base + buffer * kBuffer + L::kBytes, wave, l);
    if (wave < kStatRow / 32) {
      const int which = wave / (kStatRow / 64), t0 = 64 * (wave % (kStatRow / 64));
      const float* p = uniform((which ? a.D : a.lse) + stat0 + (int64_t)h * a.B * a.s.T + r);
      load_lds4(p, 4u * min(t0 + l, left - 1), __builtin_amdgcn_readfirstlane(base + Z::kStats + 4 * (((t & 1) * 2 + which) * kStatRow + t0)));
    }
  };
  constexpr bool kAhead = kBuffers == 2 || NP == 3;          // the next tile's loads run beside this one's products
  if (kAhead && first < count) load(first, kBuffers == 2 ? first & 1 : 0);
  Parts<NP> k[8], v[8];
  row_operand<T>(k, row_at<T>(a.k, sp, keyc, hk), l);
  row_operand<T>(v, row_at<T>(a.v, sp, keyc, hk), l);
  floatx16 dk[4], dv[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    zero(dk[dt]);
    zero(dv[dt]);
  }
  const typename L::RowReader rows(base, l);
  const typename L::ColReader cols(base, l);
  auto walk = [&](int from, int to, auto parts) __attribute__((always_inline)) {
    constexpr int kParts = decltype(parts)::value;
    for (int t = from; t < to; ++t) {
      const int buffer = kBuffers == 2 ? t & 1 : 0;
      char *Q = lds + buffer * kBuffer, *dO = Q + L::kBytes;
      const float* st = reinterpret_cast<const float*>(lds + Z::kStats) + (t & 1) * 2 * kStatRow;
      if constexpr (kBuffers == 1) {
        if (t > first) __syncthreads();                        // every wave is through with the last tile
        if (!kAhead) load(t, 0);
        lq.store(Q, wave, l);
        ld.store(dO, wave, l);
      }
      wait_loads();
      __syncthreads();
      if (kAhead && t + 1 < count) load(t + 1, buffer ^ 1);
      const int r0 = i0 + t % tiles * N;
      if (j0 >= sp.len) continue;
#pragma unroll 1                                             // (unrolled, two such products at once do not fit the registers)
      for (int n = split; n < N / 32; n += kSplit) {
        const int i32 = r0 + 32 * n;                           // the 32 queries of this product
        const int see = i32 < i1 ? seen<32>(a, i32, j0) : 0;
        if (!see) continue;
        // (for this product alone: kept over the loop, the 8 addresses of rows would cost registers)
        typename L::RowReader r = rows;
        typename L::ColReader c = cols;
        const int shift = buffer * kBuffer + 32 * n * 256;
        r.at = here(rows.at + shift);
        c.at[0] = here(cols.at[0] + shift);
        c.at[1] = here(cols.at[1] + shift);
        floatx16 s, p;
        zero(s);
        zero(p);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          mma32(s, r.read(0, 0, ks), k[ks]);
          mma32(p, r.read(L::kBytes, 0, ks), v[ks]);
        }
        if constexpr (NP == 1) reads_ahead<3, 16>();           // (1: 293 us, 2 280, 3 278, 4 281; 4 x 4096 tokens, window 1024)
        asm volatile("" : "+v"(s), "+v"(p));
        const float* stats = st + 32 * n + 8 * (here(l) >> 5);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float y[8];
          load8(stats + 16 * x, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[8 * x + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * x + e], a.scale_l2, -y[e]));
          load8(stats + kStatRow + 16 * x, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) p[8 * x + e] = s[8 * x + e] * (p[8 * x + e] - y[e]);
        }
        if (see == 1 || i32 + 32 > i1) {
          const int lh = here(l), i = i32 + 8 * (lh >> 5), j = j0 + (lh & 31);
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const int ir = i + 16 * (y >> 3) + (y & 7);
            const bool on = ir < i1 && visible(a, ir, j);
            s[y] = on ? s[y] : 0.f;
            p[y] = on ? p[y] : 0.f;
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const auto w = parts_at<kParts>(s, x), ds = parts_at<kParts>(p, x);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            mma32(dv[dt], c.read(L::kBytes, 16 * x, dt), w);
            mma32(dk[dt], c.read(0, 16 * x, dt), ds);
          }
        }
      }
    }
  };
  // Queries that see few keys, then the others of a head (a loop each: both kinds in one would spill registers)
  if constexpr (kP == 1) {
    const int few = std::clamp((kFine - i0 + N - 1) / N, 0, tiles);
    for (int t = first; t < count;) {
      const int head = t / tiles * tiles, end = min(head + tiles, count), mid = std::clamp(head + few, t, end);
      walk(t, mid, Number<2>{});
      walk(mid, end, Number<1>{});
      t = end;
    }
  } else {
    walk(first, count, Number<kP>{});
  }
  __syncthreads();                                           // the tiles are free
  if constexpr (kSplit > 1) {
    join_waves<kGroups, kSplit, 2>({&dk, &dv}, lds, group, split, l);
    if (split) return;
  }
  if (j0 >= sp.len) return;
  const int left = sp.len - j0;
  if (parts) {
    char* own = lds + group * 32 * kHead * 4;
    store_rows<float>(dk, a.scale, own, parts + 32 * group * kHead, kHead, 32, l);
    store_rows<float>(dv, 1.f, own, parts + (kKeys + 32 * group) * kHead, kHead, 32, l);
    return;
  }
  char* own = lds + group * 32 * kHead * sizeof(T);
  const int64_t o = (((int64_t)sp.b * a.s.T + sp.t0 + j0) * a.Hkv + hk) * kHead;
  store_rows<T>(dk, a.scale, own, static_cast<T*>(a.dk) + o, (int64_t)a.Hkv * kHead, left, l);
  store_rows<T>(dv, 1.f, own, static_cast<T*>(a.dv) + o, (int64_t)a.Hkv * kHead, left, l);
}

// (One kernel for both kinds of blocks would spill registers, and what reads those back waits for the tiles on their way.)
template <typename T, int kGroups, bool kFarPart, int kP>
__global__ __launch_bounds__(256, (WindowType<T>::NP == 1 ? 2 : 1)) void window_dkv_kernel(WindowArgs a) {
  extern __shared__ __align__(1024) char lds[];
  window_dkv<T, kGroups, kFarPart, kP>(a, lds, blockIdx.x);
}

// dk and dv of what came in parts: of all keys (near_split > 1) or a sequence's first tokens; the near queries' parts and
// those of the far ones, in their order.
template <typename T>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
  const int hk = blockIdx.x % a.Hkv, unit = blockIdx.x / a.Hkv, share = a.H / a.Hkv;
  Span sp;
  int block;
  if (a.near_split > 1) {
    sp = slot_of(a.s, unit, a.near_keys, block);
    if (block < 0) return;
  } else {
    sp = holder(a.s, a.near_at, unit, a.near_first, block);
  }
  const int k0 = block * a.near_keys;
  const int64_t end = (int64_t)k0 + a.near_keys - 1 + a.W;
  const bool far_too = k0 < a.S && end < sp.len;
  if (k0 >= sp.len || (a.near_split == 1 && !far_too)) return;         // (written as they were)
  const int start = start_of(a.s, sp);
  const int near = a.near_keys * kHead, far = a.far_keys * kHead;
  const float* parts = a.near_parts + (int64_t)blockIdx.x * a.near_split * 2 * near;
  for (int u = threadIdx.x + 256 * blockIdx.y; u < 2 * near / 8; u += 256 * gridDim.y) {
    const int which = 8 * u >= near, t = u / 16 - which * a.near_keys, key = k0 + t, e = 8 * (u % 16);
    if (key >= sp.len) continue;
    float x[8];
    load8(parts + which * near + t * kHead + e, x);
    for (int i = 1; i < a.near_split; ++i) {
      float y[8];
      load8(parts + (2 * i + which) * near + t * kHead + e, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] += y[k];
    }
    if (far_too && key < a.S) {                              // (the others have no far queries)
      const int fb = key / a.far_keys, at = which * far + key % a.far_keys * kHead + e;
      for (int c = 0; end + (int64_t)c * a.far_rows < sp.len; ++c) {
        const int place = c ? a.far_places + a.more_at.at(sp.n, start, c - 1) * a.far_first + fb : a.far_at.at(sp.n, start, fb);
        for (int h = 0; h < share; ++h) {
          float y[8];
          load8(a.far_parts + ((int64_t)place * a.H + hk * share + h) * 2 * far + at, y);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] += y[i];
        }
      }
    }
    T* to = static_cast<T*>(which ? a.dv : a.dk);
    store8(to + (((int64_t)sp.b * a.s.T + sp.t0 + key) * a.Hkv + hk) * kHead + e, x);
  }
}

}  // namespace gsa

namespace gsa_host {
namespace {

struct WindowPlan {
  int64_t slots, near, far;   // blocks of queries of all sequences, of keys, of parts of far queries (0: no far queries)
  int queries, near_keys, near_split, near_first, far_keys, far_first, far_rows, W, S;   // queries: of a block
  gsa::FirstPlaces near_at, far_at, more_at;
  int near_places, far_places, more;
  size_t D, near_parts, far_parts;
  size_t workspace() const { return D + near_parts + far_parts; }
};
// Places for `blocks` blocks of `keys` first tokens of each sequence of at least `least` tokens: how many.
int64_t first_places(int64_t tokens, int64_t N, int64_t least, int blocks, int keys, gsa::FirstPlaces& p) {
  const int64_t by_start = tokens / least * blocks, by_token = tokens / keys;
  if (N * blocks <= std::min(by_start, by_token)) return p = {0, blocks}, N * blocks;
  if (by_start <= by_token) return p = {(int)least, blocks}, by_start;
  return p = {keys, 1}, by_token;
}
bool window_plan(int B, int T, int N, int packed, int H, int Hkv, int window, int sinks, int dtype, WindowPlan& z) {
  z = WindowPlan{};
  if (B < 1 || T < 1 || N < 1 || Hkv < 1 || H < Hkv || H % Hkv || H > 65535 || window < 1 || sinks < 0 || !dtype_size(dtype)) return false;
  z.W = std::min(window, T);
  z.S = std::min(sinks, T);
  if ((int64_t)z.W + z.S >= T) {                             // every earlier token is visible: the window alone says so
    z.W = T;
    z.S = 0;
  }
  auto slots = [&](int n) { return packed ? (int64_t)T / n + N : (int64_t)B * (((int64_t)T + n - 1) / n); };
  // 64 queries a block (two waves share their queries, each takes half of the keys) while 128 leave CUs idle: us forward, 16
  // heads on 4, window 1024, by 128 / 64 queries: T = 512 18 / 13, T = 1024, window 256 18 / 14, T = 2048 35 / 28, T = 4096 48 / 54,
  // B = 4 145 / 182; 4 heads T = 2000 33 / 21; fp32 B = 2 T = 1537, 4 heads 112 / 77, T = 4096, 16 heads 188 / 292.
  // (32 queries, four waves each a quarter of the keys: 15 at T = 512, 27 at T = 2000, worse at all others.)
  z.queries = slots(128) * H <= 256 ? 64 : 128;
  z.slots = slots(z.queries);
  // a grid of 256 threads a block: a launch has less than 2^32 of them
  if (slots(32) > (1 << 23) / H || (int64_t)B * T >= (int64_t)1 << 31) return false;
  // 64 keys a block (two waves share their keys, each takes half of the queries) while 128 leave CUs idle: us forward and
  // backward, 16 heads on 4, window 1024, by 128 / 64: T = 4096 252 / 245, B = 4 T = 4096 644 / 655, T = 16384 718 / 735;
  // on 16 heads T = 2048 146 / 144, T = 4096 212 / 215; window 64, T = 8192 170 / 156.  fp32 always 64, for its registers.
  z.near_keys = dtype == GSA_DTYPE_BF16 && slots(128) * Hkv >= 512 ? 128 : 64;
  z.far_keys = dtype == GSA_DTYPE_BF16 ? 32 : 64;
  z.near = slots(z.near_keys);
  // A block's queries in parts (summed by window_join_kernel) where the blocks are fewer than the card takes at once, two a CU, fp32
  // one; at least 4 tiles a part.  us backward, by parts: bf16, 16 heads on 4, T = 512 1: 69  4: 41  8: 38 (taken: 8); T = 2048, window
  // 1024 1: 167  2: 120  4: 103 (taken)  8: 113; T = 4096 1: 214  2: 189 (taken)  4: 197; 8 heads on 1, T = 4096 1: 808  4: 271
  // 8: 189 (taken); T = 300, 4 heads 1: 27 (taken)  2: 28; 512 blocks (16 heads, T = 2048) 1: 92 (taken)  2: 110; fp32 B = 2
  // T = 1537, 4 heads on 2, window 256 1: 154  2: 127 (taken)  4: 145; 256 blocks 1: 493 (taken)  2: 512.
  const int64_t room = (dtype == GSA_DTYPE_BF16 ? 512 : 256) / (z.near * Hkv);
  z.near_split = (int)std::clamp<int64_t>(H / Hkv * ((z.W + (int64_t)z.near_keys) / 64) / 4, 1, std::max<int64_t>(1, room));
  int64_t parts = 0;                                         // places for sums of far queries
  const int64_t least = (int64_t)z.W + z.near_keys;                  // tokens of a sequence that has far queries, at least
  if (z.S && least <= T) {
    z.near_first = std::min((z.S + z.near_keys - 1) / z.near_keys, (T - z.W) / z.near_keys);
    z.far_first = std::min((z.S + z.far_keys - 1) / z.far_keys, (T - z.W) / z.near_keys * (z.near_keys / z.far_keys));
    const int64_t tokens = (int64_t)B * T;
    z.near_places = (int)first_places(tokens, N, least, z.near_first, z.near_keys, z.near_at);
    z.far_places = (int)first_places(tokens, N, least, z.far_first, z.far_keys, z.far_at);
    // 512 far queries a part, 128 where that leaves CUs idle; more of them where the parts are many (they fill the card without,
    // and each leaves 32 KiB, so that the workspace would grow with T times the first tokens).  By the tokens alone: sequences add a
    // first part each, however many queries a part has.  us backward, 60000 tokens and 600 sequences of 17 beside them, 16 heads on
    // 4, window 64, 4 first: with all far queries of a head in one block, which is what 600 parts would ask for, 2628, so 1202.
    int64_t rows = tokens / 512 * z.far_first * H >= 256 ? 512 : 128;
    while (tokens / rows * z.far_first * H > 8192) rows *= 2;
    z.far_rows = (int)std::min<int64_t>(rows, INT_MAX);
    z.more = (int)((T - least) / rows);
    // (only packed sequences, whose lengths the host does not know, have blocks without work: 64 of 576 cost 9 us of 36)
    const int64_t more = packed ? tokens / rows : (int64_t)B * z.more;
    if (packed) z.more_at = {z.far_rows, 1}; else z.more_at = {0, z.more};
    z.far = z.far_places + more * z.far_first;
    parts = z.far_places + tokens / rows * z.far_first;
  }
  z.D = up((size_t)H * B * T * 4);
  z.near_parts = (z.near_split > 1 ? (size_t)z.near * z.near_split : (size_t)z.near_places) * Hkv * 2 * z.near_keys * 128 * 4;
  z.far_parts = (size_t)parts * H * 2 * z.far_keys * 128 * 4;
  return true;
}

int window_args(const gsa_window_args* x, bool backward, gsa::WindowArgs& a, WindowPlan& z) {
  if (!x || !x->q || !x->k || !x->v || !x->o) return GSA_ERR_NULL;
  if (backward && (!x->dout || !x->dq || !x->dk || !x->dv || !x->lse || !x->ws)) return GSA_ERR_NULL;
  if (!dtype_size(x->dtype)) return GSA_ERR_DTYPE;
  if (x->d != 128 || (x->cu_seqlens ? x->B != 1 || (x->cu_bytes != 4 && x->cu_bytes != 8) : x->N != x->B)) return GSA_ERR_SHAPE;
  if (!window_plan(x->B, x->T, x->N, x->cu_seqlens != nullptr, x->H, x->Hkv, x->window, x->sinks, x->dtype, z)) return GSA_ERR_SHAPE;
  if (backward && x->ws_bytes < z.workspace()) return GSA_ERR_SHAPE;
  // a tile's rows are addressed by 32-bit offsets
  for (int64_t st : {x->q_st, x->k_st, x->v_st, backward ? x->do_st : (int64_t)0})
    if (st < 0 || st * 64 * dtype_size(x->dtype) >= (int64_t)1 << 31) return GSA_ERR_SHAPE;
  auto vec = [&](const void* p, int64_t sb, int64_t st, int64_t sh) {
    return vec_ok(p, sb, st, x->dtype) && sh % (x->dtype == GSA_DTYPE_BF16 ? 8 : 4) == 0;
  };
  if (!vec(x->q, x->q_sb, x->q_st, x->q_sh) || !vec(x->k, x->k_sb, x->k_st, x->k_sh) || !vec(x->v, x->v_sb, x->v_st, x->v_sh) ||
      (backward && !vec(x->dout, x->do_sb, x->do_st, x->do_sh)))
    return GSA_ERR_ALIGN;
  for (const void* p : {(const void*)x->o, (const void*)x->o_low, (const void*)x->dq, (const void*)x->dk, (const void*)x->dv, (const void*)x->ws})
    if (p && !aligned(p, 16)) return GSA_ERR_ALIGN;
  if (!aligned(x->lse, 4) || (x->cu_seqlens && !aligned(x->cu_seqlens, x->cu_bytes))) return GSA_ERR_ALIGN;
  a = gsa::WindowArgs{};
  a.s = {x->cu_seqlens, x->cu_bytes == 8, x->N, x->T};
  a.q = {x->q, x->q_sb, x->q_st, x->q_sh};
  a.k = {x->k, x->k_sb, x->k_st, x->k_sh};
  a.v = {x->v, x->v_sb, x->v_st, x->v_sh};
  a.B = x->B;
  a.H = x->H;
  a.Hkv = x->Hkv;
  a.W = z.W;
  a.S = z.S;
  a.scale = x->scale;
  a.scale_l2 = x->scale * gsa::kLog2e;
  if (!backward) a.scale_l2 = std::max(a.scale_l2 < 0.f ? -a.scale_l2 : a.scale_l2, 1.17549435e-38f);
  a.o = x->o;
  a.low = x->dtype == GSA_DTYPE_BF16 ? x->o_low : nullptr;
  a.lse = x->lse;
  if (backward) {
    a.dout = {x->dout, x->do_sb, x->do_st, x->do_sh};
    a.dq = x->dq;
    a.dk = x->dk;
    a.dv = x->dv;
    char* w = static_cast<char*>(x->ws);
    a.D = reinterpret_cast<float*>(w);
    a.near_keys = z.near_keys;
    a.near_split = z.near_split;
    a.near_first = z.near_first;
    a.near_at = z.near_at;
    a.far_keys = z.far_keys;
    a.far_first = z.far_first;
    a.far_rows = z.far_rows;
    a.far_at = z.far_at;
    a.far_places = z.far_places;
    a.more_at = z.more_at;
    a.more = z.more;
    a.near_parts = reinterpret_cast<float*>(w + z.D);
    a.far_parts = reinterpret_cast<float*>(w + z.D + z.near_parts);
  }
  return GSA_OK;
}
int window_outside(const gsa::WindowArgs& a, const gsa_window_args* x, bool backward, hipStream_t s) {
  if (!a.s.cu) return GSA_OK;
  const int64_t row = 128 * (int64_t)dtype_size(x->dtype);
  const gsa::Outside o = backward ? gsa::Outside{a.s, {(char*)x->dq, (char*)x->dk, (char*)x->dv}, {a.H * row, a.Hkv * row, a.Hkv * row}}
                                  : gsa::Outside{a.s, {(char*)x->o}, {a.H * row}};
  hipLaunchKernelGGL(gsa::outside_kernel, dim3(256), dim3(256), 0, s, o);
  return launch_status();
}
template <typename T, int kGroups, int kP> int launch_fwd(const gsa::WindowArgs& a, const WindowPlan& z, hipStream_t s) {
  constexpr size_t lds = gsa::WindowQueries<T, kGroups>::kBytes;
  static_assert(lds <= 160 * 1024);
  if (const int e = allow_lds<gsa::window_fwd_kernel<T, kGroups, kP>>(lds)) return e;
  hipLaunchKernelGGL((gsa::window_fwd_kernel<T, kGroups, kP>), dim3(z.slots * a.H), dim3(256), lds, s, a);
  return launch_status();
}
template <typename T, int kGroups, int kP> int launch_dq(const gsa::WindowArgs& a, const WindowPlan& z, hipStream_t s) {
  constexpr size_t lds = gsa::WindowQueries<T, kGroups>::kBytes;
  if (const int e = allow_lds<gsa::window_dq_kernel<T, kGroups, kP>>(lds)) return e;
  hipLaunchKernelGGL((gsa::window_dq_kernel<T, kGroups, kP>), dim3(z.slots * a.H), dim3(256), lds, s, a);
  return launch_status();
}
template <typename T, int kGroups, bool kFarPart, int kP> int launch_dkv(const gsa::WindowArgs& a, int64_t blocks, hipStream_t s) {
  constexpr size_t lds = gsa::WindowKeys<T, kGroups, kFarPart>::kBytes;
  static_assert(lds <= 160 * 1024);
  if (const int e = allow_lds<gsa::window_dkv_kernel<T, kGroups, kFarPart, kP>>(lds)) return e;
  hipLaunchKernelGGL((gsa::window_dkv_kernel<T, kGroups, kFarPart, kP>), dim3(blocks), dim3(256), lds, s, a);
  return launch_status();
}
template <typename T, int kP> int window_forward(const gsa::WindowArgs& a, const WindowPlan& z, hipStream_t s) {
  return z.queries == 64 ? launch_fwd<T, 2, kP>(a, z, s) : launch_fwd<T, 4, kP>(a, z, s);
}
template <typename T, int kP> int window_backward(const gsa::WindowArgs& a, const WindowPlan& z, hipStream_t s) {
  int e = z.queries == 64 ? launch_dq<T, 2, kP>(a, z, s) : launch_dq<T, 4, kP>(a, z, s);
  if (e) return e;
  const int64_t blocks = z.near * z.near_split * a.Hkv;
  if constexpr (sizeof(T) == 2) e = z.near_keys == 128 ? launch_dkv<T, 4, false, kP>(a, blocks, s) : launch_dkv<T, 2, false, kP>(a, blocks, s);
  else e = launch_dkv<T, 2, false, kP>(a, blocks, s);
  if (e) return e;
  if (z.far && (e = launch_dkv<T, sizeof(T) == 2 ? 1 : 2, true, kP>(a, z.far * a.H, s))) return e;
  if (!z.far && z.near_split == 1) return GSA_OK;
  const int64_t units = z.near_split > 1 ? z.near : z.near_places;
  hipLaunchKernelGGL(gsa::window_join_kernel<T>, dim3(units * a.Hkv, a.near_keys / 8), dim3(256), 0, s, a);
  return launch_status();
}

}  // namespace
}  // namespace gsa_host

extern "C" size_t gsa_window_attn_workspace_bytes(int B, int T, int N, int packed, int H, int Hkv, int window, int sinks, int dtype) {
  gsa_host::WindowPlan z;
  return gsa_host::window_plan(B, T, N, packed, H, Hkv, window, sinks, dtype, z) ? z.workspace() : 0;
}
extern "C" int gsa_window_attn(const gsa_window_args* x, void* stream) {
  gsa::WindowArgs a;
  gsa_host::WindowPlan z;
  if (const int e = gsa_host::window_args(x, false, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  const int e = x->dtype == GSA_DTYPE_F32 ? gsa_host::window_forward<float, 3>(a, z, s)
                : a.W + a.S <= gsa::kFine ? gsa_host::window_forward<uint16_t, 2>(a, z, s) : gsa_host::window_forward<uint16_t, 1>(a, z, s);
  return e ? e : gsa_host::window_outside(a, x, false, s);
}
extern "C" int gsa_window_attn_backward(const gsa_window_args* x, void* stream) {
  gsa::WindowArgs a;
  gsa_host::WindowPlan z;
  if (const int e = gsa_host::window_args(x, true, a, z)) return e;
  const auto s = static_cast<hipStream_t>(stream);
  const int e = x->dtype == GSA_DTYPE_F32 ? gsa_host::window_backward<float, 3>(a, z, s)
                : a.W + a.S <= gsa::kFine ? gsa_host::window_backward<uint16_t, 2>(a, z, s) : gsa_host::window_backward<uint16_t, 1>(a, z, s);
  return e ? e : gsa_host::window_outside(a, x, true, s);
}
