// Linear recurrences over whole sequences in chunks of tokens: what the gated delta rule and
// linear attention share.  Operands of the matrix instructions in bf16 parts, sequences and their
// chunks, rows of a chunk in LDS, and the launches' small parts.
#pragma once

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
// tile_row(t, 4 g + r) = 8 g + tile_at(t, r): a lane's part and one the compiler knows.
constexpr int tile_at(int t, int r) { return 32 * (t >> 1) + 4 * (t & 1) + r; }

template <int N> struct Parts { bf16x8 p[N]; };

// Rounded to bf16 by pairs (one v_cvt_pk_bf16_f32); what is left of them.
__device__ __forceinline__ uint32_t take_part(float& x, float& y) {
  uint32_t p = pack_bf16(x, y);
  asm("" : "+v"(p));                                         // (else the compiler converts x once more by itself)
  x -= bf16lo(p);
  y -= bf16hi(p);
  return p;
}
template <int N> __device__ __forceinline__ Parts<N> parts_of(const float (&x)[8]) {
  u32x4 w[N];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) w[n][i] = n + 1 < N ? take_part(a, b) : pack_bf16(a, b);
  }
  Parts<N> r;
#pragma unroll
  for (int n = 0; n < N; ++n) r.p[n] = __builtin_bit_cast(bf16x8, w[n]);
  return r;
}
__device__ __forceinline__ Parts<3> split3(const float (&x)[8]) { return parts_of<3>(x); }
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

// acc[i][n] += a[i] b[n] for NT columns of tiles: part by part over all of them, so that an
// instruction does not wait for the one before it.
template <int M, int NT, int NA, int NB>
__device__ __forceinline__ void mma_grid(floatx4 (*acc)[NT], const Parts<NA> (&a)[M], const Parts<NB> (&b)[NT]) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (i + j == o)
#pragma unroll
          for (int t = 0; t < M; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t].p[i], b[n].p[j], acc[t][n], 0, 0, 0);
}

template <typename T> struct ChunkType;
template <> struct ChunkType<uint16_t> { static constexpr int kParts = 1, kChunk = 64; };
template <> struct ChunkType<float> { static constexpr int kParts = 3, kChunk = 32; };

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
  int cu64, N, T;
  __device__ int64_t at(int n) const {
    const int64_t x = cu64 ? static_cast<const int64_t*>(cu)[n] : static_cast<const int32_t*>(cu)[n];
    return x < 0 ? 0 : x > T ? T : x;
  }
};
struct Span { int n, b, t0, len, slot0; };                   // sequence n: tokens t0 .. t0 + len - 1 of row b
__device__ __forceinline__ Span span_of(const Seqs& s, int n, int ch) {       // slots of ch tokens
  if (!s.cu) return Span{n, n, 0, s.T, n * ((s.T + ch - 1) / ch)};
  const int a = __builtin_amdgcn_readfirstlane((int)s.at(n)), e = __builtin_amdgcn_readfirstlane((int)s.at(n + 1));
  return Span{n, 0, a, e > a ? e - a : 0, a / ch + n};
}
// The sequence of a slot, and which of its pieces it is; c < 0: an empty slot.
__device__ __forceinline__ Span slot_of(const Seqs& s, int slot, int ch, int& c) {
  if (!s.cu) {
    const int nc = (s.T + ch - 1) / ch, n = slot / nc;
    c = slot - n * nc;
    return span_of(s, n, ch);
  }
  int lo = 0, hi = s.N - 1;                                  // the last n whose first slot is not behind
  while (lo < hi) {
    const int m = (lo + hi + 1) / 2;
    if (__builtin_amdgcn_readfirstlane((int)s.at(m)) / ch + m <= slot) lo = m; else hi = m - 1;
  }
  const Span r = span_of(s, lo, ch);
  c = slot - r.slot0;
  if (c < 0 || c >= (r.len + ch - 1) / ch) c = -1;
  return r;
}

template <typename T> __device__ __forceinline__ const T* row_at(const Rows& x, const Span& s, int64_t t, int h) {
  return static_cast<const T*>(x.p) + s.b * x.sb + (s.t0 + t) * x.st + h * x.sh;
}

// 8 consecutive elements of a row as an operand (zeros where !ok).
template <typename T> __device__ __forceinline__ Parts<ChunkType<T>::kParts> operand(const T* p, bool ok) {
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

constexpr int kUnit = 1024;
// A chunk's square matrices are lower triangular: of their (tile, step) operands the ones that
// are not 0 everywhere, with rows of tokens t and steps of 32 summed over (transposed: the
// steps from t's on).
template <int C> struct Square {
  static constexpr int kFrags = C == 64 ? 6 : 2;
  static constexpr int at(int tile, int js, bool transposed) {
    return C == 32 ? tile : transposed ? (tile < 2 ? 2 * tile + js : 2 + tile) : (tile < 2 ? tile : 2 * tile - 2 + js);
  }
  // its tile and step
  __device__ static int2 of(int f, bool transposed) {
    if (C == 32) return int2{f, 0};
    if (transposed) return f < 4 ? int2{f >> 1, f & 1} : int2{f - 2, 1};
    return f < 2 ? int2{f, 0} : int2{(f + 2) >> 1, f & 1};
  }
};

// A chunk's rows of 128 elements: unit (tile, step of 32 elements, part), lane's place row_slot(g, m)
// for row m's elements 8 g .. + 7.  The places turn with g, so that neither the lanes of an
// operand with rows of tokens (rows_of) nor those of its transpose (cols_of) meet in a bank.
__device__ __forceinline__ int row_slot(int g, int m) { return 16 * g + ((m + 4 * g) & 15); }
template <typename T>
__device__ __forceinline__ void stage_rows(bf16x8* dst, const Rows& x, const Span& sp, int64_t t0, int left, int h, int tid) {
  constexpr int C = ChunkType<T>::kChunk, NP = ChunkType<T>::kParts;
  for (int u = tid; u < C * 16; u += 256) {
    const int d8 = u & 15, t = u >> 4;
    const int tile = 2 * (t >> 5) + ((t >> 2) & 1), m = 4 * ((t >> 3) & 3) + (t & 3);
    const Parts<NP> p = operand<T>(row_at<T>(x, sp, t0 + t, h) + 8 * d8, t < left);
#pragma unroll
    for (int i = 0; i < NP; ++i) dst[((tile * 4 + (d8 >> 2)) * NP + i) * 64 + row_slot(d8 & 3, m)] = p.p[i];
  }
}
template <int N> __device__ __forceinline__ Parts<N> staged(const bf16x8* src, int frag, int l) {
  Parts<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.p[i] = src[(frag * N + i) * 64 + l];
  return r;
}
// Rows of tokens (tile), elements 32 ks .. + 31; slot: the lane's row_slot.
template <int N> __device__ __forceinline__ Parts<N> rows_of(const char* src, int tile, int ks, int slot) {
  return staged<N>(reinterpret_cast<const bf16x8*>(src), tile * 4 + ks, slot);
}
// The transpose: rows of elements tile_row(t, .), tokens 32 js .. + 31 (ds_read_b64_tr_b16: of 16
// lanes, lane i names row i / 4, elements 4 (i % 4) .. + 3 of 16, and gets element i of the four
// rows).  place: the lane's cols_place.
__device__ __forceinline__ int cols_place(int l) {
  const int i = l & 15;
  return 16 * row_slot(i & 3, 4 * (l >> 4) + (i >> 2));
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <int N> __device__ __forceinline__ Parts<N> cols_of(const char* src, int t, int js, int place) {
  Parts<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s16x4 x[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      x[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
          src + (((2 * js + e) * 4 + (t >> 1)) * N + i) * 1024 + place + 8 * (t & 1)));
    r.p[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
  return r;
}

// Blocks go to the 8 XCDs in turn, each with an L2 of its own: the kBlocks blocks of one head stand 8
// apart, so that they share one.  The unit (head and sequence or segment) and block of a block
// index; the grid has blocks_for(units) of them, some without a unit.
template <int kBlocks> __device__ __forceinline__ int2 unit_of(int b) {
  return kBlocks == 1 ? int2{b, 0} : int2{b / (8 * kBlocks) * 8 + b % 8, b / 8 % kBlocks};
}
constexpr int64_t blocks_for(int64_t units, int blocks) { return blocks == 1 ? units : (units + 7) / 8 * 8 * blocks; }

template <typename P> __device__ __forceinline__ const P* uniform(const P* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  const uint64_t y = (uint64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
  return (const P*)(__attribute__((address_space(1))) const P*)y;      // global memory, said so that accesses are not flat ones
}
// x, of which the compiler knows nothing: what it computes from it stays where it is used, instead of being kept
// over a loop in registers that are then spilled (and what reads those back waits for every load in flight).
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
// All loads have landed, the direct ones to LDS too, and the compiler knows it: waits of its own for registers loaded before a
// loop would stand inside it, where they wait for the next tile's direct loads, which it does not count.
// kLeft: but for the last so many.
template <int kLeft = 0> __device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0 + kLeft);
  asm volatile("" ::: "memory");
}

// `units` KiB from src (16-byte aligned) to LDS, by W waves.
template <int W> __device__ __forceinline__ void fetch(const void* src, uint32_t lds, int units, int wave, int l) {
  const char* p = uniform(static_cast<const char*>(src));
  for (int i = wave; i < units; i += W) load_lds16(p + (size_t)i * kUnit, 16u * l, __builtin_amdgcn_readfirstlane(lds + i * kUnit));
}
// The rows of a chunk (tile_row, summed over the 128 elements) straight from bf16 rows; rows behind
// the sequence are its last one again (what they give is not used).
template <int C, int W>
__device__ __forceinline__ void fetch_rows(const Rows& x, const Span& sp, int64_t t0, int left, int h, uint32_t lds, int wave, int l) {
  const uint16_t* p = uniform(row_at<uint16_t>(x, sp, t0, h));
  const int m = (l - 4 * (l >> 4)) & 15;                     // (row_slot)
#pragma unroll
  for (int i = 0; i < C / 4 / W; ++i) {
    const int f = wave + W * i, t = min(tile_row(f >> 2, m), left - 1);
    load_lds16(p, (uint32_t)(t * (int)x.st + 32 * (f & 3) + 8 * (l >> 4)) * 2u, __builtin_amdgcn_readfirstlane(lds + f * kUnit));
  }
}

// A [rows][128] fp32 matrix <-> the wave's tiles of it (rows tile_row, columns from col0).  The
// row is a uniform address, the lane's part the same for all of them.
template <int kTiles, int NT>
__device__ __forceinline__ void tiles_load(floatx4 (&S)[kTiles][NT], const float* p, int col0, int l) {
  const float* q = uniform(p) + col0;
  const uint32_t off = 8 * (l >> 4) * kHead + (l & 15);
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[t][n][r] = (q + tile_at(t, r) * kHead + 16 * n)[off];
}
template <int kTiles, int NT>
__device__ __forceinline__ void tiles_store(const floatx4 (&S)[kTiles][NT], float* p, int col0, int l) {
  float* q = const_cast<float*>(uniform(p)) + col0;
  const uint32_t off = 8 * (l >> 4) * kHead + (l & 15);
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) (q + tile_at(t, r) * kHead + 16 * n)[off] = S[t][n][r];
}

// Zeros to the rows of T that no packed sequence holds: before the first offset and behind the largest (5 us: a launch).
// 256 threads; bytes: of a token's row in each array.
struct Outside {
  Seqs s;
  char* p[5];
  int64_t bytes[5];
};
// By the first 256 threads of each of `blocks` blocks.
__device__ __forceinline__ void clear_outside(const Outside& a, int block, int blocks) {
  __shared__ int most[4];
  int hi = 0;
  const bool on = threadIdx.x < 256;
  for (int n = threadIdx.x; on && n <= a.s.N; n += 256) hi = max(hi, (int)a.s.at(n));
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) hi = max(hi, __shfl_xor(hi, o, 64));
  if (on && (threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = hi;
  __syncthreads();
  hi = max(max(most[0], most[1]), max(most[2], most[3]));
  if (!on) return;
  const int64_t lo = a.s.at(0);
  for (int i = 0; i < 5; ++i) {
    if (!a.p[i]) continue;
    auto clear = [&](int64_t from, int64_t to) {             // whole elements, 2 bytes at least
      uint16_t* p = reinterpret_cast<uint16_t*>(a.p[i] + from * a.bytes[i]);
      for (int64_t k = (int64_t)block * 256 + threadIdx.x; k < (to - from) * a.bytes[i] / 2; k += (int64_t)blocks * 256) p[k] = 0;
    };
    clear(0, lo);
    clear(hi, a.s.T);
  }
}

[[maybe_unused]] static __global__ __launch_bounds__(256) void outside_kernel(Outside a) { clear_outside(a, blockIdx.x, gridDim.x); }

}  // namespace gsa

namespace gsa_host {

constexpr size_t kAlign = 256;
inline size_t up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

// More than the default 64 KiB of LDS for a kernel (a benign race: concurrent first calls set the same attribute).
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

}  // namespace gsa_host
