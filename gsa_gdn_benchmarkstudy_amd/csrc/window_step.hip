// A cache of constant size for attention in a sliding window with first tokens, and the attention of single tokens on it.
//
// A sequence's cache has S rows of first tokens and a ring behind them: the token at position p is in row p (p < S) or
// S + (p - S) % ring.  With ring >= W every visible key of the newest token is there, and with ring >= W + n - 1 those of the
// n newest.
//
// window_write_kernel stores keys and values (those that no later token of the call overwrites).  window_step_kernel:
// one token of each row of a batch against its visible keys,
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m)
// Bound by HBM: each key and value is read once, for all query heads on it (16 at most at a time).  Each wave has its own
// running maximum, sum and output, joined within the block.  Where rows times key heads are few, the keys of a row are split
// over blocks: each leaves its part in the workspace and counts itself, the last one to arrive joins the parts in their order.
// 61 rows of 2052 keys, 16 heads on 4, bf16: 42 us for 199 MB (4.7 TB/s), the write with it; one row of 1028 keys: 10.6
// behind a write of 2.5 (nine blocks a head; one waits for the others' parts; their counters have to be clear before).
// window_write_kernel, 12289 tokens of 23 prompts: 4 key heads 17.5 us (50 MB, 2.9 TB/s), 16 80 (2.5); one prompt of 16384: 15 (4.4)
// and 57 (4.8).
#include "chunks.h"

namespace gsa {

// ---------------------------------------------------------------------------
struct Cache { char* p; int64_t sn, st, sh; };               // [slots, rows, Hkv, 128]: strides in elements
struct Places {
  const void *at, *pos;                                      // [N] slot of a sequence (null: its own number), position of its first token (null: 0)
  int at64, pos64, slots, S, ring;
  __device__ int64_t slot(int n) const {
    const int64_t s = !at ? n : at64 ? static_cast<const int64_t*>(at)[n] : static_cast<const int32_t*>(at)[n];
    return s >= 0 && s < slots ? s : -1;
  }
  __device__ int64_t position(int n) const {                 // -1: padding (from 2^62 on sums with it could pass 64 bits)
    const int64_t p = !pos ? 0 : pos64 ? static_cast<const int64_t*>(pos)[n] : static_cast<const int32_t*>(pos)[n];
    return p >= 0 && p < (int64_t)1 << 62 ? p : -1;
  }
  __device__ int64_t row(int64_t p) const { return p < S ? p : S + (p - S) % ring; }
};
struct WindowWriteArgs {
  Seqs s;
  Rows k, v;
  Cache kc, vc;
  Places places;
  int Hkv;
  uint32_t* counters;                                        // Hkv words a block to clear, nullable
};
constexpr int kWriteTokens = 64;                             // of a block

template <typename T>
__global__ __launch_bounds__(256) void window_write_kernel(WindowWriteArgs a) {
  if (a.counters)
    for (int i = threadIdx.x; i < a.Hkv; i += 256) a.counters[blockIdx.x * a.Hkv + i] = 0u;
  int c;
  const Span sp = slot_of(a.s, blockIdx.x, kWriteTokens, c);
  if (c < 0) return;
  const int64_t slot = a.places.slot(sp.n), first = a.places.position(sp.n);
  if (slot < 0 || first < 0) return;
  constexpr int kPieces = kHead * sizeof(T) / 16;
  const int t0 = c * kWriteTokens, n = min(kWriteTokens, sp.len - t0) * a.Hkv * kPieces;
  for (int u = threadIdx.x; u < n; u += 256) {
    const int piece = u % kPieces, h = u / kPieces % a.Hkv, t = t0 + u / kPieces / a.Hkv;
    const int64_t p = first + t;
    if (p >= a.places.S && (int64_t)t + a.places.ring < sp.len) continue;    // a later token takes its row
    const int64_t row = a.places.row(p);
    auto copy = [&](const Rows& x, const Cache& y) {
      const u32x4 z = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(row_at<T>(x, sp, t, h)) + 16 * piece);
      *reinterpret_cast<u32x4*>(y.p + (slot * y.sn + row * y.st + h * y.sh) * (int64_t)sizeof(T) + 16 * piece) = z;
    };
    copy(a.k, a.kc);
    copy(a.v, a.vc);
  }
}

struct WindowStepArgs {
  const void* q; int64_t q_sn, q_sh;                         // [N, H, 128]
  Cache kc, vc;
  Places places;
  int H, Hkv, W, splits, chunk;                              // chunk: keys of a block
  float scale_l2;
  Rows k, v;                                                 // [N, Hkv, 128]: keys and values that the blocks write themselves (null: written)
  int N;
  void* o;                                                   // [N, H, 128]
  float* parts;                                              // [N][Hkv][splits][H / Hkv][kStepPart]
  uint32_t* counters;                                        // [N][Hkv]
};
constexpr int kStepPart = kHead + 2;                         // o, m, l

// The new keys and values of row n's sequence, its own and those of other rows on the same slot, to the cache: one key head, by
// each block that reads them (several blocks may write the same).  Written from the CU that reads, so nothing but the wait
// orders the two.
template <typename T> __device__ __forceinline__ void write_new(const WindowStepArgs& a, int n, int hk, int64_t slot) {
  if (!a.k.p) return;
  constexpr int kPieces = kHead * sizeof(T) / 16;
  const int wave = threadIdx.x >> 6, l = lane_id(), piece = l % kPieces;
  auto put = [&](int j) {
    const int64_t p = a.places.position(j);
    if (p < 0 || l >= 2 * kPieces) return;
    const Rows& x = l < kPieces ? a.k : a.v;
    const Cache& y = l < kPieces ? a.kc : a.vc;
    const u32x4 z = *reinterpret_cast<const u32x4*>(static_cast<const char*>(x.p) + (j * x.sb + hk * x.sh) * (int64_t)sizeof(T) + 16 * piece);
    *reinterpret_cast<u32x4*>(y.p + (slot * y.sn + a.places.row(p) * y.st + hk * y.sh) * (int64_t)sizeof(T) + 16 * piece) = z;
  };
  if (!a.places.at) {
    if (wave == 0) put(n);
  } else {
    for (int j0 = 64 * wave; j0 < a.N; j0 += 256)
      for (uint64_t same = ballot64(j0 + l < a.N && a.places.slot(min(j0 + l, a.N - 1)) == slot); same; same &= same - 1)
        put(j0 + __builtin_ctzll(same));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// The visible keys of a row's token in order, e = 0 .. count - 1: tokens 0 .. first - 1, then those of the window.
struct Visible {
  int first, count, turn, S, ring;                           // turn: the ring's row of the window's first token
  __device__ Visible(const Places& x, int64_t p, int W) : S(x.S), ring(x.ring) {
    first = (int)(p + 1 < S ? p + 1 : S);
    const int64_t from = p - W + 1 > S ? p - W + 1 : S;
    count = first + (p >= from ? (int)(p - from + 1) : 0);
    turn = p >= from ? (int)((from - S) % ring) : 0;
  }
  __device__ int row(int e) const {
    const int r = turn + e - first;
    return e < first ? e : S + (r >= ring ? r - ring : r);
  }
};

// No score above -infinity: NaN, as 0 / 0 (cut3 leaves more than 0 above the line).
__device__ __forceinline__ float quotient(float y, float x) { return x == 0.f ? __builtin_nanf("") : y / x; }

// What a block's four waves hold of `heads` heads (part: o, m, l of each), joined: the outputs where the block has all of the
// row's keys, else the block's part.
template <typename T, int kHeads>
__device__ __forceinline__ void join_block(float (*part)[kHeads][kStepPart], int heads, bool whole, T* out, float* mine) {
  for (int u = threadIdx.x; u < heads * kHead; u += 256) {
    const int h = u / kHead, d = u % kHead;
    float top = part[0][h][kHead];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, part[w][h][kHead]);
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = part[w][h][kHead], f = mw == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(mw - top);
      x = __builtin_fmaf(part[w][h][kHead + 1], f, x);
      y = __builtin_fmaf(part[w][h][d], f, y);
    }
    if (whole) {
      out[u] = from_f32<T>(quotient(y, x));
    } else {
      float* to = mine + h * kStepPart;
      part_store(to + d, y);
      if (d == 0) {
        part_store(to + kHead, top);
        part_store(to + kHead + 1, x);
      }
    }
  }
}
// The parts of a row's blocks, by the last one to arrive, in their order.  Several loads are on their way at once.
template <typename T>
__device__ __forceinline__ void join_row(const WindowStepArgs& a, int n, int hk, int parts, int share, T* out, float* scratch) {
  constexpr int kSome = 64;
  float *tops = scratch, *sums = scratch + kSome;            // (the waves' parts have been read)
  uint32_t& arrived = *reinterpret_cast<uint32_t*>(scratch + 2 * kSome);
  const int tid = threadIdx.x, wave = tid >> 6, l = lane_id();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    arrived = __hip_atomic_fetch_add(a.counters + (int64_t)n * a.Hkv + hk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != (uint32_t)(parts - 1)) return;
  const float* const all = a.parts + ((int64_t)n * a.Hkv + hk) * a.splits * share * kStepPart;
  const int64_t step = (int64_t)share * kStepPart;
  for (int h0 = 0; h0 < share; h0 += kSome) {
    const int heads = min(kSome, share - h0);
    if (h0) __syncthreads();
    for (int h = wave; h < heads; h += 4) {                  // a wave a head: the maximum and the sum over its parts
      const float* at = all + (h0 + h) * kStepPart + kHead;
      float top = -__builtin_inff(), x = 0.f;
      for (int s = l; s < parts; s += 64) top = fmaxf(top, part_load(at + s * step));
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
      for (int s = l; s < parts; s += 64) {
        const float ms = part_load(at + s * step), f = ms == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ms - top);
        x = __builtin_fmaf(part_load(at + s * step + 1), f, x);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
      if (l == 0) {
        tops[h] = top;
        sums[h] = x;
      }
    }
    __syncthreads();
    for (int u = tid; u < heads * kHead; u += 256) {
      const int h = u / kHead;
      const float *at = all + (h0 + h) * kStepPart, top = tops[h];
      float y = 0.f;
      for (int s = 0; s < parts; s += 8) {
        float m[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* ps = at + min(s + i, parts - 1) * step;
          m[i] = part_load(ps + kHead);
          v[i] = part_load(ps + u % kHead);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (s + i < parts) y = __builtin_fmaf(v[i], m[i] == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[i] - top), y);
      }
      out[h0 * kHead + u] = from_f32<T>(quotient(y, sums[h]));
    }
  }
}

// fp32: 16 lanes take a key, each 8 elements (a wave: 4 keys), and keep their own running maximum, sum and output.
// kHeads query heads of a key head at a time.
template <int kHeads>
__global__ __launch_bounds__(256) void window_step_f32_kernel(WindowStepArgs a) {
  constexpr int kKeys = 4;                                   // of 16 lanes on their way at once
  __shared__ float part[4][kHeads][kStepPart];
  const int tid = threadIdx.x, wave = tid >> 6, l = lane_id(), li = l & 15, group = tid >> 4;
  const int split = blockIdx.x, hk = blockIdx.y, n = blockIdx.z, share = a.H / a.Hkv;
  const int64_t slot = a.places.slot(n), p = a.places.position(n);
  float* out = static_cast<float*>(a.o) + ((int64_t)n * a.H + hk * share) * kHead;
  if (slot < 0 || p < 0) {                                   // a row of padding
    if (split == 0)
      for (int i = tid; i < share * kHead; i += 256) out[i] = 0.f;
    return;
  }
  const Visible see(a.places, p, a.W);
  const int parts = (see.count + a.chunk - 1) / a.chunk;
  if (split >= parts) return;
  write_new<float>(a, n, hk, slot);
  const int e0 = split * a.chunk, e1 = min(see.count, e0 + a.chunk);
  const float* kb = reinterpret_cast<const float*>(a.kc.p) + slot * a.kc.sn + hk * a.kc.sh + 8 * li;
  const float* vb = reinterpret_cast<const float*>(a.vc.p) + slot * a.vc.sn + hk * a.vc.sh + 8 * li;
  float* const mine = a.parts + (((int64_t)n * a.Hkv + hk) * a.splits + split) * share * kStepPart;

  for (int h0 = 0; h0 < share; h0 += kHeads) {
    const int heads = min(kHeads, share - h0);
    float q[kHeads][8], o[kHeads][8], m[kHeads], sum[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      load8(static_cast<const float*>(a.q) + n * a.q_sn + (hk * share + h0 + min(h, heads - 1)) * a.q_sh + 8 * li, q[h]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[h][i] *= a.scale_l2;
        o[h][i] = 0.f;
      }
      m[h] = -__builtin_inff();
      sum[h] = 0.f;
    }
    for (int e = e0 + group; e < e1; e += 16 * kKeys) {
      float k[kKeys][8], v[kKeys][8];
#pragma unroll
      for (int x = 0; x < kKeys; ++x) {
        const int64_t r = see.row(min(e + 16 * x, e1 - 1));
        load8(kb + r * a.kc.st, k[x]);
        load8(vb + r * a.vc.st, v[x]);
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float s[kKeys], top = m[h];
#pragma unroll
        for (int x = 0; x < kKeys; ++x) {
          float y = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) y = __builtin_fmaf(q[h][i], k[x][i], y);
          s[x] = e + 16 * x < e1 ? row16_sum(y) : -__builtin_inff();
          top = fmaxf(top, s[x]);
        }
        const float f = top == m[h] ? 1.f : __builtin_amdgcn_exp2f(m[h] - top);
        const float minus = top == -__builtin_inff() ? 0.f : top;
        m[h] = top;
        sum[h] *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[h][i] *= f;
#pragma unroll
        for (int x = 0; x < kKeys; ++x) {
          const float w = __builtin_amdgcn_exp2f(s[x] - minus);
          if (e + 16 * x < e1) {
            sum[h] += w;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[h][i] = __builtin_fmaf(w, v[x][i], o[h][i]);
          }
        }
      }
    }
    // the wave's four groups, then the block's four waves
    if (h0) __syncthreads();                                 // part is read below
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float top = fmaxf(m[h], __shfl_xor(m[h], 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float f = m[h] == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[h] - top);
      float x = sum[h] * f;
      x += __shfl_xor(x, 16, 64);
      x += __shfl_xor(x, 32, 64);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float y = o[h][i] * f;
        y += __shfl_xor(y, 16, 64);
        y += __shfl_xor(y, 32, 64);
        if (l < 16) part[wave][h][8 * li + i] = y;
      }
      if (l == 0) {
        part[wave][h][kHead] = top;
        part[wave][h][kHead + 1] = x;
      }
    }
    __syncthreads();
    join_block<float, kHeads>(part, heads, parts == 1, out + h0 * kHead, mine + h0 * kStepPart);
  }
  if (parts > 1) join_row<float>(a, n, hk, parts, share, out, &part[0][0][0]);
}

// bf16: a wave takes 32 keys at a time, with 16 query heads of a key head in the columns of both products
// (v_mfma_f32_16x16x32_bf16; fewer heads leave columns idle, which costs nothing here): S = K Q^T with the keys' rows straight
// from memory, O^T = V^T P with V through the wave's own LDS (direct loads, transposed reads).  Key row m of tile t stands for
// key tile_row(t, m), so that a lane's 8 scores are the 8 keys that it has to hold of P.  The next 32 keys' loads run beside
// the products.  P enters as three bf16 parts (24 bits), cut and not rounded, and at least 2^-126 each: none is negative or 0,
// so that an infinity of V stays one.
__device__ __forceinline__ Parts<3> cut3(const float (&x)[8]) {
  u32x4 w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      const float least = 1.17549435e-38f;
      const uint32_t ua = __float_as_uint(fmaxf(a, least)), ub = __float_as_uint(fmaxf(b, least));
      w[n][i] = __builtin_amdgcn_perm(ub, ua, 0x07060302);   // the upper halves
      a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
      b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    }
  }
  Parts<3> r;
#pragma unroll
  for (int n = 0; n < 3; ++n) r.p[n] = __builtin_bit_cast(bf16x8, w[n]);
  return r;
}
constexpr int kStepTile = 32 * 256;                          // V of 32 keys in LDS, unit u of key t in place u ^ turn
__device__ __forceinline__ int step_turn(int t) { return (t & 7) << 1 | (t >> 3 & 1); }

__global__ __launch_bounds__(256, 2) void window_step_bf16_kernel(WindowStepArgs a) {
  constexpr int kHeads = 16;
  __shared__ __align__(16) char lds[4 * 2 * kStepTile];      // per wave two buffers; then the waves' parts
  static_assert(sizeof(lds) >= 4 * kHeads * kStepPart * 4);
  auto part = reinterpret_cast<float (*)[kHeads][kStepPart]>(lds);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane_id(), g = l >> 4, m16 = l & 15;
  const int split = blockIdx.x, hk = blockIdx.y, n = blockIdx.z, share = a.H / a.Hkv;
  const int64_t slot = a.places.slot(n), p = a.places.position(n);
  uint16_t* out = static_cast<uint16_t*>(a.o) + ((int64_t)n * a.H + hk * share) * kHead;
  if (slot < 0 || p < 0) {                                   // a row of padding
    if (split == 0)
      for (int i = tid; i < share * kHead; i += 256) out[i] = 0;
    return;
  }
  const Visible see(a.places, p, a.W);
  const int parts = (see.count + a.chunk - 1) / a.chunk;
  if (split >= parts) return;
  write_new<uint16_t>(a, n, hk, slot);
  const int e0 = split * a.chunk, e1 = min(see.count, e0 + a.chunk);
  const uint16_t* kb = reinterpret_cast<const uint16_t*>(a.kc.p) + slot * a.kc.sn + hk * a.kc.sh;
  const uint16_t* vb = reinterpret_cast<const uint16_t*>(a.vc.p) + slot * a.vc.sn + hk * a.vc.sh;
  float* const mine = a.parts + (((int64_t)n * a.Hkv + hk) * a.splits + split) * share * kStepPart;
  char* const own = lds + wave * 2 * kStepTile;
  const uint32_t own_at = lds_addr(own);
  // transposed reads: keys 8 g + 4 e + i / 4 of the tile, elements 16 dt + 4 (i % 4) .. + 3
  int col[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
    col[d] = (8 * g + (m16 >> 2)) * 256 + 8 * (m16 & 1) + 16 * ((2 * d + ((m16 & 3) >> 1)) ^ (2 * (m16 >> 2) + (g & 1)));

  for (int h0 = 0; h0 < share; h0 += kHeads) {
    const int heads = min(kHeads, share - h0);
    bf16x8 q[4];
    {
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + n * a.q_sn + (hk * share + h0 + min(m16, heads - 1)) * a.q_sh + 8 * g;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) q[ks] = *reinterpret_cast<const bf16x8*>(qp + 32 * ks);
    }
    floatx4 o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), sum = 0.f;
    bf16x8 k[2][4];
    auto load = [&](int e, int buffer) {                     // keys e .. e + 31 (past the last: it again)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint16_t* at = kb + (int64_t)see.row(min(e + 8 * (m16 >> 2) + 4 * t + (m16 & 3), e1 - 1)) * a.kc.st + 8 * g;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) k[t][ks] = *reinterpret_cast<const bf16x8*>(at + 32 * ks);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 4 * j + g;
        load_lds16_at(vb + (int64_t)see.row(min(e + t, e1 - 1)) * a.vc.st + 8 * (m16 ^ step_turn(t)),
                      __builtin_amdgcn_readfirstlane(own_at + buffer * kStepTile + j * 1024));
      }
    };
    int e = e0 + 32 * wave, buffer = 0;
    if (e < e1) load(e, 0);
    for (; e < e1; e += 128, buffer ^= 1) {
      wait_loads();
      floatx4 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[t][ks], q[ks], s[t], 0, 0, 0);
      }
      if (e + 128 < e1) load(e + 128, buffer ^ 1);
      float x[8], top = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = e + 8 * g + i < e1 ? s[i >> 2][i & 3] * a.scale_l2 : -__builtin_inff();
        top = fmaxf(top, x[i]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float f = top == m ? 1.f : __builtin_amdgcn_exp2f(m - top), minus = top == -__builtin_inff() ? 0.f : top;
      m = top;
      sum *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - minus);
        sum += x[i];
      }
      const Parts<3> w = cut3(x);
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        s16x4 y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          y[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
              own + buffer * kStepTile + col[dt & 3] + 1024 * i + 16 * ((dt & 4 ? 8 : 0) ^ (8 * i))));
        const bf16x8 v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7));
        o[dt] *= f;
#pragma unroll
        for (int i = 2; i >= 0; --i) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w.p[i], o[dt], 0, 0, 0);
      }
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    __syncthreads();                                         // the waves' buffers are free
    if (m16 < heads) {
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave][m16][16 * dt + 4 * g + r] = o[dt][r];
      if (g == 0) {
        part[wave][m16][kHead] = m;
        part[wave][m16][kHead + 1] = sum;
      }
    }
    __syncthreads();
    join_block<uint16_t, kHeads>(part, heads, parts == 1, out + h0 * kHead, mine + h0 * kStepPart);
    if (h0 + kHeads < share) __syncthreads();
  }
  if (parts > 1) join_row<uint16_t>(a, n, hk, parts, share, out, &part[0][0][0]);
}

}  // namespace gsa

namespace gsa_host {
namespace {

// Keys of a block (a multiple of 128: four waves of 32) and blocks of a row and key head: a row's keys are split where the key
// heads of all rows are fewer than half of the blocks that the card wants, one a CU in bf16, two in fp32.  us in a graph, 16 heads on
// 4, by blocks in all (the write, 4-5, included); the join is what more of them cost:
//   1 row, window 1024: 12.3 (9 blocks a head: 36)        16 rows, 4096:  64 blocks 36   256: 30.5 (taken)   512: 31.5  1024: 35
//   1 row, 8192:   256: 18.3 (taken)  512: 23.8  1024: 24.6    24 rows, 2048:  96: 32.9   192: 26.9 (taken)   288: 31.0
//   4 rows, 4096:  128: 19.3  256: 17.7 (taken)  512: 20.3     33 rows, 2048: 132: 33.6 (taken)  264: 39.8   396: 33.0
//   1 row, 65536:  256: 38.7 (taken)  512: 46.7  4096: 119     61 rows, 2048: 244: 45.0 (taken)  488: 49.4   976: 53.5
//   fp32, 16 rows, 4096:  256: 57.7  512: 54.1 (taken)  1024: 57.3    33 rows, 2048:  132: 89.8  396: 56.7 (taken)  528: 70.2
struct StepPlan { int chunk, splits; size_t counters, parts; };
bool step_plan(int N, int H, int Hkv, int window, int sinks, int dtype, StepPlan& z) {
  if (!dtype_size(dtype) || N < 1 || N > 65535 || Hkv < 1 || Hkv > 65535 || H < Hkv || H % Hkv || window < 1 || sinks < 0 ||
      (int64_t)window + sinks >= 1 << 30)
    return false;
  const int64_t keys = (int64_t)window + sinks, heads = (int64_t)N * Hkv;
  const int64_t want = std::max<int64_t>(1, (dtype == GSA_DTYPE_BF16 ? 256 : 512) / heads);
  z.chunk = (int)((std::max<int64_t>(1, (keys + want - 1) / want) + 127) / 128 * 128);
  z.splits = (int)((keys + z.chunk - 1) / z.chunk);
  z.counters = up((size_t)heads * 4);
  z.parts = z.splits > 1 ? (size_t)N * z.splits * H * gsa::kStepPart * 4 : 0;
  return true;
}
constexpr int kLooked = 512;                                 // indices that a block looks through
int places(const void* at, int at_bytes, const void* pos, int pos_bytes, int slots, int rows, int sinks, gsa::Places& p) {
  if (slots < 1 || sinks < 0 || rows <= sinks || rows >= 1 << 30) return GSA_ERR_SHAPE;    // (rows are added up in 32 bits)
  if ((at && at_bytes != 4 && at_bytes != 8) || (pos && pos_bytes != 4 && pos_bytes != 8)) return GSA_ERR_SHAPE;
  if ((at && !aligned(at, at_bytes)) || (pos && !aligned(pos, pos_bytes))) return GSA_ERR_ALIGN;
  p = {at, pos, at_bytes == 8, pos_bytes == 8, slots, sinks, rows - sinks};
  return GSA_OK;
}
bool cache_ok(const void* p, int64_t sn, int64_t st, int64_t sh, int dtype) {
  return vec_ok(p, sn, st, dtype) && sh % (dtype == GSA_DTYPE_BF16 ? 8 : 4) == 0;
}
int launch_write(const gsa::WindowWriteArgs& a, int64_t blocks, int dtype, hipStream_t s) {
  if (dtype == GSA_DTYPE_BF16) hipLaunchKernelGGL(gsa::window_write_kernel<uint16_t>, dim3(blocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(gsa::window_write_kernel<float>, dim3(blocks), dim3(256), 0, s, a);
  return launch_status();
}
int launch_step(const gsa::WindowStepArgs& a, int N, int dtype, hipStream_t s) {
  const dim3 grid(a.splits, a.Hkv, N);
  const int share = a.H / a.Hkv;
  // fp32, 16 rows of 2048 keys, query heads of a key head at a time: 16 heads on 4: 1 93, 2 54, 4 38 us; 64 on 8: 343, 178, 99
  if (dtype == GSA_DTYPE_BF16) hipLaunchKernelGGL(gsa::window_step_bf16_kernel, grid, dim3(256), 0, s, a);
  else if (share == 1) hipLaunchKernelGGL(gsa::window_step_f32_kernel<1>, grid, dim3(256), 0, s, a);
  else if (share == 2) hipLaunchKernelGGL(gsa::window_step_f32_kernel<2>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(gsa::window_step_f32_kernel<4>, grid, dim3(256), 0, s, a);
  return launch_status();
}

}  // namespace
}  // namespace gsa_host

extern "C" int gsa_window_cache_write(const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st,
                                      int64_t v_sh, const void* cu_seqlens, int cu_bytes, int B, int T, int N, int Hkv, int d, int dtype,
                                      const void* positions, int pos_bytes, const void* cache_idx, int idx_bytes, void* k_cache,
                                      int64_t kc_sn, int64_t kc_st, int64_t kc_sh, void* v_cache, int64_t vc_sn, int64_t vc_st, int64_t vc_sh,
                                      int slots, int rows, int sinks, void* stream) {
  using namespace gsa_host;
  if (!k || !v || !k_cache || !v_cache) return GSA_ERR_NULL;
  if (!dtype_size(dtype)) return GSA_ERR_DTYPE;
  if (B < 1 || T < 1 || N < 1 || Hkv < 1 || Hkv > 65535 || d != 128) return GSA_ERR_SHAPE;
  if (cu_seqlens ? B != 1 || (cu_bytes != 4 && cu_bytes != 8) : N != B) return GSA_ERR_SHAPE;
  const int64_t blocks = cu_seqlens ? (int64_t)T / gsa::kWriteTokens + N : (int64_t)B * ((T + gsa::kWriteTokens - 1) / gsa::kWriteTokens);
  if (blocks >= 1 << 23 || (!cache_idx && N > slots)) return GSA_ERR_SHAPE;
  gsa::WindowWriteArgs a{};
  if (const int e = places(cache_idx, idx_bytes, positions, pos_bytes, slots, rows, sinks, a.places)) return e;
  if (!cache_ok(k, k_sb, k_st, k_sh, dtype) || !cache_ok(v, v_sb, v_st, v_sh, dtype) || !cache_ok(k_cache, kc_sn, kc_st, kc_sh, dtype) ||
      !cache_ok(v_cache, vc_sn, vc_st, vc_sh, dtype) || (cu_seqlens && !aligned(cu_seqlens, cu_bytes)))
    return GSA_ERR_ALIGN;
  a.s = {cu_seqlens, cu_bytes == 8, N, T};
  a.k = {k, k_sb, k_st, k_sh};
  a.v = {v, v_sb, v_st, v_sh};
  a.kc = {static_cast<char*>(k_cache), kc_sn, kc_st, kc_sh};
  a.vc = {static_cast<char*>(v_cache), vc_sn, vc_st, vc_sh};
  a.Hkv = Hkv;
  return launch_write(a, blocks, dtype, static_cast<hipStream_t>(stream));
}

extern "C" size_t gsa_window_step_workspace_bytes(int N, int H, int Hkv, int window, int sinks, int dtype) {
  gsa_host::StepPlan z;
  return gsa_host::step_plan(N, H, Hkv, window, sinks, dtype, z) ? z.counters + z.parts : 0;
}
extern "C" int gsa_window_step(const void* q, int64_t q_sn, int64_t q_sh, const void* k, int64_t k_sn, int64_t k_sh, const void* v,
                               int64_t v_sn, int64_t v_sh, const void* positions, int pos_bytes, const void* cache_idx, int idx_bytes,
                               void* k_cache, int64_t kc_sn, int64_t kc_st, int64_t kc_sh, void* v_cache, int64_t vc_sn, int64_t vc_st,
                               int64_t vc_sh, int N, int slots, int rows, int H, int Hkv, int d, int window, int sinks, float scale,
                               int dtype, void* o, void* ws, size_t ws_bytes, void* stream) {
  using namespace gsa_host;
  if (!q || !positions || !k_cache || !v_cache || !o || !ws || !k != !v) return GSA_ERR_NULL;
  if (!dtype_size(dtype)) return GSA_ERR_DTYPE;
  StepPlan z;
  if (d != 128 || !step_plan(N, H, Hkv, window, sinks, dtype, z) || rows < (int64_t)window + sinks || (!cache_idx && N > slots)) return GSA_ERR_SHAPE;
  if (ws_bytes < z.counters + z.parts) return GSA_ERR_SHAPE;
  gsa::Places p;
  if (const int e = places(cache_idx, idx_bytes, positions, pos_bytes, slots, rows, sinks, p)) return e;
  if (!cache_ok(k_cache, kc_sn, kc_st, kc_sh, dtype) || !cache_ok(v_cache, vc_sn, vc_st, vc_sh, dtype) || !cache_ok(q, q_sn, 0, q_sh, dtype) ||
      (k && (!cache_ok(k, k_sn, 0, k_sh, dtype) || !cache_ok(v, v_sn, 0, v_sh, dtype))) || !aligned(o, 16) || !aligned(ws, 16))
    return GSA_ERR_ALIGN;
  const auto s = static_cast<hipStream_t>(stream);
  auto* counters = static_cast<uint32_t*>(ws);
  const gsa::Cache kc{static_cast<char*>(k_cache), kc_sn, kc_st, kc_sh}, vc{static_cast<char*>(v_cache), vc_sn, vc_st, vc_sh};
  // Whole rows: each block writes what it reads, a launch less.  It looks through all indices for that, so where they are many
  // the write has a launch of its own.  us with it / without: 61 rows of 2052 keys 45.0 / 42.2, 33 of 516 15.5 / 13.5, 300 of 132
  // 26.7 / 26.0, 300 of 1028 124 / 121, 1000 of 260 116 / 131, 4000 of 132 75 / 107 (without indices 75 / 75).
  const bool writes = k && z.splits == 1 && (!cache_idx || N <= kLooked);
  if (k && !writes) {
    // each row a sequence of one token; its block clears the row's counters too
    const gsa::WindowWriteArgs w{{nullptr, 0, N, 1}, {k, k_sn, 0, k_sh}, {v, v_sn, 0, v_sh}, kc, vc, p, Hkv, z.splits > 1 ? counters : nullptr};
    if (const int e = launch_write(w, N, dtype, s)) return e;
  } else if (!k && z.splits > 1) {
    if (const int e = launch_clear(counters, N * Hkv, s)) return e;
  }
  const gsa::WindowStepArgs a{q, q_sn, q_sh, kc, vc, p, H, Hkv, window, z.splits, z.chunk, scale * gsa::kLog2e,
                              {writes ? k : nullptr, k_sn, 0, k_sh}, {writes ? v : nullptr, v_sn, 0, v_sh}, N, o,
                              reinterpret_cast<float*>(static_cast<char*>(ws) + z.counters), counters};
  return launch_step(a, N, dtype, s);
}
