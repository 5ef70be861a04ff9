// A cache of constant size for attention in a sliding window with first tokens, and the attention of single tokens on it.
//
// A sequence's cache has S rows of first tokens and a ring behind them: the token at position p is in row p (p < S) or
// S + (p - S) % ring.  With ring >= W every visible key of the newest token is there, and with ring >= W + n - 1 those of the
// n newest.
//
// window_write_kernel stores keys and values (those that no later token of the call overwrites).  window_step_kernel:
// one token of each row of a batch against its visible keys,
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m)
// Bound by HBM: each key and value is read once, for all query heads on it; 2 flops a byte and query head.  16 lanes take
// a key, each 8 elements in fp32 (a wave: 4 keys), and keep their own running maximum, sum and output; these are
// joined within the wave, then within the block.  Where rows times key heads are few, the keys of a row are split over
// blocks: each leaves its part in the workspace and counts itself, the last one to arrive joins the parts in their order.
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
  __device__ int64_t position(int n) const {
    return !pos ? 0 : pos64 ? static_cast<const int64_t*>(pos)[n] : static_cast<const int32_t*>(pos)[n];
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
  void* o;                                                   // [N, H, 128]
  float* parts;                                              // [N][Hkv][splits][H / Hkv][kStepPart]
  uint32_t* counters;                                        // [N][Hkv]
};
constexpr int kStepPart = kHead + 2;                         // o, m, l

// kHeads query heads of a key head at a time
template <typename T, int kHeads>
__global__ __launch_bounds__(256) void window_step_kernel(WindowStepArgs a) {
  constexpr int kKeys = 4;                                   // of 16 lanes on their way at once
  __shared__ float part[4][kHeads][kStepPart];
  __shared__ uint32_t arrived;
  const int tid = threadIdx.x, wave = tid >> 6, l = lane_id(), li = l & 15, group = tid >> 4;
  const int split = blockIdx.x, hk = blockIdx.y, n = blockIdx.z, share = a.H / a.Hkv;
  const int64_t slot = a.places.slot(n), p = a.places.position(n);
  T* out = static_cast<T*>(a.o) + ((int64_t)n * a.H + hk * share) * kHead;
  if (slot < 0 || p < 0) {                                   // a row of padding
    if (split == 0)
      for (int i = tid; i < share * kHead; i += 256) out[i] = (T)0;
    return;
  }
  // visible keys in order: tokens 0 .. first - 1, then from .. p
  const int S = a.places.S, ring = a.places.ring;
  const int first = (int)(p + 1 < S ? p + 1 : S);
  const int64_t from = p - a.W + 1 > S ? p - a.W + 1 : S;
  const int count = first + (p >= from ? (int)(p - from + 1) : 0);
  const int parts = (count + a.chunk - 1) / a.chunk;
  if (split >= parts) return;
  const int e0 = split * a.chunk, e1 = min(count, e0 + a.chunk);
  const int turn = p >= from ? (int)((from - S) % ring) : 0; // the ring's row of token `from`
  const T* kb = reinterpret_cast<const T*>(a.kc.p) + slot * a.kc.sn + hk * a.kc.sh + 8 * li;
  const T* vb = reinterpret_cast<const T*>(a.vc.p) + slot * a.vc.sn + hk * a.vc.sh + 8 * li;
  auto row = [&](int e) -> int64_t {
    if (e < first) return e;
    const int r = turn + e - first;
    return S + (r >= ring ? r - ring : r);
  };
  float* const mine = a.parts + (((int64_t)n * a.Hkv + hk) * a.splits + split) * share * kStepPart;

  for (int h0 = 0; h0 < share; h0 += kHeads) {
    const int heads = min(kHeads, share - h0);
    float q[kHeads][8], o[kHeads][8], m[kHeads], sum[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const T* qp = static_cast<const T*>(a.q) + n * a.q_sn + (hk * share + h0 + min(h, heads - 1)) * a.q_sh + 8 * li;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[h][i] = to_f32(qp[i]) * a.scale_l2;
        o[h][i] = 0.f;
      }
      m[h] = -__builtin_inff();
      sum[h] = 0.f;
    }
    for (int e = e0 + group; e < e1; e += 16 * kKeys) {
      float k[kKeys][8], v[kKeys][8];
#pragma unroll
      for (int x = 0; x < kKeys; ++x) {
        const int64_t r = row(min(e + 16 * x, e1 - 1));
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
      const float f = m[h] == -__builtin_inff() ? (sum[h] == 0.f ? 0.f : sum[h]) : __builtin_amdgcn_exp2f(m[h] - top);
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
    for (int u = tid; u < heads * kHead; u += 256) {
      const int h = u / kHead, d = u % kHead;
      float top = part[0][h][kHead];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, part[w][h][kHead]);
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = part[w][h][kHead], f = mw == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mw - top);
        x += mw == -__builtin_inff() ? part[w][h][kHead + 1] : part[w][h][kHead + 1] * f;
        y += mw == -__builtin_inff() ? part[w][h][d] : part[w][h][d] * f;
      }
      if (parts == 1) {
        out[(h0 + h) * kHead + d] = from_f32<T>(y / x);
      } else {
        float* to = mine + (h0 + h) * kStepPart;
        part_store(to + d, y);
        if (d == 0) {
          part_store(to + kHead, top);
          part_store(to + kHead + 1, x);
        }
      }
    }
  }
  if (parts == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    arrived = __hip_atomic_fetch_add(a.counters + (int64_t)n * a.Hkv + hk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != (uint32_t)(parts - 1)) return;
  const float* const all = a.parts + ((int64_t)n * a.Hkv + hk) * a.splits * share * kStepPart;
  for (int u = tid; u < share * kHead; u += 256) {
    const float* at = all + u / kHead * kStepPart;
    const int d = u % kHead;
    float top = -__builtin_inff();
    for (int s = 0; s < parts; ++s) top = fmaxf(top, part_load(at + (int64_t)s * share * kStepPart + kHead));
    float x = 0.f, y = 0.f;
    for (int s = 0; s < parts; ++s) {
      const float* ps = at + (int64_t)s * share * kStepPart;
      const float ms = part_load(ps + kHead), f = ms == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ms - top);
      x = __builtin_fmaf(part_load(ps + kHead + 1), f, x);
      y = __builtin_fmaf(part_load(ps + d), f, y);
    }
    out[u] = from_f32<T>(y / x);
  }
}

}  // namespace gsa

namespace gsa_host {
namespace {

// Keys of a block and blocks of a row and key head: as few keys (64 at least) as give some 1024 blocks.
struct StepPlan { int chunk, splits; size_t counters, parts; };
bool step_plan(int N, int H, int Hkv, int window, int sinks, StepPlan& z) {
  if (N < 1 || N > 65535 || Hkv < 1 || Hkv > 65535 || H < Hkv || H % Hkv || window < 1 || sinks < 0 ||
      (int64_t)window + sinks >= 1 << 30)
    return false;
  const int64_t keys = (int64_t)window + sinks, heads = (int64_t)N * Hkv;
  const int64_t want = std::max<int64_t>(1, 1024 / heads);
  z.chunk = (int)std::max<int64_t>(64, (keys + want - 1) / want);
  z.splits = (int)((keys + z.chunk - 1) / z.chunk);
  z.counters = up((size_t)heads * 4);
  z.parts = z.splits > 1 ? (size_t)N * z.splits * H * gsa::kStepPart * 4 : 0;
  return true;
}
int places(const void* at, int at_bytes, const void* pos, int pos_bytes, int slots, int rows, int sinks, gsa::Places& p) {
  if (slots < 1 || sinks < 0 || rows <= sinks) return GSA_ERR_SHAPE;
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
template <typename T> int launch_step(const gsa::WindowStepArgs& a, int N, hipStream_t s) {
  const dim3 grid(a.splits, a.Hkv, N);
  const int share = a.H / a.Hkv;
  if (share == 1) hipLaunchKernelGGL((gsa::window_step_kernel<T, 1>), grid, dim3(256), 0, s, a);
  else if (share == 2) hipLaunchKernelGGL((gsa::window_step_kernel<T, 2>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((gsa::window_step_kernel<T, 4>), grid, dim3(256), 0, s, a);
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

extern "C" size_t gsa_window_step_workspace_bytes(int N, int H, int Hkv, int window, int sinks) {
  gsa_host::StepPlan z;
  return gsa_host::step_plan(N, H, Hkv, window, sinks, z) ? z.counters + z.parts : 0;
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
  if (d != 128 || !step_plan(N, H, Hkv, window, sinks, z) || rows < (int64_t)window + sinks || (!cache_idx && N > slots)) return GSA_ERR_SHAPE;
  if (ws_bytes < z.counters + z.parts) return GSA_ERR_SHAPE;
  gsa::Places p;
  if (const int e = places(cache_idx, idx_bytes, positions, pos_bytes, slots, rows, sinks, p)) return e;
  if (!cache_ok(k_cache, kc_sn, kc_st, kc_sh, dtype) || !cache_ok(v_cache, vc_sn, vc_st, vc_sh, dtype) || !cache_ok(q, q_sn, 0, q_sh, dtype) ||
      (k && (!cache_ok(k, k_sn, 0, k_sh, dtype) || !cache_ok(v, v_sn, 0, v_sh, dtype))) || !aligned(o, 16) || !aligned(ws, 16))
    return GSA_ERR_ALIGN;
  const auto s = static_cast<hipStream_t>(stream);
  auto* counters = static_cast<uint32_t*>(ws);
  const gsa::Cache kc{static_cast<char*>(k_cache), kc_sn, kc_st, kc_sh}, vc{static_cast<char*>(v_cache), vc_sn, vc_st, vc_sh};
  if (k) {
    // each row a sequence of one token; its block clears the row's counters too
    const gsa::WindowWriteArgs w{{nullptr, 0, N, 1}, {k, k_sn, 0, k_sh}, {v, v_sn, 0, v_sh}, kc, vc, p, Hkv, z.splits > 1 ? counters : nullptr};
    if (const int e = launch_write(w, N, dtype, s)) return e;
  } else if (z.splits > 1) {
    if (const int e = launch_clear(counters, N * Hkv, s)) return e;
  }
  const gsa::WindowStepArgs a{q, q_sn, q_sh, kc, vc, p, H, Hkv, window, z.splits, z.chunk, scale * gsa::kLog2e, o,
                              reinterpret_cast<float*>(static_cast<char*>(ws) + z.counters), counters};
  return dtype == GSA_DTYPE_BF16 ? launch_step<uint16_t>(a, N, s) : launch_step<float>(a, N, s);
}
