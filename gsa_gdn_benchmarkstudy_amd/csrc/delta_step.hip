// The gated delta rule for one token of each sequence of a serving batch, the states
// updated in place.
//
//   S' = e^g S,  u = beta (v - S'^T k),  S = S' + k u^T,  o = scale S^T q     (S [128 x 128] fp32)
//
// Bound by HBM: 64 KiB of state are read and written for each row and v head, 6 flops an
// element.  The columns of S do not depend on each other, so a block takes kCols of them,
// its piece of S in registers: one read, one write, two sums over the rows.  203 rows of 16 v heads:
// 58 us for 376 MB, 6.5 TB/s (a part of the states is in the last-level cache); one row: 4.5 us.
#include "gsa_common.h"

namespace gsa {

struct StepArgs {
  const void *q, *k, *v;              // [N, Hk, 128] (q, k), [N, Hv, 128] (v): strides of rows and heads
  int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh;
  const float* g; int64_t g_sn, g_sh;
  const void* beta; int64_t b_sn, b_sh; int beta_bf16;
  const void* at; int at64;           // [N] state of a row; null: the row itself
  float* state; int64_t s_sn, s_sh;   // [slots, Hv, 128, 128]
  void* o;                            // [N, Hv, 128]
  int N, slots, Hk, Hv;
  float scale;
};

__device__ __forceinline__ int64_t step_slot(const StepArgs& a, int n) {
  const int64_t s = !a.at ? n : a.at64 ? static_cast<const int64_t*>(a.at)[n] : static_cast<const int32_t*>(a.at)[n];
  return s >= 0 && s < a.slots ? s : -1;
}
template <typename T> __device__ __forceinline__ float elem(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 2) return bf16lo(static_cast<const T*>(p)[i]); else return static_cast<const T*>(p)[i];
}

template <typename T, int kCols>
__global__ __launch_bounds__(256) void delta_step_kernel(StepArgs a) {
  constexpr int kLanes = kCols / 4;                  // lanes of a row of the piece
  constexpr int kGroups = 256 / kLanes;              // rows side by side
  constexpr int kRows = 128 / kGroups;               // rows of a lane: group + kGroups * i
  __shared__ float qs[128], ks[128];
  __shared__ floatx4 red[2][4][kLanes];
  __shared__ int found[2];
  static_assert(64 % kLanes == 0, "a wave holds whole rows");
  const int tid = threadIdx.x, n0 = blockIdx.z, h = blockIdx.y, col = blockIdx.x * kCols + 4 * (tid % kLanes);
  const int group = tid / kLanes;
  const int64_t slot = step_slot(a, n0);
  T* out = static_cast<T*>(a.o) + ((int64_t)n0 * a.Hv + h) * 128;
  if (slot < 0) {                                    // a row of padding: no state, output 0
    if (tid < kCols) out[blockIdx.x * kCols + tid] = (T)0;
    return;
  }
  float* S = a.state + slot * a.s_sn + h * a.s_sh + col;
  floatx4 s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) s[i] = *reinterpret_cast<const floatx4*>(S + (group + kGroups * i) * 128);

  // Rows of the batch that name one state are one sequence's tokens, in the batch's order: the
  // block of the first of them takes them all.  Each block looks through all N indices, which grows with N squared
  // (4 heads, without indices and with: 4096 rows 432 and 509 us, 8192 889 and 1214, 16384 1873 and 3350, 65535 7.7 and 42 ms).
  int more = 0;
  if (a.at) {
    if (tid == 0) found[0] = found[1] = 0;
    __syncthreads();
    for (int j = tid; j < a.N; j += 256)
      if (j != n0 && step_slot(a, j) == slot) found[j > n0] = 1;
    __syncthreads();
    if (found[0]) return;
    more = found[1];
  }

  for (int n = n0;;) {
    const int hk = h / (a.Hv / a.Hk);
    if (tid < 128) {
      qs[tid] = elem<T>(a.q, n * a.q_sn + hk * a.q_sh + tid);
      ks[tid] = elem<T>(a.k, n * a.k_sn + hk * a.k_sh + tid);
    }
    const float decay = expf(a.g[n * a.g_sn + h * a.g_sh]);
    const int64_t bi = n * a.b_sn + h * a.b_sh;
    const float beta = a.beta_bf16 ? bf16lo(static_cast<const uint16_t*>(a.beta)[bi]) : static_cast<const float*>(a.beta)[bi];
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = elem<T>(a.v, n * a.v_sn + h * a.v_sh + col + c);
    __syncthreads();

    auto join = [&](floatx4 p, int which) {          // the sum over all rows, in every lane of the columns
#pragma unroll
      for (int m = kLanes; m < 64; m <<= 1)
#pragma unroll
        for (int c = 0; c < 4; ++c) p[c] += __shfl_xor(p[c], m, 64);
      if ((tid & 63) < kLanes) red[which][tid >> 6][tid % kLanes] = p;
      __syncthreads();
      return red[which][0][tid % kLanes] + red[which][1][tid % kLanes] + red[which][2][tid % kLanes] + red[which][3][tid % kLanes];
    };
    floatx4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float kk = ks[group + kGroups * i];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[i][c] *= decay;
        p[c] = __builtin_fmaf(s[i][c], kk, p[c]);
      }
    }
    p = join(p, 0);
    floatx4 u, o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) u[c] = beta * (v[c] - p[c]);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float kk = ks[group + kGroups * i], qq = qs[group + kGroups * i];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[i][c] = __builtin_fmaf(kk, u[c], s[i][c]);
        o[c] = __builtin_fmaf(s[i][c], qq, o[c]);
      }
    }
    o = join(o, 1);
    if (group == 0) {
      T* to = static_cast<T*>(a.o) + ((int64_t)n * a.Hv + h) * 128 + col;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (sizeof(T) == 2) to[c] = (T)f32_to_bf16_bits(o[c] * a.scale); else to[c] = o[c] * a.scale;
      }
    }
    if (!more) break;
    do ++n; while (n < a.N && step_slot(a, n) != slot);
    if (n >= a.N) break;
    __syncthreads();                                 // qs, ks and red are read above
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) *reinterpret_cast<floatx4*>(S + (group + kGroups * i) * 128) = s[i];
}

}  // namespace gsa

extern "C" int gsa_delta_step(const void* q, int64_t q_sn, int64_t q_sh, const void* k, int64_t k_sn, int64_t k_sh, const void* v,
                              int64_t v_sn, int64_t v_sh, const float* g, int64_t g_sn, int64_t g_sh, const void* beta,
                              int64_t b_sn, int64_t b_sh, int beta_dtype, const void* state_idx, int idx_bytes, float* state,
                              int64_t s_sn, int64_t s_sh, int N, int slots, int Hk, int Hv, int d, float scale, int dtype, void* o,
                              void* stream) {
  using namespace gsa_host;
  if (!q || !k || !v || !g || !beta || !state || !o) return GSA_ERR_NULL;
  if (!dtype_size(dtype) || !dtype_size(beta_dtype)) return GSA_ERR_DTYPE;
  if (N < 1 || N > 65535 || slots < 1 || Hk < 1 || Hv < Hk || Hv % Hk || Hv > 65535 || d != 128) return GSA_ERR_SHAPE;
  if (state_idx ? idx_bytes != 4 && idx_bytes != 8 : N > slots) return GSA_ERR_SHAPE;
  if (!aligned(state, 16) || s_sn % 4 || s_sh % 4 || !aligned(state_idx, state_idx ? idx_bytes : 1) || !aligned(g, 4) ||
      !aligned(beta, dtype_size(beta_dtype)))
    return GSA_ERR_ALIGN;
  for (const void* p : {q, k, v, (const void*)o})
    if (!aligned(p, dtype_size(dtype))) return GSA_ERR_ALIGN;
  const gsa::StepArgs a{q, k, v, q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, g, g_sn, g_sh, beta, b_sn, b_sh, beta_dtype == GSA_DTYPE_BF16,
                        state_idx, idx_bytes == 8, state, s_sn, s_sh, o, N, slots, Hk, Hv, scale};
  const auto st = static_cast<hipStream_t>(stream);
  const dim3 grid(4, Hv, N);
  if (dtype == GSA_DTYPE_BF16) hipLaunchKernelGGL((gsa::delta_step_kernel<uint16_t, 32>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((gsa::delta_step_kernel<float, 32>), grid, dim3(256), 0, st, a);
  return launch_status();
}
