// RMS norm with the residual's addition, forward and backward, and with an output
// in e4m3 with one scale a row.
//
//   h = round(x + res)   (x itself without a residual)
//   y = h r w,  r = (mean h^2 + eps)^-1/2
//   dh = dh_in + r (dy w - n mean(dy w n)),  n = h r;   dw = sum over rows of dy n
//
// Bound by HBM: every element is read once and written once, nothing else moves but
// the partial sums of dw.  A row is held in the registers of kTpr lanes
// (16 for heads of 128 up to 1024 for rows of 32768), 8 consecutive elements a slot, so
// that a lane's access is 16 (bf16) or 32 bytes; statistics in fp32.  16384 rows of 2048 in bf16
// with a residual: 46 us forward (268 MB, 5.8 TB/s), 51 backward and 5 for dw; 12289 rows of 4096
// to e4m3: 69 us (352 MB, 5.1 TB/s).
#include "gsa_common.h"

namespace gsa {

// Row r of a tensor whose rows lie in groups of `inner`: base + (r / inner) * s0 + (r % inner) * s1.
struct NormRows {
  const void* p;
  int64_t s0, s1;
};
template <typename T>
__device__ __forceinline__ const T* norm_row(const NormRows& x, int64_t r, int inner) {
  const int64_t o = inner == 1 ? r : r / inner;
  return static_cast<const T*>(x.p) + o * x.s0 + (r - o * inner) * x.s1;
}

// Slot: 8 elements from e0 of a row of D.  kVec: whole slots only, 16-byte aligned rows.
template <bool kVec, typename T>
__device__ __forceinline__ void slot_load(const T* row, int e0, int D, float (&x)[8]) {
  if (kVec) {
    if (e0 < D) {
      load8(row + e0, x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = 0.f;
      if (e0 + i < D) {
        if constexpr (sizeof(T) == 2) v = bf16lo(row[e0 + i]); else v = row[e0 + i];
      }
      x[i] = v;
    }
  }
}
// The same as it is stored, and turned to fp32.
template <typename T> struct RawSlot { u32x4 v[sizeof(T) / 2]; };
template <bool kVec, typename T>
__device__ __forceinline__ RawSlot<T> slot_raw(const T* row, int e0, int D) {
  RawSlot<T> r;
  if (kVec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = e0 < D ? reinterpret_cast<const u32x4*>(row + e0)[i] : u32x4{0, 0, 0, 0};
  } else {
    float x[8];
    slot_load<false>(row, e0, D, x);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r.v[0][i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i >> 2][i & 3] = __float_as_uint(x[i]);
    }
  }
  return r;
}
template <typename T> __device__ __forceinline__ void slot_floats(const RawSlot<T>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w = r.v[0][i >> 1];
      x[i] = i & 1 ? bf16hi(w) : bf16lo(w);
    } else {
      const uint32_t w = r.v[i >> 2][i & 3];
      x[i] = __uint_as_float(w);
    }
  }
}
template <bool kVec, typename T>
__device__ __forceinline__ void slot_store(T* row, int e0, int D, const float (&x)[8]) {
  if (kVec) {
    if (e0 < D) store8(row + e0, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e0 + i < D) {
        if constexpr (sizeof(T) == 2) row[e0 + i] = (T)f32_to_bf16_bits(x[i]); else row[e0 + i] = x[i];
      }
  }
}

// The larger of two, NaN if either is (as torch's amax).
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || a != a) ? a : b; }

// Sum (kMax: largest) over the kTpr lanes of a row, the same in all of them.  red: one float
// for each wave of the block, not in use by anyone on entry; free again after the next call's
// first barrier.
template <int kTpr, bool kMax>
__device__ __forceinline__ float row_all(float v, float* red) {
  auto join = [](float a, float b) { return kMax ? max_nan(a, b) : a + b; };
  v = join(v, dpp<0x128>(v));
  v = join(v, dpp<0x124>(v));
  v = join(v, dpp<0x122>(v));
  v = join(v, dpp<0x121>(v));
  if constexpr (kTpr >= 64) {
    v = join(v, __shfl_xor(v, 16, 64));
    v = join(v, __shfl_xor(v, 32, 64));
  }
  if constexpr (kTpr > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < kTpr / 64; ++i) v = join(v, red[i]);
  }
  return v;
}

constexpr int norm_threads(int tpr) { return tpr > 256 ? tpr : 256; }

struct NormFwd {
  NormRows x, res;        // res.p null: no residual
  const void* w;
  void* y;                // [rows, D]: T, or e4m3 (kFp8)
  void* h;                // [rows, D] T, null without a residual
  float* rstd;            // [rows], nullable
  float* scale;           // [rows] (kFp8)
  int64_t rows;
  int inner, D;
  float eps;
};

// 8 values as e4m3 bytes, rounded to nearest even; |x| <= 448 or NaN.
__device__ __forceinline__ uint2 pack_e4m3(const float (&x)[8]) {
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], b, true);
  return uint2{(uint32_t)a, (uint32_t)b};
}

template <typename T, int kTpr, int kSlots, bool kVec, bool kFp8>
__global__ __launch_bounds__(norm_threads(kTpr)) void rms_norm_kernel(NormFwd a) {
  __shared__ float red[2][norm_threads(kTpr) / 64];
  const int li = threadIdx.x % kTpr;
  const int64_t r = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (norm_threads(kTpr) / kTpr) + threadIdx.x / kTpr;
  if (r >= a.rows) return;                       // (all of a block of one row together)
  const T* x = norm_row<T>(a.x, r, a.inner);
  float h[kSlots][8];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) slot_load<kVec>(x, 8 * (li + s * kTpr), a.D, h[s]);
  if (a.res.p) {
    const T* res = norm_row<T>(a.res, r, a.inner);
    T* hout = static_cast<T*>(a.h) + r * a.D;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      float z[8];
      slot_load<kVec>(res, 8 * (li + s * kTpr), a.D, z);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[s][i] = Elem<T>::rnd(h[s][i] + z[i]);
      slot_store<kVec>(hout, 8 * (li + s * kTpr), a.D, h[s]);
    }
  }
  float w[kSlots][8];                            // on its way while the sum is joined
#pragma unroll
  for (int s = 0; s < kSlots; ++s) slot_load<kVec>(static_cast<const T*>(a.w), 8 * (li + s * kTpr), a.D, w[s]);
  float q = 0.f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) q = __builtin_fmaf(h[s][i], h[s][i], q);
  q = row_all<kTpr, false>(q, red[0]);
  const float rstd = 1.f / __builtin_sqrtf(q / (float)a.D + a.eps);
  if (a.rstd && li == 0) a.rstd[r] = rstd;
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) h[s][i] = h[s][i] * rstd * w[s][i];
  if constexpr (!kFp8) {
    T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) slot_store<kVec>(y, 8 * (li + s * kTpr), a.D, h[s]);
  } else {
    float m = 0.f;
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, __builtin_fabsf(h[s][i]));
    m = row_all<kTpr, true>(m, red[1]);
    float sc = m / 448.f;
    if (sc == 0.f) sc = 1.f;
    if (li == 0) a.scale[r] = sc;
    uint8_t* y = static_cast<uint8_t*>(a.y) + r * a.D;
    // y / scale by one reciprocal a row and a step of Newton's on the quotient, which rounds as a division does:
    // in bf16 one value in 10000 is exactly between two of e4m3, where the product alone went to either side
    // (12289 rows of 4096: 71 us with the step and without).  Below 2^-100 the reciprocal would overflow.
    const bool tiny = sc < 0x1p-100f;
    const float up = tiny ? 0x1p100f : 1.f, inv = 1.f / (sc * up);
    const float by = sc <= 3.4e38f ? sc * up : 0.f;  // (an infinite scale: finite values are 0, as in a division)
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int e0 = 8 * (li + s * kTpr);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = h[s][i] * up, q = x * inv, v = __builtin_fmaf(__builtin_fmaf(-q, by, x), inv, q);
        h[s][i] = v > 448.f ? 448.f : v < -448.f ? -448.f : v;     // (NaN stays)
      }
      const uint2 p = pack_e4m3(h[s]);
      if (kVec) {
        if (e0 < a.D) *reinterpret_cast<uint2*>(y + e0) = p;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e0 + i < a.D) y[e0 + i] = (uint8_t)((i < 4 ? p.x : p.y) >> (8 * (i & 3)));
      }
    }
  }
}

struct NormBwd {
  NormRows h, dy, dh;     // dh.p null: none
  const void* w;
  const float* rstd;
  void* dx;               // [rows, D]
  float* part;            // [blocks, D]
  int64_t rows;
  int inner, D, per;      // rows of a block: per * (rows at a time)
};

// Each block walks over consecutive rows, its share of dw in registers; the block's rows at a
// time are joined through LDS at its end.  The next row's loads are on their way while a row is
// summed (16384 rows of 2048 in bf16: 85 us without, 54 with, 268 MB: 5.0 TB/s).
template <typename T, int kTpr, int kSlots, bool kVec>
__global__ __launch_bounds__(norm_threads(kTpr)) void rms_norm_bwd_kernel(NormBwd a) {
  constexpr int kRows = norm_threads(kTpr) / kTpr;
  constexpr bool kAhead = kTpr < 1024;           // (a block of 1024 has no registers for it, nor to keep w)
  __shared__ float red[2][norm_threads(kTpr) / 64];
  __shared__ float join[kRows > 1 ? kSlots * kTpr * 8 : 1];
  const int li = threadIdx.x % kTpr, sub = threadIdx.x / kTpr;
  RawSlot<T> w[kAhead ? kSlots : 1], hr[kSlots], yr[kSlots], zr[kSlots];
  float dw[kSlots][8];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    if constexpr (kAhead) w[s] = slot_raw<kVec>(static_cast<const T*>(a.w), 8 * (li + s * kTpr), a.D);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[s][i] = 0.f;
  }
  const int64_t r0 = (int64_t)blockIdx.x * a.per * kRows + sub;
  float rstd = 0.f;
  auto load = [&](int64_t r) {                   // (past the last row that one again: no load under a condition)
    r = r < a.rows ? r : a.rows - 1;
    const T* hp = norm_row<T>(a.h, r, a.inner);
    const T* yp = norm_row<T>(a.dy, r, a.inner);
    const T* zp = norm_row<T>(a.dh.p ? a.dh : a.dy, r, a.inner);
    rstd = a.rstd[r];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      hr[s] = slot_raw<kVec>(hp, 8 * (li + s * kTpr), a.D);
      yr[s] = slot_raw<kVec>(yp, 8 * (li + s * kTpr), a.D);
      if (kAhead && a.dh.p) zr[s] = slot_raw<kVec>(zp, 8 * (li + s * kTpr), a.D);
    }
  };
  if (kAhead) load(r0);
  for (int it = 0; it < a.per; ++it) {
    const int64_t r = r0 + (int64_t)it * kRows;
    if (r >= a.rows) break;                      // (all of a block of one row together)
    if (!kAhead) load(r);
    const float rs = rstd;
    float h[kSlots][8], d[kSlots][8];
    RawSlot<T> z[kAhead ? kSlots : 1];
    float c = 0.f;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      float x[8];
      slot_floats<T>(hr[s], h[s]);
      slot_floats<T>(yr[s], d[s]);
      if constexpr (kAhead) {
        slot_floats<T>(w[s], x);
        z[s] = zr[s];
      } else {
        slot_load<kVec>(static_cast<const T*>(a.w), 8 * (li + s * kTpr), a.D, x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[s][i] *= rs;
        dw[s][i] = __builtin_fmaf(d[s][i], h[s][i], dw[s][i]);
        d[s][i] *= x[i];
        c = __builtin_fmaf(d[s][i], h[s][i], c);
      }
    }
    if (kAhead) load(r + kRows);
    c = row_all<kTpr, false>(c, red[it & 1]) / (float)a.D;
    T* dx = static_cast<T*>(a.dx) + r * a.D;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[s][i] = rs * __builtin_fmaf(-h[s][i], c, d[s][i]);
      if (a.dh.p) {
        float x[8];
        if constexpr (kAhead) slot_floats<T>(z[s], x);
        else slot_load<kVec>(norm_row<T>(a.dh, r, a.inner), 8 * (li + s * kTpr), a.D, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[s][i] += x[i];
      }
      slot_store<kVec>(dx, 8 * (li + s * kTpr), a.D, d[s]);
    }
  }
  if constexpr (kRows > 1) {                     // sums in the order of the rows: the same on every run
    for (int k = 0; k < kRows; ++k) {
      if (sub == k) {
#pragma unroll
        for (int s = 0; s < kSlots; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float* p = &join[i * kSlots * kTpr + li + s * kTpr];
            *p = k == 0 ? dw[s][i] : *p + dw[s][i];
          }
      }
      __syncthreads();
    }
    if (sub == 0) {
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[s][i] = join[i * kSlots * kTpr + li + s * kTpr];
    }
  }
  if (sub == 0) {
    float* part = a.part + (int64_t)blockIdx.x * a.D;
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * (li + s * kTpr) + i < a.D) part[8 * (li + s * kTpr) + i] = dw[s][i];
  }
}

// dw from the blocks' sums: 16 columns a block, 64 lanes' worth of parts side by side.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* part, int blocks, int D, T* dw) {
  __shared__ float s[64][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, col = blockIdx.x * 16 + x;
  float v = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int b = y; b < blocks; b += 64) v += part[(int64_t)b * D + col];
  }
  s[y][x] = v;
  __syncthreads();
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {             // the same order on every run
    if (y < o) s[y][x] += s[y + o][x];
    __syncthreads();
  }
  if (y == 0 && col < D) {
    v = s[0][x];
    if constexpr (sizeof(T) == 2) dw[col] = (T)f32_to_bf16_bits(v); else dw[col] = v;
  }
}

}  // namespace gsa

namespace gsa_host {
namespace {

constexpr int kNormMaxD = 32768;

// Lanes and slots of a row of D, the same for any number of rows (so that a row's result does not
// depend on them).  Rows of over 1024 take a block each: a wave with four slots was slower both
// for one row of 2048 (4.0 us, by a block 2.4) and for 16384 (58 us, 53; backward 57, 54).
struct NormShape { int tpr, slots; };
NormShape norm_shape(int D) {
  if (D <= 128) return {16, 1};
  if (D <= 512) return {64, 1};
  if (D <= 1024) return {64, 2};
  if (D <= 2048) return {256, 1};
  if (D <= 4096) return {256, 2};
  if (D <= 8192) return {256, 4};
  return {1024, D <= 16384 ? 2 : 4};
}

template <typename F>
int with_shape(const NormShape& s, F&& f) {
  if (s.tpr == 16) return f.template operator()<16, 1>();
  if (s.tpr == 64) return s.slots == 1 ? f.template operator()<64, 1>() : f.template operator()<64, 2>();
  if (s.tpr == 256) return s.slots == 1 ? f.template operator()<256, 1>()
                         : s.slots == 2 ? f.template operator()<256, 2>() : f.template operator()<256, 4>();
  return s.slots == 2 ? f.template operator()<1024, 2>() : f.template operator()<1024, 4>();
}

int norm_check(int64_t rows, int inner, int D, int dtype) {
  if (!dtype_size(dtype)) return GSA_ERR_DTYPE;
  if (rows < 1 || inner < 1 || rows % inner || D < 1 || D > kNormMaxD || rows > (int64_t)0x7fffffff) return GSA_ERR_SHAPE;
  return GSA_OK;
}
// Every pointer is its elements' alignment; whole slots of 16 bytes (e4m3: 8) where all of it allows that.
bool norm_vec(int D, int dtype, std::initializer_list<gsa::NormRows> in, std::initializer_list<const void*> out) {
  if (D % 8) return false;
  for (const auto& r : in)
    if (r.p && !(vec_ok(r.p, r.s0, r.s1, dtype))) return false;
  for (const void* p : out)
    if (p && !aligned(p, 16)) return false;
  return true;
}
bool elem_ok(int dtype, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (p && !aligned(p, dtype_size(dtype))) return false;
  return true;
}

// Blocks of the backward pass and the rows that each takes, `at` at a time.
int norm_blocks(int64_t rows, int at, int* per) {
  const int64_t steps = (rows + at - 1) / at;
  *per = (int)((steps + 1023) / 1024);
  return (int)((steps + *per - 1) / *per);
}

template <typename T, bool kFp8>
int launch_norm(const gsa::NormFwd& a, bool vec, hipStream_t stream) {
  return with_shape(norm_shape(a.D), [&]<int kTpr, int kSlots>() {
    constexpr int kThreads = gsa::norm_threads(kTpr);
    // one dimension of a launch holds less than 2^32 threads (more are cut off without an error)
    constexpr int64_t kMost = 1 << 21;
    const int64_t blocks = (a.rows + kThreads / kTpr - 1) / (kThreads / kTpr);
    const dim3 grid((unsigned)std::min(blocks, kMost), (unsigned)((blocks + kMost - 1) / kMost));
    if (vec) hipLaunchKernelGGL((gsa::rms_norm_kernel<T, kTpr, kSlots, true, kFp8>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((gsa::rms_norm_kernel<T, kTpr, kSlots, false, kFp8>), grid, dim3(kThreads), 0, stream, a);
    return launch_status();
  });
}

int norm_forward(bool fp8, const void* x, int64_t x_s0, int64_t x_s1, const void* res, int64_t r_s0, int64_t r_s1, const void* w,
                 float eps, int64_t rows, int inner, int D, int dtype, void* y, void* h, float* rstd, float* scale, void* stream) {
  if (!x || !w || !y || (res && !h) || (fp8 && !scale)) return GSA_ERR_NULL;
  if (const int e = norm_check(rows, inner, D, dtype)) return e;
  if (!elem_ok(dtype, {x, res, w, h, fp8 ? nullptr : y}) || !aligned(rstd, 4) || !aligned(scale, 4)) return GSA_ERR_ALIGN;
  const gsa::NormFwd a{{x, x_s0, x_s1}, {res, r_s0, r_s1}, w, y, h, rstd, scale, rows, inner, D, eps};
  const bool vec = norm_vec(D, dtype, {a.x, a.res, {w, 0, 0}}, {y, h});
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == GSA_DTYPE_BF16) return fp8 ? launch_norm<uint16_t, true>(a, vec, s) : launch_norm<uint16_t, false>(a, vec, s);
  return fp8 ? launch_norm<float, true>(a, vec, s) : launch_norm<float, false>(a, vec, s);
}

template <typename T>
int norm_backward(gsa::NormBwd a, void* dw, bool vec, hipStream_t stream) {
  int blocks = 0;
  const int e = with_shape(norm_shape(a.D), [&]<int kTpr, int kSlots>() {
    constexpr int kThreads = gsa::norm_threads(kTpr);
    blocks = norm_blocks(a.rows, kThreads / kTpr, &a.per);
    if (vec) hipLaunchKernelGGL((gsa::rms_norm_bwd_kernel<T, kTpr, kSlots, true>), dim3(blocks), dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((gsa::rms_norm_bwd_kernel<T, kTpr, kSlots, false>), dim3(blocks), dim3(kThreads), 0, stream, a);
    return launch_status();
  });
  if (e) return e;
  hipLaunchKernelGGL(gsa::rms_norm_dw_kernel<T>, dim3((a.D + 15) / 16), dim3(1024), 0, stream, a.part, blocks, a.D,
                     static_cast<T*>(dw));
  return launch_status();
}

}  // namespace
}  // namespace gsa_host

extern "C" int gsa_rms_norm(const void* x, int64_t x_s0, int64_t x_s1, const void* res, int64_t r_s0, int64_t r_s1, const void* w,
                            float eps, int64_t rows, int inner, int D, int dtype, void* y, void* h, float* rstd, void* stream) {
  return gsa_host::norm_forward(false, x, x_s0, x_s1, res, r_s0, r_s1, w, eps, rows, inner, D, dtype, y, h, rstd, nullptr, stream);
}

extern "C" int gsa_rms_norm_fp8(const void* x, int64_t x_s0, int64_t x_s1, const void* res, int64_t r_s0, int64_t r_s1,
                                const void* w, float eps, int64_t rows, int inner, int D, int dtype, void* y, float* scale,
                                void* h, void* stream) {
  return gsa_host::norm_forward(true, x, x_s0, x_s1, res, r_s0, r_s1, w, eps, rows, inner, D, dtype, y, h, nullptr, scale, stream);
}

extern "C" size_t gsa_rms_norm_backward_workspace_bytes(int64_t rows, int D) {
  if (rows < 1 || D < 1 || D > gsa_host::kNormMaxD) return 0;
  const int tpr = gsa_host::norm_shape(D).tpr;
  int per = 0;
  return (size_t)gsa_host::norm_blocks(rows, gsa::norm_threads(tpr) / tpr, &per) * D * 4;
}

extern "C" int gsa_rms_norm_backward(const void* h, int64_t h_s0, int64_t h_s1, const void* dy, int64_t dy_s0, int64_t dy_s1,
                                     const void* dh, int64_t dh_s0, int64_t dh_s1, const void* w, const float* rstd,
                                     int64_t rows, int inner, int D, int dtype, void* dx, void* dw, void* ws, size_t ws_bytes,
                                     void* stream) {
  using namespace gsa_host;
  if (!h || !dy || !w || !rstd || !dx || !dw || !ws) return GSA_ERR_NULL;
  if (const int e = norm_check(rows, inner, D, dtype)) return e;
  if (ws_bytes < gsa_rms_norm_backward_workspace_bytes(rows, D)) return GSA_ERR_SHAPE;
  if (!elem_ok(dtype, {h, dy, dh, w, dx, dw}) || !aligned(rstd, 4) || !aligned(ws, 4)) return GSA_ERR_ALIGN;
  const gsa::NormBwd a{{h, h_s0, h_s1}, {dy, dy_s0, dy_s1}, {dh, dh_s0, dh_s1}, w, rstd, dx, static_cast<float*>(ws), rows, inner, D, 0};
  const bool vec = norm_vec(D, dtype, {a.h, a.dy, a.dh, {w, 0, 0}}, {dx});
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == GSA_DTYPE_BF16 ? norm_backward<uint16_t>(a, dw, vec, s) : norm_backward<float>(a, dw, vec, s);
}
