// quant_rows.cu — rows rounded to 8 bits with a scale each: of values as they are, and of a root-mean-
// square norm with the residual's addition in front of it.
//
// With t_j = x_j (quantize) or t_j = f32(h_j w_j), h = round(x + r) (norm), and m = max_j |t_j|:
//     q_j = round_half_even(127 t_j / m),   scale = m / 127  [* 1 / sqrt(mean(h^2) + eps)]
// The norm's factor is the same for the whole row, so it cancels in q and enters the scale alone: a row
// needs one reduction of the pair (sum h^2, max |t|), after which every value is rounded from registers.
//
// q is the exact quotient's rounding, not that of f32 arithmetic: t * (127 / m) is off by less than
// 127 * 2^-23 = 1.6e-5, so a value further than kBorder = 2^-15 from a border between two integers is
// rounded right in f32, and the few others (6e-5 of them) are divided in 64 bits, where the quotient of
// two f32 values cannot cross or miss a border.  The result then depends on no order of operations.
//
// The maximum is taken on the bit patterns of |t| as integers, which order like the values with
// infinity and NaN on top: a row that holds either is seen by the same reduction.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "../../../include/b200_kernels.h"

namespace b200k {
namespace {

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kBorder = 0.5f - 1.0f / 32768.0f;
constexpr float kRoundMagic = 12582912.0f;     // 1.5 * 2^23: adding it rounds |v| < 2^22 to an integer
constexpr int kMaxThreads = 1024;

struct RowArgs {
  const void* x;
  const void* r;        // residual, or null
  const void* w;        // norm weight
  void* h;              // x + r rounded, or null; may be x or r
  int8_t* q;
  float* scale;
  long long ldx, ldr, ldh, ldq;
  int rows, cols;
  int w_type;           // 0 f32, 1 bf16, 2 f16
  float eps;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }

// VEC consecutive elements as f32; one 4-, 8- or 16-byte access each (two of 16 for eight f32).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&o)[VEC]) {
  const Pack<T, VEC> k = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = to_f32(k.v[i]);
}
template <int VEC>
__device__ __forceinline__ void load_weight(const void* w, int type, long long at, float (&o)[VEC]) {
  if (type == 0) load_vec<float, VEC>((const float*)w + at, o);
  else if (type == 1) load_vec<__nv_bfloat16, VEC>((const __nv_bfloat16*)w + at, o);
  else load_vec<__half, VEC>((const __half*)w + at, o);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// round_half_even(127 t / m) as a byte; inv = 127 / m in f32.
__device__ __forceinline__ uint32_t round_i8(float t, float inv, float m) {
  const float v = t * inv;
  const float s = v + kRoundMagic;
  uint32_t k = __float_as_uint(s);
  // also taken where inv overflowed (m below 127 / FLT_MAX) and v is no number
  if (!(fabsf(v - (s - kRoundMagic)) < kBorder)) k = (uint32_t)__double2int_rn(127.0 * (double)t / (double)m);
  return k & 0xffu;
}

// Sum and maximum over the threads of one row: the warp, or (BLOCK) the whole block.
template <bool BLOCK>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& mx) {
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if constexpr (BLOCK) {
    __shared__ float s_ss[32];
    __shared__ uint32_t s_mx[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) {
      s_ss[warp] = ss;
      s_mx[warp] = mx;
    }
    __syncthreads();
    ss = lane < warps ? s_ss[lane] : 0.f;
    mx = lane < warps ? s_mx[lane] : 0u;
    __syncthreads();                             // the slots may be written again
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = __reduce_max_sync(0xffffffffu, mx);
  }
}

// What a row's reduction says: 127 / m (0 for a row of zeros or of values that are no numbers), m, and
// the scale.
struct RowScale {
  float inv, m, scale;
  bool live;
};
__device__ __forceinline__ RowScale row_scale(uint32_t mx, float rstd) {
  RowScale s;
  s.m = __uint_as_float(mx);
  s.live = mx != 0 && mx < kInfBits;
  s.inv = s.live ? 127.0f / s.m : 0.f;
  s.scale = mx >= kInfBits ? __uint_as_float(0x7fc00000u) : s.m / 127.0f * rstd;
  return s;
}
// 1 / sqrt(ss / n + eps), where ss may be the sum of squares of values scaled by 2^-96.
__device__ __forceinline__ float inv_rms(float ss, int n, float eps) { return 1.0f / sqrtf(ss / (float)n + eps); }

// One row per warp (!BLOCK) or per block; each thread keeps NV vectors of VEC elements in registers.
template <typename T, bool NORM, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? kMaxThreads : 128) quant_rows_kernel(const RowArgs a) {
  const int warp = threadIdx.x >> 5;
  const int tid = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31);
  const int step = BLOCK ? (int)blockDim.x : 32;
  const long long row = BLOCK ? (long long)blockIdx.x : (long long)blockIdx.x * 4 + warp;
  if (row >= a.rows) return;                     // whole warps (whole blocks) only
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = NORM && a.r ? (const T*)a.r + row * a.ldr : nullptr;
  T* h = NORM && a.h ? (T*)a.h + row * a.ldh : nullptr;
  float t[NV][VEC];
  float hv[NORM ? NV : 1][VEC];
  float ss = 0.f;
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * step + tid) * VEC;
    if (at + VEC <= a.cols) {
      load_vec<T, VEC>(x + at, t[i]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) t[i][e] = at + e < a.cols ? to_f32(x[at + e]) : 0.f;
    }
  }
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (i * step + tid) * VEC;
      if (r) {
        float rv[VEC];
        if (at + VEC <= a.cols) {
          load_vec<T, VEC>(r + at, rv);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) rv[e] = at + e < a.cols ? to_f32(r[at + e]) : 0.f;
        }
        // h is the sum as it is stored; the norm reads it so, whether or not it is written out
        Pack<T, VEC> k;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          from_f32(t[i][e] + rv[e], &k.v[e]);
          t[i][e] = to_f32(k.v[e]);
        }
        if (h) {
          if (at + VEC <= a.cols) {
            *reinterpret_cast<Pack<T, VEC>*>(h + at) = k;
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (at + e < a.cols) h[at + e] = k.v[e];
          }
        }
      }
      float wv[VEC];
      if (at + VEC <= a.cols) {
        load_weight<VEC>(a.w, a.w_type, at, wv);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float one[1] = {0.f};
          if (at + e < a.cols) load_weight<1>(a.w, a.w_type, at + e, one);
          wv[e] = one[0];
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        hv[i][e] = t[i][e];
        ss = fmaf(t[i][e], t[i][e], ss);
        t[i][e] *= wv[e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) mx = max(mx, abs_bits(t[i][e]));
  reduce_row<BLOCK>(ss, mx);
  float rstd = 1.f;
  if constexpr (NORM) {
    rstd = inv_rms(ss, a.cols, a.eps);
    if (abs_bits(ss) >= kInfBits && mx < kInfBits) {   // finite values whose squares overflow: of h * 2^-96
      constexpr float kDown = 1.262177448353619e-29f;
      float s2 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s2 = fmaf(hv[i][e] * kDown, hv[i][e] * kDown, s2);
      uint32_t none = 0;
      reduce_row<BLOCK>(s2, none);
      rstd = inv_rms(s2, a.cols, 0.f) * kDown;
    }
  }
  const RowScale s = row_scale(mx, rstd);
  if (tid == 0) a.scale[row] = s.scale;
  int8_t* q = a.q + row * a.ldq;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * step + tid) * VEC;
    if (at >= a.cols) continue;
    Pack<int8_t, VEC> k;
#pragma unroll
    for (int e = 0; e < VEC; ++e) k.v[e] = (int8_t)(s.live ? round_i8(t[i][e], s.inv, s.m) : 0u);
    if (at + VEC <= a.cols) {
      *reinterpret_cast<Pack<int8_t, VEC>*>(q + at) = k;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (at + e < a.cols) q[at + e] = k.v[e];
    }
  }
}

// Rows longer than a block's registers hold: the row is walked once for the sums and once more to be
// rounded (its second reading comes from L2).  One block per row, one element per access.
template <typename T, bool NORM>
__global__ void __launch_bounds__(kMaxThreads) quant_long_rows_kernel(const RowArgs a) {
  const long long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = NORM && a.r ? (const T*)a.r + row * a.ldr : nullptr;
  T* h = NORM && a.h && a.r ? (T*)a.h + row * a.ldh : nullptr;
  // the value the norm reads at j; after the first walk h holds it (and may lie over x or r)
  auto value = [&](long long j, bool first) {
    if (!r) return to_f32(x[j]);
    if (h && !first) return to_f32(h[j]);
    T v;
    from_f32(to_f32(x[j]) + to_f32(r[j]), &v);
    if (h) h[j] = v;
    return to_f32(v);
  };
  auto weight = [&](long long j) {
    float w[1] = {1.f};
    if constexpr (NORM) load_weight<1>(a.w, a.w_type, j, w);
    return w[0];
  };
  float ss = 0.f;
  uint32_t mx = 0;
  for (long long j = threadIdx.x; j < a.cols; j += blockDim.x) {
    const float v = value(j, true);
    ss = fmaf(v, v, ss);
    mx = max(mx, abs_bits(v * weight(j)));
  }
  reduce_row<true>(ss, mx);
  float rstd = 1.f;
  if constexpr (NORM) {
    rstd = inv_rms(ss, a.cols, a.eps);
    if (abs_bits(ss) >= kInfBits && mx < kInfBits) {
      constexpr float kDown = 1.262177448353619e-29f;
      float s2 = 0.f;
      for (long long j = threadIdx.x; j < a.cols; j += blockDim.x) {
        const float v = value(j, false) * kDown;
        s2 = fmaf(v, v, s2);
      }
      uint32_t none = 0;
      reduce_row<true>(s2, none);
      rstd = inv_rms(s2, a.cols, 0.f) * kDown;
    }
  }
  const RowScale s = row_scale(mx, rstd);
  if (threadIdx.x == 0) a.scale[row] = s.scale;
  int8_t* q = a.q + row * a.ldq;
  for (long long j = threadIdx.x; j < a.cols; j += blockDim.x)
    q[j] = (int8_t)(s.live ? round_i8(value(j, false) * weight(j), s.inv, s.m) : 0u);
}

template <typename T, bool NORM, int VEC, int NV>
int LaunchRows(const RowArgs& a, int threads, cudaStream_t st) {
  if (threads == 32) quant_rows_kernel<T, NORM, VEC, NV, false><<<(a.rows + 3) / 4, 128, 0, st>>>(a);
  else quant_rows_kernel<T, NORM, VEC, NV, true><<<a.rows, threads, 0, st>>>(a);
  return 0;
}

template <typename T, bool NORM, int VEC>
int LaunchVec(const RowArgs& a, cudaStream_t st) {
  const int vecs = (a.cols + VEC - 1) / VEC;
  constexpr int kMost = 32 / VEC;                // 32 elements a thread
  if (vecs <= 32 * kMost) {
    if (vecs <= 8 * kMost) return LaunchRows<T, NORM, VEC, kMost / 4>(a, 32, st);
    return LaunchRows<T, NORM, VEC, kMost>(a, 32, st);
  }
  if (vecs <= kMaxThreads * kMost) return LaunchRows<T, NORM, VEC, kMost>(a, ((vecs + kMost - 1) / kMost + 31) / 32 * 32, st);
  quant_long_rows_kernel<T, NORM><<<a.rows, kMaxThreads, 0, st>>>(a);
  return 0;
}

template <typename T, bool NORM>
int LaunchT(const RowArgs& a, cudaStream_t st) {
  auto at16 = [](const void* p, long long ld) { return (uintptr_t)p % 16 == 0 && ld * (long long)sizeof(T) % 16 == 0; };
  const bool wide = at16(a.x, a.ldx) && (uintptr_t)a.q % 8 == 0 && a.ldq % 8 == 0 &&
                    (!NORM || ((!a.r || at16(a.r, a.ldr)) && (!a.h || at16(a.h, a.ldh)) && (uintptr_t)a.w % 16 == 0));
  return wide ? LaunchVec<T, NORM, 8>(a, st) : LaunchVec<T, NORM, 1>(a, st);
}

template <bool NORM>
int Launch(const RowArgs& a, int dtype, cudaStream_t st) {
  if (dtype == B200_DT_F32) LaunchT<float, NORM>(a, st);
  else if (dtype == B200_DT_BF16) LaunchT<__nv_bfloat16, NORM>(a, st);
  else LaunchT<__half, NORM>(a, st);
  CountLaunches();
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int ElementBytes(int dtype) { return dtype == B200_DT_F32 ? 4 : dtype == B200_DT_BF16 || dtype == B200_DT_F16 ? 2 : 0; }
bool Aligned(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }

}  // namespace

int QuantizeI8(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols, int dtype,
               cudaStream_t st) {
  const int es = ElementBytes(dtype);
  if (!es || rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX || ldx < cols || ldq < cols) return -1;
  if (rows == 0) return 0;
  if (!scale || !Aligned(scale, 4) || (cols && (!x || !q || !Aligned(x, es)))) return -1;
  RowArgs a = {};
  a.x = x;
  a.q = q;
  a.scale = scale;
  a.ldx = ldx;
  a.ldq = ldq;
  a.rows = (int)rows;
  a.cols = (int)cols;
  return Launch<false>(a, dtype, st);
}

int RmsNormI8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, void* h, int64_t ldh,
              int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols, int dtype, int weight_dtype, float eps,
              cudaStream_t st) {
  const int es = ElementBytes(dtype), ws = ElementBytes(weight_dtype);
  if (!es || !ws || rows < 0 || cols <= 0 || rows > INT32_MAX || cols > INT32_MAX || ldx < cols || ldq < cols) return -1;
  if (!(eps > 0.f) || eps > 3.4e38f || (residual && ldr < cols) || (h && ldh < cols) || (h && !residual)) return -1;
  if (rows == 0) return 0;
  if (!x || !q || !scale || !weight || !Aligned(scale, 4) || !Aligned(x, es) || !Aligned(weight, ws) ||
      (residual && !Aligned(residual, es)) || (h && !Aligned(h, es)))
    return -1;
  RowArgs a = {};
  a.x = x;
  a.r = residual;
  a.w = weight;
  a.h = h;
  a.q = q;
  a.scale = scale;
  a.ldx = ldx;
  a.ldr = ldr;
  a.ldh = ldh;
  a.ldq = ldq;
  a.rows = (int)rows;
  a.cols = (int)cols;
  a.w_type = weight_dtype == B200_DT_F32 ? 0 : weight_dtype == B200_DT_BF16 ? 1 : 2;
  a.eps = eps;
  return Launch<true>(a, dtype, st);
}

}  // namespace b200k

extern "C" int b200_quantize_i8(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols,
                                int dtype, void* stream) {
  return b200k::QuantizeI8(x, ldx, q, ldq, scale, rows, cols, dtype, (cudaStream_t)stream);
}

extern "C" int b200_rms_norm_i8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, void* h,
                                int64_t ldh, int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols, int dtype,
                                int weight_dtype, float eps, void* stream) {
  return b200k::RmsNormI8(x, ldx, residual, ldr, weight, h, ldh, q, ldq, scale, rows, cols, dtype, weight_dtype, eps,
                          (cudaStream_t)stream);
}
