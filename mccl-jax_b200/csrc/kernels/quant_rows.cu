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
// The maximum keeps a NaN, and across threads it is taken on the bit patterns of |t| as integers, which order
// like the values with infinity and NaN on top: a row that holds either is seen by the same reduction.
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
constexpr float kDown = 1.262177448353619e-29f;    // 2^-96
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
  float eps;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// x + r rounded to their type.  A 16-bit sum rounded at once is the f32 sum rounded: f32's 24 bits are at
// least two more than twice the 8 or 11 of the 16-bit types, where rounding twice changes nothing.
__device__ __forceinline__ float add_rn(float x, float r) { return x + r; }
__device__ __forceinline__ __nv_bfloat16 add_rn(__nv_bfloat16 x, __nv_bfloat16 r) { return __hadd_rn(x, r); }
__device__ __forceinline__ __half add_rn(__half x, __half r) { return __hadd_rn(x, r); }
__device__ __forceinline__ void add_rn2(float* x, const float* r) {
  x[0] += r[0];
  x[1] += r[1];
}
template <typename T2, typename T>
__device__ __forceinline__ void add_rn2_16(T* x, const T* r) {
  const T2 s = __hadd2_rn(T2{x[0], x[1]}, T2{r[0], r[1]});
  x[0] = s.x;
  x[1] = s.y;
}
__device__ __forceinline__ void add_rn2(__nv_bfloat16* x, const __nv_bfloat16* r) { add_rn2_16<__nv_bfloat162>(x, r); }
__device__ __forceinline__ void add_rn2(__half* x, const __half* r) { add_rn2_16<__half2>(x, r); }

// Two f32 operations in one instruction.
struct F2 {
  float x, y;
};
__device__ __forceinline__ uint64_t bits(F2 v) { return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ F2 floats(uint64_t b) { return {__uint_as_float((uint32_t)b), __uint_as_float((uint32_t)(b >> 32))}; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return floats(d);
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
  return floats(d);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return floats(d);
}
// The larger of m and |a|; NaN if either is.
__device__ __forceinline__ float max_abs(float m, float a) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(m), "f"(fabsf(a)));
  return d;
}

// VEC consecutive elements: one 4-, 8- or 16-byte access (two of 16 for eight f32).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Pack {
  T v[VEC];
};
// Elements at .. at + VEC - 1 of a row of `cols`, those past its end as `none`.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p, int at, int cols, T none) {
  Pack<T, VEC> k;
  if (VEC == 1 || at + VEC <= cols) {
    if (at < cols) k = *reinterpret_cast<const Pack<T, VEC>*>(p + at);
    else k.v[0] = none;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) k.v[e] = at + e < cols ? p[at + e] : none;
  }
  return k;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, int at, int cols, const Pack<T, VEC>& k) {
  if (at + VEC <= cols) {
    *reinterpret_cast<Pack<T, VEC>*>(p + at) = k;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (at + e < cols) p[at + e] = k.v[e];
  }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The few values next to a border, out of line: 127 t / m in 64 bits.
__device__ __noinline__ uint32_t round_exact(float t, float m) { return (uint32_t)__double2int_rn(127.0 * (double)t / (double)m); }

__device__ __forceinline__ uint32_t round_i8(float t, float inv, float m) {
  const float v = t * inv;
  const float s = v + kRoundMagic;
  // also taken where inv overflowed (m below 127 / FLT_MAX) and v is no number
  if (!(fabsf(v - (s - kRoundMagic)) < kBorder)) return round_exact(t, m);
  return __float_as_uint(s);
}

// round_half_even(127 t_i / m) of eight values, packed into 8 bytes; inv = 127 / m in f32, off where it is not
// finite (m below 127 / FLT_MAX).  One branch for the eight: 1.5 % of warps have a value next to a border.
__device__ __noinline__ uint2 round8_exact(F2 a, F2 b, F2 c, F2 d, float m) {
  const float t[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  uint32_t q[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i / 4] |= (round_exact(t[i], m) & 0xffu) << (8 * (i & 3));
  return make_uint2(q[0], q[1]);
}
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
__device__ __forceinline__ uint2 round8(const F2 (&t)[4], float inv, float m) {
  F2 s[4];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 v = mul2(t[i], {inv, inv});
    s[i] = add2(v, {kRoundMagic, kRoundMagic});
    const F2 k = add2(s[i], {-kRoundMagic, -kRoundMagic});
    const F2 d = fma2(k, {-1.f, -1.f}, v);
    far = max_abs(max_abs(far, d.x), d.y);       // NaN where inv is not finite
  }
  if (!(far < kBorder)) return round8_exact(t[0], t[1], t[2], t[3], m);
  return make_uint2(low_bytes(s[0].x, s[0].y, s[1].x, s[1].y), low_bytes(s[2].x, s[2].y, s[3].x, s[3].y));
}

// Sum and maximum over the threads of one row: the warp, or (BLOCK) the whole block.
template <bool BLOCK, bool SUM>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& mx) {
  if (SUM) {
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
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
    if (SUM) {
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
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

// One row per warp (!BLOCK) or per block; each thread keeps NV vectors of VEC elements in registers.  All
// loads of a row are issued before the first is used.
template <typename T, typename W, bool NORM, int VEC, int NV, bool BLOCK, int MAXT>
__global__ void __launch_bounds__(MAXT) quant_rows_kernel(const RowArgs a) {
  const int tid = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31);
  const int step = BLOCK ? (int)blockDim.x : 32;
  const long long row = BLOCK ? (long long)blockIdx.x : (long long)blockIdx.x * (MAXT / 32) + (threadIdx.x >> 5);
  if (row >= a.rows) return;                     // whole warps (whole blocks) only
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = NORM && a.r ? (const T*)a.r + row * a.ldr : nullptr;
  T* h = NORM && a.h ? (T*)a.h + row * a.ldh : nullptr;
  const W* w = (const W*)a.w;
  const T zero = T(0.f);
  const W wzero = W(0.f);
  Pack<T, VEC> xv[NV], rv[NORM ? NV : 1];
  Pack<W, VEC> wv[NORM ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) xv[i] = load_pack<T, VEC>(x, (i * step + tid) * VEC, a.cols, zero);
  if constexpr (NORM) {
    if (r) {
#pragma unroll
      for (int i = 0; i < NV; ++i) rv[i] = load_pack<T, VEC>(r, (i * step + tid) * VEC, a.cols, zero);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) wv[i] = load_pack<W, VEC>(w, (i * step + tid) * VEC, a.cols, wzero);
    if (r) {
      // h is the sum as it is stored; the norm reads it so, whether or not it is written out
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (VEC == 1) {
          xv[i].v[0] = add_rn(xv[i].v[0], rv[i].v[0]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) add_rn2(&xv[i].v[e], &rv[i].v[e]);
        }
        if (h) store_pack<T, VEC>(h, (i * step + tid) * VEC, a.cols, xv[i]);
      }
    }
  }
  // The thread's values in pairs, numbered through its vectors.  h stays in its own type and t = h w is formed
  // anew when it is rounded: fewer registers than t itself.
  auto h2 = [&](int p) { return F2{to_f32(xv[2 * p / VEC].v[2 * p % VEC]), to_f32(xv[(2 * p + 1) / VEC].v[(2 * p + 1) % VEC])}; };
  auto t2 = [&](int p) {
    if constexpr (NORM)
      return mul2(h2(p), F2{to_f32(wv[2 * p / VEC].v[2 * p % VEC]), to_f32(wv[(2 * p + 1) / VEC].v[(2 * p + 1) % VEC])});
    else
      return h2(p);
  };
  constexpr int kPairs = NV * VEC / 2;
  F2 ss2 = {0.f, 0.f};
  float mx = 0.f;
#pragma unroll
  for (int p = 0; p < kPairs; ++p) {
    if constexpr (NORM) {
      const F2 v = h2(p);
      ss2 = fma2(v, v, ss2);
    }
    const F2 t = t2(p);
    mx = max_abs(max_abs(mx, t.x), t.y);
  }
  float ss = ss2.x + ss2.y;
  uint32_t top = abs_bits(mx);
  reduce_row<BLOCK, NORM>(ss, top);
  float rstd = 1.f;
  if constexpr (NORM) {
    rstd = inv_rms(ss, a.cols, a.eps);
    if (abs_bits(ss) >= kInfBits && top < kInfBits) {  // finite values whose squares overflow: of h * 2^-96
      float s2 = 0.f;
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const F2 v = mul2(h2(p), {kDown, kDown});
        s2 = fmaf(v.x, v.x, fmaf(v.y, v.y, s2));
      }
      uint32_t none = 0;
      reduce_row<BLOCK, true>(s2, none);
      rstd = inv_rms(s2, a.cols, 0.f) * kDown;
    }
  }
  const RowScale s = row_scale(top, rstd);
  if (tid == 0) a.scale[row] = s.scale;
  int8_t* q = a.q + row * a.ldq;
#pragma unroll
  for (int g = 0; g < kPairs / 4; ++g) {         // eight values at a time: a vector, or eight of one element
    const int at = (VEC == 1 ? 8 * g * step + tid : (g * step + tid) * 8);
    if (at >= a.cols) continue;
    const F2 t[4] = {t2(4 * g), t2(4 * g + 1), t2(4 * g + 2), t2(4 * g + 3)};
    const uint2 k = s.live ? round8(t, s.inv, s.m) : make_uint2(0u, 0u);
    if constexpr (VEC == 8) {
      if (at + 8 <= a.cols) {
        *reinterpret_cast<uint2*>(q + at) = k;
        continue;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = at + (VEC == 1 ? e * step : e);
      if (j < a.cols) q[j] = (int8_t)((e < 4 ? k.x : k.y) >> (8 * (e & 3)));
    }
  }
}

// Rows longer than a block's registers hold: the row is walked once for the sums and once more to be
// rounded (its second reading comes from L2).  One block per row, one element per access.
template <typename T, typename W, bool NORM>
__global__ void __launch_bounds__(kMaxThreads) quant_long_rows_kernel(const RowArgs a) {
  const long long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = NORM && a.r ? (const T*)a.r + row * a.ldr : nullptr;
  T* h = NORM && a.h ? (T*)a.h + row * a.ldh : nullptr;
  const W* w = (const W*)a.w;
  // the value the norm reads at j; after the first walk h holds it (and may lie over x or r)
  auto value = [&](long long j, bool first) {
    if (!r) return to_f32(x[j]);
    if (h && !first) return to_f32(h[j]);
    const T v = add_rn(x[j], r[j]);
    if (h) h[j] = v;
    return to_f32(v);
  };
  auto t_of = [&](float v, long long j) {
    if constexpr (NORM) return v * to_f32(w[j]);
    else return v;
  };
  float ss = 0.f;
  uint32_t mx = 0;
  for (long long j = threadIdx.x; j < a.cols; j += blockDim.x) {
    const float v = value(j, true);
    ss = fmaf(v, v, ss);
    mx = max(mx, abs_bits(t_of(v, j)));
  }
  reduce_row<true, NORM>(ss, mx);
  float rstd = 1.f;
  if constexpr (NORM) {
    rstd = inv_rms(ss, a.cols, a.eps);
    if (abs_bits(ss) >= kInfBits && mx < kInfBits) {
      float s2 = 0.f;
      for (long long j = threadIdx.x; j < a.cols; j += blockDim.x) {
        const float v = value(j, false) * kDown;
        s2 = fmaf(v, v, s2);
      }
      uint32_t none = 0;
      reduce_row<true, true>(s2, none);
      rstd = inv_rms(s2, a.cols, 0.f) * kDown;
    }
  }
  const RowScale s = row_scale(mx, rstd);
  if (threadIdx.x == 0) a.scale[row] = s.scale;
  int8_t* q = a.q + row * a.ldq;
  for (long long j = threadIdx.x; j < a.cols; j += blockDim.x)
    q[j] = (int8_t)(s.live ? round_i8(t_of(value(j, false), j), s.inv, s.m) : 0u);
}

// The launch of a row: `threads` of them, 32 for a warp.
template <typename T, typename W, bool NORM, int VEC, int NV>
void LaunchBlock(const RowArgs& a, int vecs, cudaStream_t st) {
  const int threads = ((vecs + NV - 1) / NV + 31) / 32 * 32;
  if (threads <= 256) quant_rows_kernel<T, W, NORM, VEC, NV, true, 256><<<a.rows, threads, 0, st>>>(a);
  else quant_rows_kernel<T, W, NORM, VEC, NV, true, kMaxThreads><<<a.rows, threads, 0, st>>>(a);
}
template <typename T, typename W, bool NORM, int VEC, int NV>
void LaunchWarp(const RowArgs& a, cudaStream_t st) {
  quant_rows_kernel<T, W, NORM, VEC, NV, false, 128><<<(a.rows + 3) / 4, 128, 0, st>>>(a);
}

template <typename T, typename W, bool NORM>
void LaunchTW(const RowArgs& a, cudaStream_t st) {
  auto at16 = [](const void* p, long long ld) { return (uintptr_t)p % 16 == 0 && ld * (long long)sizeof(T) % 16 == 0; };
  const bool wide = at16(a.x, a.ldx) && (uintptr_t)a.q % 8 == 0 && a.ldq % 8 == 0 &&
                    (!NORM || ((!a.r || at16(a.r, a.ldr)) && (!a.h || at16(a.h, a.ldh)) && (uintptr_t)a.w % 16 == 0));
  const bool many = a.rows >= 148 * 8;
  if (wide) {
    const int vecs = (a.cols + 7) / 8;
    if (vecs <= 32 || (many && vecs <= 128)) {
      if (vecs <= 32) return LaunchWarp<T, W, NORM, 8, 1>(a, st);
      if (vecs <= 64) return LaunchWarp<T, W, NORM, 8, 2>(a, st);
      if (vecs <= 96) return LaunchWarp<T, W, NORM, 8, 3>(a, st);
      return LaunchWarp<T, W, NORM, 8, 4>(a, st);
    }
    if (vecs <= 256 || (!many && vecs <= kMaxThreads)) return LaunchBlock<T, W, NORM, 8, 1>(a, vecs, st);
    if (vecs <= 512) return LaunchBlock<T, W, NORM, 8, 2>(a, vecs, st);
    if (vecs <= 2 * kMaxThreads && (sizeof(T) == 4 || sizeof(W) == 4)) return LaunchBlock<T, W, NORM, 8, 2>(a, vecs, st);
    if (vecs <= 4 * kMaxThreads) return LaunchBlock<T, W, NORM, 8, 4>(a, vecs, st);
  } else {
    if (a.cols <= 256) return LaunchWarp<T, W, NORM, 1, 8>(a, st);
    if (a.cols <= 8 * kMaxThreads) return LaunchBlock<T, W, NORM, 1, 8>(a, a.cols, st);
    if (a.cols <= 32 * kMaxThreads) return LaunchBlock<T, W, NORM, 1, 32>(a, a.cols, st);
  }
  quant_long_rows_kernel<T, W, NORM><<<a.rows, kMaxThreads, 0, st>>>(a);
}

template <typename T, bool NORM>
void LaunchT(const RowArgs& a, int wtype, cudaStream_t st) {
  if constexpr (!NORM) LaunchTW<T, float, NORM>(a, st);
  else if (wtype == B200_DT_F32) LaunchTW<T, float, NORM>(a, st);
  else if (wtype == B200_DT_BF16) LaunchTW<T, __nv_bfloat16, NORM>(a, st);
  else LaunchTW<T, __half, NORM>(a, st);
}

template <bool NORM>
int Launch(const RowArgs& a, int dtype, int wtype, cudaStream_t st) {
  if (dtype == B200_DT_F32) LaunchT<float, NORM>(a, wtype, st);
  else if (dtype == B200_DT_BF16) LaunchT<__nv_bfloat16, NORM>(a, wtype, st);
  else LaunchT<__half, NORM>(a, wtype, st);
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
  return Launch<false>(a, dtype, 0, st);
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
  a.eps = eps;
  return Launch<true>(a, dtype, weight_dtype, st);
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
