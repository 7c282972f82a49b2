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

// Two elements of a row in registers: one word for a 16-bit type, two for f32.  (Kept as words: arrays of 16-bit
// values cost the compiler several byte permutes an element.)
template <typename T>
constexpr int kPairWords = (int)sizeof(T) / 2;
template <typename T>
struct Pair {
  uint32_t w[kPairWords<T>];
};
__device__ __forceinline__ F2 unpack(Pair<float> p) { return {__uint_as_float(p.w[0]), __uint_as_float(p.w[1])}; }
__device__ __forceinline__ F2 unpack(Pair<__nv_bfloat16> p) {
  return {__uint_as_float(p.w[0] << 16), __uint_as_float(p.w[0] & 0xffff0000u)};
}
__device__ __forceinline__ F2 unpack(Pair<__half> p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p.w[0]));
  return {f.x, f.y};
}
__device__ __forceinline__ Pair<float> add_rn2(Pair<float> x, Pair<float> r) {
  const F2 s = add2(unpack(x), unpack(r));
  return {{__float_as_uint(s.x), __float_as_uint(s.y)}};
}
__device__ __forceinline__ Pair<__nv_bfloat16> add_rn2(Pair<__nv_bfloat16> x, Pair<__nv_bfloat16> r) {
  Pair<__nv_bfloat16> s;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(s.w[0]) : "r"(x.w[0]), "r"(r.w[0]));
  return s;
}
__device__ __forceinline__ Pair<__half> add_rn2(Pair<__half> x, Pair<__half> r) {
  Pair<__half> s;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(s.w[0]) : "r"(x.w[0]), "r"(r.w[0]));
  return s;
}

// The element at j, as bits; 0 past the row's end.
template <typename T>
__device__ __forceinline__ uint32_t element_bits(const T* p, int j, int cols) {
  if (j >= cols) return 0u;
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t*>(p + j);
  else return *reinterpret_cast<const uint16_t*>(p + j);
}
template <typename T>
__device__ __forceinline__ Pair<T> make_pair(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4) return {{a, b}};
  else return {{a | b << 16}};
}
// Eight elements at j, j + stride, ...: stride 1 is one 16-byte access (two for f32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int j, int stride, int cols, Pair<T> (&v)[4]) {
  if (stride == 1 && j + 8 <= cols) {
    uint4 u[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p + j)[i];
    const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < kPairWords<T>; ++k) v[i].w[k] = w[i * kPairWords<T> + k];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = make_pair<T>(element_bits(p, j + 2 * i * stride, cols), element_bits(p, j + (2 * i + 1) * stride, cols));
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int j, int stride, int cols, const Pair<T> (&v)[4]) {
  uint32_t w[4 * kPairWords<T>];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < kPairWords<T>; ++k) w[i * kPairWords<T> + k] = v[i].w[k];
  if (stride == 1 && j + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(p + j)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = j + e * stride;
      if (at >= cols) continue;
      if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[at] = w[e];
      else reinterpret_cast<uint16_t*>(p)[at] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
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

// One row per warp (!BLOCK) or per block; each thread keeps NG groups of eight values in registers: eight
// neighbours (WIDE), or eight a row of threads apart, where addresses allow no wide access.  All loads of a row
// are issued before the first is used.
template <typename T, typename W, bool NORM, bool WIDE, int NG, bool BLOCK, int MAXT>
__global__ void __launch_bounds__(MAXT) quant_rows_kernel(const RowArgs a) {
  const int tid = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31);
  const int step = BLOCK ? (int)blockDim.x : 32, stride = WIDE ? 1 : step;
  const long long row = BLOCK ? (long long)blockIdx.x : (long long)blockIdx.x * (MAXT / 32) + (threadIdx.x >> 5);
  if (row >= a.rows) return;                     // whole warps (whole blocks) only
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = NORM && a.r ? (const T*)a.r + row * a.ldr : nullptr;
  T* h = NORM && a.h ? (T*)a.h + row * a.ldh : nullptr;
  const W* w = (const W*)a.w;
  auto first = [&](int g) { return WIDE ? (g * step + tid) * 8 : 8 * g * step + tid; };   // of group g
  Pair<T> xv[NG][4], rv[NORM ? NG : 1][4];
  Pair<W> wv[NORM ? NG : 1][4];
#pragma unroll
  for (int g = 0; g < NG; ++g) load8(x, first(g), stride, a.cols, xv[g]);
  if constexpr (NORM) {
    if (r) {
#pragma unroll
      for (int g = 0; g < NG; ++g) load8(r, first(g), stride, a.cols, rv[g]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) load8(w, first(g), stride, a.cols, wv[g]);
    if (r) {
      // h is the sum as it is stored; the norm reads it so, whether or not it is written out
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int p = 0; p < 4; ++p) xv[g][p] = add_rn2(xv[g][p], rv[g][p]);
        if (h) store8(h, first(g), stride, a.cols, xv[g]);
      }
    }
  }
  // h stays in its own type and t = h w is formed anew when it is rounded: fewer registers than t itself
  auto t_of = [&](int g, int p) {
    if constexpr (NORM) return mul2(unpack(xv[g][p]), unpack(wv[g][p]));
    else return unpack(xv[g][p]);
  };
  F2 ss2 = {0.f, 0.f};
  float mx = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if constexpr (NORM) {
        const F2 v = unpack(xv[g][p]);
        ss2 = fma2(v, v, ss2);
      }
      const F2 t = t_of(g, p);
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
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const F2 v = mul2(unpack(xv[g][p]), {kDown, kDown});
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
  for (int g = 0; g < NG; ++g) {
    const int at = first(g);
    if (at >= a.cols) continue;
    const F2 t[4] = {t_of(g, 0), t_of(g, 1), t_of(g, 2), t_of(g, 3)};
    const uint2 k = s.live ? round8(t, s.inv, s.m) : make_uint2(0u, 0u);
    if (WIDE && at + 8 <= a.cols) {
      *reinterpret_cast<uint2*>(q + at) = k;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = at + e * stride;
        if (j < a.cols) q[j] = (int8_t)((e < 4 ? k.x : k.y) >> (8 * (e & 3)));
      }
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
template <typename T, typename W, bool NORM, bool WIDE, int NG>
void LaunchBlock(const RowArgs& a, int groups, cudaStream_t st) {
  const int threads = ((groups + NG - 1) / NG + 31) / 32 * 32;
  if (threads <= 256) quant_rows_kernel<T, W, NORM, WIDE, NG, true, 256><<<a.rows, threads, 0, st>>>(a);
  else quant_rows_kernel<T, W, NORM, WIDE, NG, true, kMaxThreads><<<a.rows, threads, 0, st>>>(a);
}
template <typename T, typename W, bool NORM, bool WIDE, int NG>
void LaunchWarp(const RowArgs& a, cudaStream_t st) {
  quant_rows_kernel<T, W, NORM, WIDE, NG, false, 128><<<(a.rows + 3) / 4, 128, 0, st>>>(a);
}

template <typename T, typename W, bool NORM>
void LaunchTW(const RowArgs& a, cudaStream_t st) {
  auto at16 = [](const void* p, long long ld) { return (uintptr_t)p % 16 == 0 && ld * (long long)sizeof(T) % 16 == 0; };
  const bool wide = at16(a.x, a.ldx) && (uintptr_t)a.q % 8 == 0 && a.ldq % 8 == 0 &&
                    (!NORM || ((!a.r || at16(a.r, a.ldr)) && (!a.h || at16(a.h, a.ldh)) && (uintptr_t)a.w % 16 == 0));
  const bool many = a.rows >= 148 * 8;
  const int groups = (a.cols + 7) / 8;
  if (wide) {
    if (groups <= 32 || (many && groups <= 128)) {
      if (groups <= 32) return LaunchWarp<T, W, NORM, true, 1>(a, st);
      if (groups <= 64) return LaunchWarp<T, W, NORM, true, 2>(a, st);
      if (groups <= 96) return LaunchWarp<T, W, NORM, true, 3>(a, st);
      return LaunchWarp<T, W, NORM, true, 4>(a, st);
    }
    if (groups <= 256 || (!many && groups <= kMaxThreads)) return LaunchBlock<T, W, NORM, true, 1>(a, groups, st);
    if (groups <= 512) return LaunchBlock<T, W, NORM, true, 2>(a, groups, st);
    if (groups <= 2 * kMaxThreads && (sizeof(T) == 4 || sizeof(W) == 4)) return LaunchBlock<T, W, NORM, true, 2>(a, groups, st);
    if (groups <= 4 * kMaxThreads) return LaunchBlock<T, W, NORM, true, 4>(a, groups, st);
  } else {
    if (groups <= 32) return LaunchWarp<T, W, NORM, false, 1>(a, st);
    if (groups <= kMaxThreads) return LaunchBlock<T, W, NORM, false, 1>(a, groups, st);
    if (groups <= 4 * kMaxThreads) return LaunchBlock<T, W, NORM, false, 4>(a, groups, st);
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
