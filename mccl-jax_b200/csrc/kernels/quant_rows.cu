// quant_rows.cu — rows rounded to 8 bits with a scale each: of values as they are, and of a root-mean-
// square norm with the residual's addition in front of it.
//
// With t_j = x_j (quantize) or t_j = f32(h_j w_j), h = round(x + r) (norm), and m = max_j |t_j|:
//     q_j = round_half_even(127 t_j / m),   scale = m / 127  [* 1 / sqrt(mean(h^2) + eps)]
// The norm's factor is the same for the whole row, so it cancels in q and enters the scale alone: a row
// needs one reduction of the pair (sum h^2, max |t|), after which every value is rounded from registers.
//
// q is the exact quotient's rounding, not that of f32 arithmetic: t * (127 / m) is off by less than 2^-14.9, so
// a value further than 2^-14 from a border between two integers is rounded right in f32, and the few others
// (1.2e-4 of them) are divided in 64 bits, where the quotient of two f32 values cannot cross or miss a border.
// The result then depends on no order of operations.
//
// The maximum keeps a NaN, and across threads it is taken on the bit patterns of |t| as integers, which order
// like the values with infinity and NaN on top: a row that holds either is seen by the same reduction.
//
// HBM bounds it: read and written once are 7 bytes an element for a bf16 norm with residual, 3 for bf16 rows.
// Measured on B200: norm [8192, 8192] bf16 84-87 us (5.4-5.6 TB/s), [8192, 8192] f32 133 us (6.6 TB/s), quantize
// [50257, 768] f32 31 us (6.2 TB/s), [16384, 4096] bf16 41 us (4.9 TB/s); one row of 768: 2 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "../../../include/b200_kernels.h"

namespace b200k {
namespace {

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kBorder = 0.5f - 1.0f / 16384.0f;
constexpr float kRoundMagic = 12582912.0f;     // 1.5 * 2^23: adding it rounds |v| < 2^22 to an integer
constexpr float kDown = 1.262177448353619e-29f;    // 2^-96
constexpr float kSmall = 1.5046327690525280e-36f;  // 2^-119, just above 127 * 2^-126
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
__device__ __forceinline__ uint64_t bits(F2 v) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(v.x), "f"(v.y));
  return d;
}
__device__ __forceinline__ F2 floats(uint64_t b) {
  F2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(b));
  return v;
}
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
// The largest of m, |a.x| and |a.y|; NaN if one of them is.
__device__ __forceinline__ float max_abs(float m, F2 a) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(fabsf(a.x)), "f"(fabsf(a.y)));
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

// Drops the first `bytes` of NW + EX words; the NW that follow remain.
template <int NW, int EX>
__device__ __forceinline__ void drop_bytes(uint32_t (&x)[NW + EX], int bytes) {
  if constexpr (EX == 4) {
#pragma unroll
    for (int i = 0; i < NW + 2; ++i) x[i] = bytes & 8 ? x[i + 2] : x[i];
  }
#pragma unroll
  for (int i = 0; i < NW + 1; ++i) x[i] = bytes & 4 ? x[i + 1] : x[i];
#pragma unroll
  for (int i = 0; i < NW; ++i) x[i] = __funnelshift_r(x[i], x[i + 1], 8 * (bytes & 3));
}

// The 16-byte lines that hold the eight neighbours p[j ..] of a row.  ALIGNED: they are those lines.  Else the
// lines are read whole (one that holds a byte of the row lies in the row's allocation) and shifted afterwards: two
// wide loads and some twenty integer operations in the place of eight narrow loads.  Nothing here reads what was
// loaded, so that the loads of all groups and arrays are in flight together.
template <typename T, bool ALIGNED>
struct Lines {
  static constexpr int kWords = 4 * kPairWords<T>, kLines = kWords / 4 + (ALIGNED ? 0 : 1);
  uint4 u[kLines];
  __device__ __forceinline__ void load(const T* p, int j, int cols) {
    const char* at = reinterpret_cast<const char*>(p + j);
    const char* end = reinterpret_cast<const char*>(p + cols);
    const char* line = ALIGNED ? at : at - ((uintptr_t)at & 15);
#pragma unroll
    for (int i = 0; i < kLines; ++i) {
      u[i] = make_uint4(0u, 0u, 0u, 0u);
      if ((unsigned)j < (unsigned)cols && line + 16 * i < end) u[i] = *reinterpret_cast<const uint4*>(line + 16 * i);
    }
  }
  // The eight elements; 0 past the row's end.
  __device__ __forceinline__ void take(const T* p, int j, int cols, Pair<T> (&v)[4]) const {
    uint32_t x[kWords + 4];
#pragma unroll
    for (int i = 0; i < kLines; ++i) {
      x[4 * i] = u[i].x;
      x[4 * i + 1] = u[i].y;
      x[4 * i + 2] = u[i].z;
      x[4 * i + 3] = u[i].w;
    }
    if constexpr (!ALIGNED) drop_bytes<kWords, 4>(x, (int)((uintptr_t)(p + j) & 15));
    if (j + 8 > cols) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {         // the word's elements past the end
        const int e = j + i * 4 / (int)sizeof(T);
        if (e >= cols) x[i] = 0;
        else if (sizeof(T) == 2 && e + 1 >= cols) x[i] &= 0xffffu;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < kPairWords<T>; ++k) v[i].w[k] = x[i * kPairWords<T> + k];
  }
};

// Eight neighbours to p[j ..], nothing past the row's end.  Else than ALIGNED, a lane writes the whole lines that
// begin with the last bytes of the group before it, which the lane before it holds; those at the row's ends are
// written element by element.  Every lane of the warp calls this; a lane that is `mute` only hands on its group.
template <typename E, int NW, bool ALIGNED>
__device__ __forceinline__ void store8(E* p, int j, int cols, const uint32_t (&w)[NW], bool mute) {
  constexpr int EX = NW < 4 ? NW : 4, kLine = 4 * EX;
  auto element = [&](const uint32_t* x, int e) {
    if constexpr (sizeof(E) == 4) return x[e];
    else if constexpr (sizeof(E) == 2) return (x[e / 2] >> (16 * (e & 1))) & 0xffffu;
    else return (x[e / 4] >> (8 * (e & 3))) & 0xffu;
  };
  auto put = [&](int at, uint32_t bits) {
    if constexpr (sizeof(E) == 4) reinterpret_cast<uint32_t*>(p)[at] = bits;
    else if constexpr (sizeof(E) == 2) reinterpret_cast<uint16_t*>(p)[at] = (uint16_t)bits;
    else reinterpret_cast<uint8_t*>(p)[at] = (uint8_t)bits;
  };
  auto whole = [&](int at, const uint32_t* x) {
#pragma unroll
    for (int i = 0; i < NW; i += EX) {
      if constexpr (EX == 4) reinterpret_cast<uint4*>(p + at)[i / 4] = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      else *reinterpret_cast<uint2*>(p + at) = make_uint2(x[0], x[1]);
    }
  };
  const int off = ALIGNED ? 0 : (int)((uintptr_t)(p + j) & (kLine - 1));   // the same for all lanes of a row
  uint32_t x[NW + EX];
#pragma unroll
  for (int i = 0; i < EX; ++i) x[i] = ALIGNED ? 0u : __shfl_up_sync(0xffffffffu, w[NW - EX + i], 1);
#pragma unroll
  for (int i = 0; i < NW; ++i) x[EX + i] = w[i];
  const int from = j - off / (int)sizeof(E);
  if (ALIGNED || off == 0) {
#pragma unroll
    for (int i = 0; i < NW; ++i) x[i] = w[i];
  } else {
    drop_bytes<NW, EX>(x, kLine - off);
  }
  if (mute) return;
  if (from >= 0 && from + 8 <= cols) {
    whole(from, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (from + e >= 0 && from + e < cols) put(from + e, element(x, e));
  }
}
template <typename T>
__device__ __forceinline__ void words_of(const Pair<T> (&v)[4], uint32_t (&w)[4 * kPairWords<T>]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < kPairWords<T>; ++k) w[i * kPairWords<T> + k] = v[i].w[k];
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The few values next to a border, out of line: 127 t / m in 64 bits.
__device__ __noinline__ uint32_t round_exact(float t, float m) { return (uint32_t)__double2int_rn(127.0 * (double)t / (double)m); }

// round_half_even(127 t / m), of which the low byte counts; inv as row_round gives it.
__device__ __forceinline__ uint32_t round_i8(float t, float inv, float m) {
  const float v = t * inv;
  const float s = v + kRoundMagic;
  if (!(fabsf(v - (s - kRoundMagic)) < kBorder)) return round_exact(t, m);
  return __float_as_uint(s);
}

// round_half_even(127 t_i / m) of eight values, packed into 8 bytes; inv as row_round gives it.  One
// branch for the eight: 3 % of warps have a value next to a border.
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
    far = max_abs(far, d);                       // NaN where inv is
  }
  if (!(far < kBorder)) return round8_exact(t[0], t[1], t[2], t[3], m);
  return make_uint2(low_bytes(s[0].x, s[0].y, s[1].x, s[1].y), low_bytes(s[2].x, s[2].y, s[3].x, s[3].y));
}

// Sum and maximum over the threads of one row: LANES of a warp, or (LANES 0) the whole block.
template <int LANES, bool SUM, int PLACE>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& mx) {
  constexpr int kIn = LANES ? LANES : 32;
#pragma unroll
  for (int o = kIn / 2; o; o >>= 1) {
    if (SUM) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (kIn < 32) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (kIn == 32) mx = __reduce_max_sync(0xffffffffu, mx);
  if constexpr (LANES == 0) {
    __shared__ float s_ss[32];                   // one set for each place that reduces
    __shared__ uint32_t s_mx[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) {
      s_ss[warp] = ss;
      s_mx[warp] = mx;
    }
    __syncthreads();
    ss = lane < warps ? s_ss[lane] : 0.f;
    mx = lane < warps ? s_mx[lane] : 0u;
    if (SUM) {
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
  }
}

// How a row whose largest |t| has the bits `mx` is rounded: 127 / m, or NaN for an m too small or too large for
// that to be exact enough (its values are then divided one by one).  The reciprocal is off by 2^-23, the products
// with 127 and with t by 2^-24 each: the quotient of at most 127 by less than 2^-14.9.
struct RowRound {
  float inv, m;
  bool live;                                     // not all zeros, and all numbers
};
__device__ __forceinline__ RowRound row_round(uint32_t mx) {
  RowRound s;
  s.m = __uint_as_float(mx);
  s.live = mx != 0 && mx < kInfBits;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s.m));
  s.inv = s.m > 1e-36f && s.m < 1e37f ? 127.0f * r : __uint_as_float(0x7fc00000u);
  return s;
}
// m / 127 [* 1 / sqrt(mean(h^2) + eps)]; ss is the sum of squares of down * h.
template <bool NORM>
__device__ __forceinline__ float row_scale(uint32_t mx, float ss, float down, int n, float eps) {
  if (mx >= kInfBits) return __uint_as_float(0x7fc00000u);
  const float m = __uint_as_float(mx);
  if (!NORM) return m / 127.0f;
  const float f = 1.0f / sqrtf(ss / (float)n + eps * down * down) * down;
  // an m / 127 below the normal range has lost bits that a large f would bring back into the scale
  return m < kSmall ? m * f / 127.0f : m / 127.0f * f;
}

// One row per LANES lanes of a warp, or (LANES 0) per block; each thread keeps NG groups of eight neighbours in
// registers.  All loads of a row are issued before the first is used.
//
// Rows that are not ALIGNED and take more than one warp's groups are dealt out to 31 lanes of a warp, and lane 0
// holds the group before them once more: the lines that two groups share are then written by one lane wherever
// they lie, and only a row's two ends are written element by element.
template <typename T, typename W, bool NORM, bool ALIGNED, int NG, int LANES, int MAXT>
__global__ void __launch_bounds__(MAXT, NORM && NG == 4 && MAXT == 256 ? 3 : 0) quant_rows_kernel(const RowArgs a) {
  constexpr int kLanes = LANES ? LANES : 32;
  const int tid = LANES ? (int)(threadIdx.x & (kLanes - 1)) : (int)threadIdx.x;
  const int step = LANES ? kLanes : (int)blockDim.x;
  const long long mine = LANES ? ((long long)blockIdx.x * MAXT + threadIdx.x) / kLanes : (long long)blockIdx.x;
  // lanes past the last row go with their warp: they hold zeros and write nothing
  const long long row = min(mine, (long long)a.rows - 1);
  const int cols = mine < a.rows ? a.cols : 0;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = NORM && a.r ? (const T*)a.r + row * a.ldr : nullptr;
  T* h = NORM && a.h ? (T*)a.h + row * a.ldh : nullptr;
  const W* w = (const W*)a.w;
  constexpr bool kTwice = !ALIGNED && (LANES == 0 || NG > 1);
  const bool again = kTwice && (threadIdx.x & 31) == 0;         // holds a group of the lane before it
  // the thread's g-th group begins here (before 0 or past the end: none)
  Pair<T> xv[NG][4];
  Pair<W> wv[NORM ? NG : 1][4];
  auto first = [&](int g) {
    if constexpr (!kTwice) return (g * step + tid) * 8;
    else return ((g * (step >> 5) + (tid >> 5)) * 31 + (tid & 31) - 1) * 8;
  };
  auto write_h = [&](int g) {
    uint32_t words[4 * kPairWords<T>];
    words_of(xv[g], words);
    store8<T, 4 * kPairWords<T>, ALIGNED>(h, first(g), cols, words, again);
  };
  Lines<T, ALIGNED> xl[NG], rl[NORM ? NG : 1];
  Lines<W, ALIGNED> wl[NORM ? NG : 1];
#pragma unroll
  for (int g = 0; g < NG; ++g) xl[g].load(x, first(g), cols);
  if constexpr (NORM) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      rl[g].load(r, first(g), r ? cols : 0);
      if (ALIGNED) wl[g].load(w, first(g), cols);
    }
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) xl[g].take(x, first(g), cols, xv[g]);
  if constexpr (NORM) {
    if (r) {
      // h is the sum as it is stored; the norm reads it so, whether or not it is written out
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        Pair<T> rv[4];
        rl[g].take(r, first(g), cols, rv);
#pragma unroll
        for (int p = 0; p < 4; ++p) xv[g][p] = add_rn2(xv[g][p], rv[p]);
        if (ALIGNED && h) write_h(g);
      }
    }
    // (lines that have to be shifted take twice the registers: the weights', which every row reads, come last)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (!ALIGNED) wl[g].load(w, first(g), cols);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) wl[g].take(w, first(g), cols, wv[g]);
  }
  F2 t[NG][4], ss2 = {0.f, 0.f};
  float mx = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      t[g][p] = unpack(xv[g][p]);
      if constexpr (NORM) {
        ss2 = fma2(t[g][p], t[g][p], ss2);
        t[g][p] = mul2(t[g][p], unpack(wv[g][p]));
      }
      mx = max_abs(mx, t[g][p]);
    }
  float ss = again ? 0.f : ss2.x + ss2.y;
  uint32_t top = abs_bits(mx);
  reduce_row<LANES, NORM, 0>(ss, top);
  if constexpr (NORM) {
    // Lanes write each other's elements here, and h may lie over x or r: after the reduction, which a thread
    // enters with its loads done.
    if (!ALIGNED && h) {
#pragma unroll
      for (int g = 0; g < NG; ++g) write_h(g);
    }
  }
  float down = 1.f;                              // what h was multiplied by for ss
  if constexpr (NORM) {
    // finite values whose squares overflow: of h * 2^-96 (the rows of a warp go there together)
    const bool over = abs_bits(ss) >= kInfBits && top < kInfBits;
    if (LANES == 0 ? over : __any_sync(0xffffffffu, over)) {
      float s2 = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const F2 v = mul2(unpack(xv[g][p]), {kDown, kDown});
          s2 = fmaf(v.x, v.x, fmaf(v.y, v.y, s2));
        }
      if (again) s2 = 0.f;
      uint32_t none = 0;
      reduce_row<LANES, true, 1>(s2, none);
      if (over) {
        ss = s2;
        down = kDown;
      }
    }
  }
  if (tid == 0 && mine < a.rows) a.scale[row] = row_scale<NORM>(top, ss, down, a.cols, a.eps);
  const RowRound s = row_round(top);
  int8_t* q = a.q + row * a.ldq;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint2 k = s.live ? round8(t[g], s.inv, s.m) : make_uint2(0u, 0u);
    const uint32_t words[2] = {k.x, k.y};
    store8<int8_t, 2, ALIGNED>(q, first(g), cols, words, again);
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
  // a thread's squares in 64 bits: thousands of them added one by one in 32 would all be rounded the same way
  double sum = 0.0;
  uint32_t mx = 0;
  for (long long j = threadIdx.x; j < a.cols; j += blockDim.x) {
    const float v = value(j, true);
    if constexpr (NORM) sum = fma((double)v, (double)v, sum);
    mx = max(mx, abs_bits(t_of(v, j)));
  }
  float ss = (float)sum;
  reduce_row<0, NORM, 0>(ss, mx);
  float down = 1.f;
  if constexpr (NORM) {
    if (abs_bits(ss) >= kInfBits && mx < kInfBits) {
      ss = (float)(sum * ((double)kDown * (double)kDown));
      uint32_t none = 0;
      reduce_row<0, true, 1>(ss, none);
      down = kDown;
    }
  }
  if (threadIdx.x == 0) a.scale[row] = row_scale<NORM>(mx, ss, down, a.cols, a.eps);
  const RowRound s = row_round(mx);
  int8_t* q = a.q + row * a.ldq;
  for (long long j = threadIdx.x; j < a.cols; j += blockDim.x)
    q[j] = (int8_t)(s.live ? round_i8(t_of(value(j, false), j), s.inv, s.m) : 0u);
}

// FROM and TO: the smallest and the largest block that the caller's rows come to.
template <typename T, typename W, bool NORM, bool ALIGNED, int NG, int FROM = 256, int TO = kMaxThreads>
void LaunchBlock(const RowArgs& a, int groups, cudaStream_t st) {
  // not aligned: 31 groups a warp, and a lane past the last group, which writes the end of its last line
  const int per = ALIGNED ? 32 * NG : 31 * NG, threads = ((groups + (ALIGNED ? 0 : 1) + per - 1) / per) * 32;
  if constexpr (FROM <= 256) {
    if (TO == 256 || threads <= 256) return quant_rows_kernel<T, W, NORM, ALIGNED, NG, 0, 256><<<a.rows, threads, 0, st>>>(a);
  }
  if constexpr (FROM <= 512 && TO >= 512) {
    if (TO == 512 || threads <= 512) return quant_rows_kernel<T, W, NORM, ALIGNED, NG, 0, 512><<<a.rows, threads, 0, st>>>(a);
  }
  if constexpr (TO > 512) quant_rows_kernel<T, W, NORM, ALIGNED, NG, 0, kMaxThreads><<<a.rows, threads, 0, st>>>(a);
}
template <typename T, typename W, bool NORM, bool ALIGNED, int NG, int LANES>
void LaunchWarp(const RowArgs& a, cudaStream_t st) {
  constexpr int kRows = 128 / LANES;
  quant_rows_kernel<T, W, NORM, ALIGNED, NG, LANES, 128><<<(unsigned)(((long long)a.rows + kRows - 1) / kRows), 128, 0, st>>>(a);
}

template <typename T, typename W, bool NORM, bool ALIGNED>
void LaunchTW(const RowArgs& a, cudaStream_t st) {
  const bool many = a.rows >= 148 * 8;
  const int groups = (int)((a.cols + 7ll) / 8);
  const int lanes = groups + (ALIGNED ? 0 : 1);  // see LaunchBlock
  if (lanes <= 8) return LaunchWarp<T, W, NORM, ALIGNED, 1, 8>(a, st);
  if (lanes <= 16) return LaunchWarp<T, W, NORM, ALIGNED, 1, 16>(a, st);
  if (lanes <= 32) return LaunchWarp<T, W, NORM, ALIGNED, 1, 32>(a, st);
  if constexpr (ALIGNED) {
    // Few rows: as many threads a row as it has groups (latency).  Many: more groups a thread, so that more bytes
    // are in flight for each reduction; norm rows, with three times the registers, best at two (bf16 16384 x 4096:
    // 103, 78, 87 us with 1, 2, 4 groups), quantised rows at four (62, 47, 41 us).
    if (!many && groups <= kMaxThreads) return LaunchBlock<T, W, NORM, true, 1>(a, groups, st);
    if (groups <= 64) return LaunchWarp<T, W, NORM, true, 2, 32>(a, st);
    if (groups <= 96) return LaunchWarp<T, W, NORM, true, 3, 32>(a, st);
    if constexpr (NORM && sizeof(T) + sizeof(W) == 4) {
      // (more than 512 groups of 16-bit values: four, in blocks of at most 256 threads, three to an SM; 8192 x 8192
      // bf16: 84 us, with two groups and 512 threads 93)
      if (groups <= 512) return LaunchBlock<T, W, true, true, 2, 256, 256>(a, groups, st);
      if (groups <= 1024) return LaunchBlock<T, W, true, true, 4, 256, 256>(a, groups, st);
      if (groups <= 2 * kMaxThreads) return LaunchBlock<T, W, true, true, 2, kMaxThreads>(a, groups, st);
      if (groups <= 4 * kMaxThreads) return LaunchBlock<T, W, true, true, 4, kMaxThreads>(a, groups, st);
    } else if constexpr (NORM) {
      if (groups <= 2 * kMaxThreads) return LaunchBlock<T, W, true, true, 2>(a, groups, st);
      if (groups <= 4 * kMaxThreads) return LaunchBlock<T, W, true, true, 4, kMaxThreads>(a, groups, st);
    } else {
      if (groups <= 128) return LaunchWarp<T, W, false, true, 4, 32>(a, st);
      if (groups <= 4 * kMaxThreads) return LaunchBlock<T, W, false, true, 4>(a, groups, st);
    }
  } else {
    // bf16 16384 x 4096 norm: 172 and 140 us with 1 and 2 groups; 8192 x 1003: 25 and 29 us
    if (groups <= 256 || (!(NORM && many) && lanes <= kMaxThreads / 32 * 31)) return LaunchBlock<T, W, NORM, false, 1>(a, groups, st);
    if (lanes <= kMaxThreads / 32 * 31 * 2) return LaunchBlock<T, W, NORM, false, 2, NORM ? 256 : kMaxThreads>(a, groups, st);
    if (lanes <= kMaxThreads / 32 * 31 * 4) return LaunchBlock<T, W, NORM, false, 4, kMaxThreads>(a, groups, st);
  }
  quant_long_rows_kernel<T, W, NORM><<<a.rows, kMaxThreads, 0, st>>>(a);
}
template <typename T, typename W, bool NORM>
void LaunchAligned(const RowArgs& a, cudaStream_t st) {
  auto at16 = [](const void* p, long long ld) { return (uintptr_t)p % 16 == 0 && ld * (long long)sizeof(T) % 16 == 0; };
  const bool aligned = at16(a.x, a.ldx) && (uintptr_t)a.q % 8 == 0 && a.ldq % 8 == 0 &&
                       (!NORM || ((!a.r || at16(a.r, a.ldr)) && (!a.h || at16(a.h, a.ldh)) && (uintptr_t)a.w % 16 == 0));
  if (aligned) LaunchTW<T, W, NORM, true>(a, st);
  else LaunchTW<T, W, NORM, false>(a, st);
}

template <typename T, bool NORM>
void LaunchT(const RowArgs& a, int wtype, cudaStream_t st) {
  if constexpr (!NORM) LaunchAligned<T, float, NORM>(a, st);
  else if (wtype == B200_DT_F32) LaunchAligned<T, float, NORM>(a, st);
  else if (wtype == B200_DT_BF16) LaunchAligned<T, __nv_bfloat16, NORM>(a, st);
  else LaunchAligned<T, __half, NORM>(a, st);
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
      (residual && !Aligned(residual, es)) || (h && !Aligned(h, es)) || (h && h == x && ldh != ldx) ||
      (h && h == residual && ldh != ldr))
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
