// Rows to 8-bit operands of the scaled matmul, for sm_100a: e4m3 codes and one e8m0 scale (a power of
// two in one byte, biased by 127) per 128 consecutive columns of a row. Two kernels:
//   cake_quantize_rows_sm100      v = x, or silu(gate) * up of a [gate | up] row
//   cake_rms_norm_quantize_sm100  h = x + residual, v = h / sqrt(mean(h^2) + eps) * weight
// The scale of a group is the least power of two s >= 2^-127 with max |v| <= 448 s (448 is e4m3's largest
// value, so nothing saturates); 1 where the group is all zeros; NaN, with NaN codes throughout, where the
// group holds an infinity or a NaN. v / s is exact but for values more than 2^22 below the group's
// largest, which are far below half of e4m3's smallest step: the rounding to e4m3 (nearest even) is the
// only one after v, whose arithmetic is in 32 bits.
//
// Both kernels are one pass over HBM, every byte read and written once. What stands between them and its rate
// is instructions, so: a group is 8 lanes of 16 elements (three shuffles for its maximum, and the scale's
// arithmetic once per 16 elements); the maximum of 16-bit types is taken on their packed bits; f32 arithmetic
// goes in pairs; whole vectors are loaded and stored without looking at their elements.
//
// Measured (device time, HBM at 6.54 TB/s by a plain copy): quantise 16384 x 8192 bf16 59 us (6.8 TB/s; 86 us with
// 16 lanes a group, 93 registers and scalar maxima); gated 4001 x 11008 f16 33 us (6.6 TB/s; 72 us with
// expf and a division); norm with residual 8192 x 8192 bf16 71 us (6.6 TB/s; 103 us at 117 registers, two
// blocks an SM). One row of 8192: 3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cake_host.h"
#include "cake_ptx.cuh"

namespace cake {
namespace {

constexpr int kGroup = 128;  // columns that share a scale
constexpr int kVec = 8;      // elements of a vector: one or two 16-byte loads
constexpr int kGroupLanes = 8;
constexpr int kLaneVecs = 2;  // vectors of a lane in its group, 64 elements apart: a warp's loads stay contiguous
constexpr int kQuantThreads = 256;

// ------------------------------------------------------------------------------ pairs of f32

struct F2 {
  uint64_t v;  // low word first
};

__device__ __forceinline__ F2 pack2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// ------------------------------------------------------------------------------ vectors

// Eight elements as they lie in memory: four 32-bit words of a 16-bit type, eight of f32.
template <typename T>
struct Raw {
  static constexpr int kWords = kVec * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
};

// The vector at `ptr`, aligned to its elements only; elements from `valid` on are zero. The 16-byte pieces that
// hold a valid element are loaded whole (such a piece is in the same page as that element) and the bytes
// shifted into place, which costs two operations an element; loading them one by one took four times as long.
template <typename T>
__device__ __forceinline__ void load_shifted(Raw<T>& r, const T* ptr, int valid) {
  constexpr int kPieces = Raw<T>::kWords / 4 + 1;
  const uintptr_t address = reinterpret_cast<uintptr_t>(ptr);
  const int offset = static_cast<int>(address & 15);
  const uint4* piece = reinterpret_cast<const uint4*>(address & ~static_cast<uintptr_t>(15));
  const int end = valid > 0 ? offset + valid * static_cast<int>(sizeof(T)) : 0;
  uint32_t w[4 * kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (16 * i < end) v = piece[i];
    w[4 * i] = v.x;
    w[4 * i + 1] = v.y;
    w[4 * i + 2] = v.z;
    w[4 * i + 3] = v.w;
  }
#pragma unroll
  for (int i = 0; i + 2 < 4 * kPieces; ++i) w[i] = offset & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i + 3 < 4 * kPieces; ++i) w[i] = offset & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; ++i) r.w[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], (offset & 2) * 8) : w[i];
  if (valid < kVec) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; ++i) {
      constexpr int kPer = 4 / static_cast<int>(sizeof(T));  // elements of a word
      const int left = valid - kPer * i;
      r.w[i] &= left >= kPer ? 0xFFFFFFFFu : left == 1 && kPer == 2 ? 0xFFFFu : 0u;
    }
  }
}

// VEC: vectors are 16-byte aligned, and all or none of their elements valid.
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(Raw<T>& r, const T* ptr, int valid) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; i += 4) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (valid > 0) v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(ptr) + i);
      r.w[i] = v.x;
      r.w[i + 1] = v.y;
      r.w[i + 2] = v.z;
      r.w[i + 3] = v.w;
    }
  } else {
    load_shifted(r, ptr, valid);
  }
}

// The norm's loads: an aligned whole vector is looked for first, as its weights' are always and its rows' often
// (3000 x 5001 in rows of 5008: 46 -> 35 us; 8192 x 8192 in rows of 8321: 125 -> 113 us). The quantiser, which
// has four groups' loads in flight, loses by the branch (44 -> 48 us).
template <typename T, bool VEC>
__device__ __forceinline__ void load_norm(Raw<T>& r, const T* ptr, int valid) {
  if (VEC || (valid >= kVec && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0)) load_raw<T, true>(r, ptr, valid);
  else load_shifted(r, ptr, valid);
}

template <typename T>
__device__ __forceinline__ F2 widen(const Raw<T>& r, int pair);
template <>
__device__ __forceinline__ F2 widen<float>(const Raw<float>& r, int pair) {
  return pack2(__uint_as_float(r.w[2 * pair]), __uint_as_float(r.w[2 * pair + 1]));
}
template <>
__device__ __forceinline__ F2 widen<__nv_bfloat16>(const Raw<__nv_bfloat16>& r, int pair) {
  return pack2(__uint_as_float(r.w[pair] << 16), __uint_as_float(r.w[pair] & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ F2 widen<__half>(const Raw<__half>& r, int pair) {
  __half2 h;
  memcpy(&h, &r.w[pair], 4);
  const float2 f = __half22float2(h);
  return pack2(f.x, f.y);
}

__device__ __forceinline__ void narrow(uint32_t* w, int pair, F2 v, float) {
  float lo, hi;
  unpack2(v, lo, hi);
  w[2 * pair] = __float_as_uint(lo);
  w[2 * pair + 1] = __float_as_uint(hi);
}
__device__ __forceinline__ void narrow(uint32_t* w, int pair, F2 v, __nv_bfloat16) {
  float lo, hi;
  unpack2(v, lo, hi);
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  memcpy(&w[pair], &b, 4);
}
__device__ __forceinline__ void narrow(uint32_t* w, int pair, F2 v, __half) {
  float lo, hi;
  unpack2(v, lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  memcpy(&w[pair], &h, 4);
}

// Rounds four pairs to T and stores elements [0, valid).
template <typename T, bool VEC>
__device__ __forceinline__ void store_as(T* ptr, const F2* v, int valid) {
  uint32_t w[Raw<T>::kWords];
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) narrow(w, i, v[i], T());
  if (VEC ? valid > 0 : valid >= kVec && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; i += 4)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(ptr) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else if (!VEC) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (i < valid) {
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(ptr)[i] = w[i];
        else reinterpret_cast<uint16_t*>(ptr)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
      }
    }
  }
}

// ------------------------------------------------------------------------------ scale and codes

// Magnitudes are compared as integers: that order is the magnitudes' own, with every NaN above infinity,
// so a NaN is never lost as it would be by a floating-point maximum. The same holds for the 16-bit types,
// two at a time.
// (f32 values in registers go through the hardware's NaN-keeping maximum of magnitudes, three at a time.)
__device__ __forceinline__ float largest_abs(float a, F2 v) {
  float lo, hi, r;
  unpack2(v, lo, hi);
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(lo), "f"(hi));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t largest_raw(uint32_t a, const Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < Raw<T>::kWords; ++i) {
    if (sizeof(T) == 4) a = max(a, r.w[i] & 0x7FFFFFFFu);
    else a = __vmaxu2(a, r.w[i] & 0x7FFF7FFFu);
  }
  return a;
}

__device__ __forceinline__ uint32_t group_max(uint32_t a) {
#pragma unroll
  for (int d = kGroupLanes / 2; d > 0; d >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, d));
  return a;
}

// The group's largest magnitude as f32 bits, from the lanes' largest_raw.
template <typename T>
__device__ __forceinline__ uint32_t group_max_raw(uint32_t a);
template <>
__device__ __forceinline__ uint32_t group_max_raw<float>(uint32_t a) { return group_max(a); }
__device__ __forceinline__ uint32_t group_max_packed(uint32_t a) {
#pragma unroll
  for (int d = kGroupLanes / 2; d > 0; d >>= 1) a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, d));
  return max(a & 0xFFFFu, a >> 16);
}
template <>
__device__ __forceinline__ uint32_t group_max_raw<__nv_bfloat16>(uint32_t a) { return group_max_packed(a) << 16; }
template <>
__device__ __forceinline__ uint32_t group_max_raw<__half>(uint32_t a) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(group_max_packed(a)))));
}

// Scale byte of a group whose largest magnitude has the bits `a`. With a = 1.m * 2^(E - 127) and
// 448 = 1.75 * 2^8 the exponent is E - 127 - 8, one more where 1.m > 1.75, which is what adding 2 - 1.75 =
// 0x200000 less one to the bits carries over.
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
  const int e = max(static_cast<int>((a + 0x1FFFFFu) >> 23) - 8, 0);
  return a >= 0x7F800000u ? 255u : a == 0 ? 127u : static_cast<uint32_t>(e);
}

// 2^(127 - byte): a normal number, for bytes up to 247; NaN for byte 255, which makes every code NaN.
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7FC00000u : (254u - byte) << 23); }

// Four values to codes, rounded to nearest even.
__device__ __forceinline__ uint32_t to_codes(F2 a, F2 b) {
  float a0, a1, b0, b1;
  unpack2(a, a0, a1);
  unpack2(b, b0, b1);
  uint32_t r;
  asm("{\n\t"
      ".reg .b16 l, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h};\n\t"
      "}"
      : "=r"(r)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
  return r;
}

// Stores a vector's codes [0, valid); VEC: as one 8-byte store.
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* ptr, const F2* v, F2 inverse, int valid) {
  const uint32_t lo = to_codes(mul2(v[0], inverse), mul2(v[1], inverse)), hi = to_codes(mul2(v[2], inverse), mul2(v[3], inverse));
  if (VEC ? valid > 0 : valid >= kVec && (reinterpret_cast<uintptr_t>(ptr) & 7) == 0) {
    *reinterpret_cast<uint2*>(ptr) = make_uint2(lo, hi);
  } else if (!VEC) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i < valid) ptr[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

// Elements of the vector at `col` that a row of `cols` has. VEC: all or none.
template <bool VEC>
__device__ __forceinline__ int valid_at(int col, int cols) {
  if (VEC) return col < cols ? kVec : 0;
  return min(max(cols - col, 0), kVec);
}

// ------------------------------------------------------------------------------ quantise

// Division by a number known at launch, for dividends below 2^31: multiply, shift.
struct FastDivisor {
  uint32_t d, magic, shift;
};

__device__ __forceinline__ uint32_t divide(uint32_t n, const FastDivisor& f) { return (__umulhi(n, f.magic) + n) >> f.shift; }

FastDivisor fast_divisor(uint32_t d) {
  FastDivisor f;
  f.d = d;
  f.shift = 0;
  while ((1ull << f.shift) < d) ++f.shift;
  f.magic = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
  return f;
}

struct QuantizeParams {
  const void* x;
  uint8_t* q;
  uint8_t* scales;
  uint32_t x_stride, q_stride, scales_stride;  // elements (bytes) between rows
  uint32_t items;  // rows * groups, below 2^31
  int32_t cols;
  FastDivisor by_groups;
};

// silu(x) = x / (1 + exp(-x)) with exp(-x) = 2^-(p + l), p the product x log2(e) rounded down and l >= 0 what
// that lost: 2^-l = 1 - l ln(2) to the last bit, so that far from zero the exponent's rounding does not show.
// Where exp(-x) is 2^126 or more (x below -87.3) the result is -0: the estimates' forms without subnormals are
// four instructions shorter each. Relative error below 9 * 2^-24: the
// estimate of 2^-p 4, its correction 1, the sum 1, the estimate of its reciprocal 2, the product 1. No
// comparison or selection: the integer pipe is what bounds the gated kernel.
__device__ __forceinline__ float silu(float x) {
  constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596303e-8f;  // their sum is log2(e) to 2^-49
  constexpr float kLn2 = 0.693147182f;
  const float p = __fmul_rd(x, kLog2e);
  float lost, e, y;
  // Saturating: no more than a guard for x log2(e) beyond f32, where p and the difference are not numbers.
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(lost) : "f"(x), "f"(kLog2e), "f"(-p));
  const float correction = fmaf(x, -kLog2eRest * kLn2, fmaf(lost, -kLn2, 1.f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-p));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(e, correction, 1.f)));
  return x * y;
}

// A lane takes UNROLL groups that are 32 apart, so that a block's groups lie next to each other and every
// lane has that many groups' loads in flight.
template <typename T, bool GATE, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) cake_quantize_rows_sm100(const __grid_constant__ QuantizeParams p) {
  constexpr int kUnroll = (sizeof(T) == 4 || GATE) ? 2 : 4;
  constexpr int kApart = kQuantThreads / kGroupLanes;
  grid_dependency_wait();
  grid_dependency_trigger();
  const int lane = threadIdx.x % kGroupLanes;
  const uint32_t first = blockIdx.x * (kUnroll * kApart) + threadIdx.x / kGroupLanes;
  uint32_t row[kUnroll];
  int col[kUnroll];
  bool live[kUnroll];
  Raw<T> x[kUnroll][kLaneVecs], up[GATE ? kUnroll : 1][kLaneVecs];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t item = first + u * kApart;  // at most 127 past the last: a row that only live items use
    live[u] = item < p.items;
    uint32_t group;
    row[u] = divide(item, p.by_groups);
    group = item - row[u] * p.by_groups.d;
    col[u] = static_cast<int>(group) * kGroup + lane * kVec;
    const T* src = static_cast<const T*>(p.x) + static_cast<uint64_t>(row[u]) * p.x_stride + col[u];
#pragma unroll
    for (int v = 0; v < kLaneVecs; ++v) {
      // Items past the end load and store nothing.
      const int valid = live[u] ? valid_at<VEC>(col[u] + v * kGroupLanes * kVec, p.cols) : 0;
      load_raw<T, VEC>(x[u][v], src + v * kGroupLanes * kVec, valid);
      if (GATE) load_raw<T, VEC>(up[GATE ? u : 0][v], src + p.cols + v * kGroupLanes * kVec, valid);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    F2 v[kLaneVecs][kVec / 2];
    uint32_t a = 0;
    if (GATE) {
      float magnitude = 0.f;
#pragma unroll
      for (int k = 0; k < kLaneVecs; ++k)
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
          float x0, x1, u0, u1;
          unpack2(widen<T>(x[u][k], i), x0, x1);
          unpack2(widen<T>(up[GATE ? u : 0][k], i), u0, u1);
          x0 = silu(x0) * u0;
          x1 = silu(x1) * u1;
          v[k][i] = pack2(x0, x1);
          magnitude = largest_abs(magnitude, v[k][i]);
        }
      a = group_max(__float_as_uint(magnitude));
    } else {
#pragma unroll
      for (int k = 0; k < kLaneVecs; ++k) a = largest_raw<T>(a, x[u][k]);
      a = group_max_raw<T>(a);
#pragma unroll
      for (int k = 0; k < kLaneVecs; ++k)
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) v[k][i] = widen<T>(x[u][k], i);
    }
    const uint32_t byte = scale_byte(a);
    const float inverse = inverse_scale(byte);
    uint8_t* dst = p.q + static_cast<uint64_t>(row[u]) * p.q_stride + col[u];
#pragma unroll
    for (int k = 0; k < kLaneVecs; ++k) {
      const int at = k * kGroupLanes * kVec;
      store_codes<VEC>(dst + at, v[k], pack2(inverse, inverse), live[u] ? valid_at<VEC>(col[u] + at, p.cols) : 0);
    }
    if (lane == 0 && live[u]) p.scales[static_cast<uint64_t>(row[u]) * p.scales_stride + col[u] / kGroup] = static_cast<uint8_t>(byte);
  }
}

// ------------------------------------------------------------------------------ norm

struct NormParams {
  const void* x;
  const void* residual;  // or null
  void* residual_out;    // with a residual only
  const void* weight;
  uint8_t* q;
  uint8_t* scales;
  uint32_t x_stride, residual_stride, residual_out_stride, q_stride, scales_stride;
  uint32_t rows;
  int32_t cols;
  float epsilon;
  double inverse_cols;
};

// 1 / sqrt(a) as the sum of two f32: the hardware's estimate and one Newton-Raphson step in double. A value next to the border
// of two codes goes to the wrong one by any error of the scale, and the whole row has the scale's; one step
// in double costs six operations a thread. Zero and infinity pass through (their step is not a number).
__device__ __forceinline__ void inverse_root(double a, float& hi, float& lo) {
  const float y = rsqrtf(static_cast<float>(a));
  hi = y;
  lo = 0.f;
  if (y > 0.f && y < __int_as_float(0x7F800000)) {
    const double z = y, root = z + 0.5 * z * fma(-a * z, z, 1.0);
    hi = static_cast<float>(root);
    lo = static_cast<float>(root - hi);
  }
}

// h (hi + lo) w with one rounding: the first product's own error, from a fused multiply-add, and what lo adds
// go into the second.
__device__ __forceinline__ F2 scaled(F2 h, F2 hi, F2 minus_hi, F2 lo, F2 w) {
  const F2 product = mul2(h, hi);
  const F2 rest = fma2(h, lo, fma2(h, hi, mul2(h, minus_hi)));
  return fma2(product, w, mul2(rest, w));
}

// THREADS threads hold one row in registers, UNITS units of 16 elements each (unit i * THREADS + t of the row:
// eight units are a group), so the sum x + residual is normalised as it is in 32 bits while its rounding is
// stored, and the stored sum may lie over x or over the residual. Without a residual there is little to load
// for a row's chain of load, reduction, weights and store, so what counts then is that chain's length and how
// many rows an SM has under way: THREADS follows the row closely, few registers, weights loaded
// before the reduction where there is room for them, and the reduction itself short (f32 shuffles in a warp, two
// to five steps between warps): 8192 x 5120 bf16 45 -> 29 us, 8192 x 2048 24 -> 15 us.
__host__ __device__ constexpr int norm_rows(int threads) { return threads <= 128 ? 256 / threads : 1; }  // rows of a block

__host__ __device__ constexpr int first_step(int v) {  // the first step of a reduction over v lanes
  int d = 1;
  while (2 * d < v) d *= 2;
  return d;
}

template <typename T, typename W, int THREADS, int UNITS, bool VEC>
__global__ void __launch_bounds__(THREADS* norm_rows(THREADS)) cake_rms_norm_quantize_sm100(const __grid_constant__ NormParams p) {
  constexpr int kRows = norm_rows(THREADS);
  constexpr int kWarps = THREADS / 32;  // warps of a row
  constexpr bool kEarlyWeights = UNITS == 1;
  __shared__ float partial[kRows][kWarps];
  grid_dependency_wait();
  grid_dependency_trigger();
  const int t = threadIdx.x % THREADS;
  const int r = threadIdx.x / THREADS;
  const uint32_t row = blockIdx.x * kRows + r;
  const bool live = row < p.rows;
  // Column of unit i's first vector; the second is 64 further on.
  auto col_of = [&](int i) { return ((i * THREADS + t) / kGroupLanes) * kGroup + (t % kGroupLanes) * kVec; };
  F2 h[UNITS][kLaneVecs][kVec / 2];
  Raw<W> early[kEarlyWeights ? kLaneVecs : 1];
  {
    Raw<T> x[UNITS][kLaneVecs], add[UNITS][kLaneVecs];
    const T* src = static_cast<const T*>(p.x) + static_cast<uint64_t>(row) * p.x_stride;
    const T* src_add = static_cast<const T*>(p.residual) + static_cast<uint64_t>(row) * p.residual_stride;
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
#pragma unroll
      for (int k = 0; k < kLaneVecs; ++k) {
        const int col = col_of(i) + k * kGroupLanes * kVec;
        const int valid = live ? valid_at<VEC>(col, p.cols) : 0;
        load_norm<T, VEC>(x[i][k], src + col, valid);
        if (p.residual) load_norm<T, VEC>(add[i][k], src_add + col, valid);
      }
    if (kEarlyWeights) {
#pragma unroll
      for (int k = 0; k < kLaneVecs; ++k) {
        const int col = col_of(0) + k * kGroupLanes * kVec;
        load_norm<W, VEC>(early[kEarlyWeights ? k : 0], static_cast<const W*>(p.weight) + col, valid_at<VEC>(col, p.cols));
      }
    }
    T* dst = static_cast<T*>(p.residual_out) + static_cast<uint64_t>(row) * p.residual_out_stride;
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
#pragma unroll
      for (int k = 0; k < kLaneVecs; ++k) {
        const int col = col_of(i) + k * kGroupLanes * kVec;
#pragma unroll
        for (int e = 0; e < kVec / 2; ++e) {
          h[i][k][e] = widen<T>(x[i][k], e);
          if (p.residual) h[i][k][e] = add2(h[i][k][e], widen<T>(add[i][k], e));
        }
        if (p.residual) store_as<T, VEC>(dst + col, h[i][k], live ? valid_at<VEC>(col, p.cols) : 0);
      }
  }
  F2 squares = pack2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
#pragma unroll
    for (int k = 0; k < kLaneVecs; ++k)
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) squares = fma2(h[i][k][e], h[i][k][e], squares);
  float even, odd;
  unpack2(squares, even, odd);
  // 16 UNITS squares a thread and a warp's threads in f32; between warps in double, where a rounding would be
  // the whole row's.
  float in_warp = even + odd;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) in_warp += __shfl_xor_sync(0xffffffffu, in_warp, d);
  double sum = in_warp;
  if (kWarps > 1) {
    if ((t & 31) == 0) partial[r][t / 32] = in_warp;
    __syncthreads();
    sum = (t & 31) < kWarps ? partial[r][t & 31] : 0.f;
#pragma unroll
    for (int d = first_step(kWarps); d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    sum = __shfl_sync(0xffffffffu, sum, 0);
  }
  float hi, lo;
  inverse_root(sum * p.inverse_cols + static_cast<double>(p.epsilon), hi, lo);
  const F2 hi2 = pack2(hi, hi), minus_hi2 = pack2(-hi, -hi), lo2 = pack2(lo, lo);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    float magnitude = 0.f;
#pragma unroll
    for (int k = 0; k < kLaneVecs; ++k) {
      const int col = col_of(i) + k * kGroupLanes * kVec;
      Raw<W> weight;  // from L1 or L2: every row of the SM reads them
      if (kEarlyWeights) weight = early[kEarlyWeights ? k : 0];
      else load_norm<W, VEC>(weight, static_cast<const W*>(p.weight) + col, valid_at<VEC>(col, p.cols));
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) {
        h[i][k][e] = scaled(h[i][k][e], hi2, minus_hi2, lo2, widen<W>(weight, e));
        magnitude = largest_abs(magnitude, h[i][k][e]);
      }
    }
    const uint32_t byte = scale_byte(group_max(__float_as_uint(magnitude)));
    const float inverse = inverse_scale(byte);
#pragma unroll
    for (int k = 0; k < kLaneVecs; ++k) {
      const int col = col_of(i) + k * kGroupLanes * kVec;
      store_codes<VEC>(p.q + static_cast<uint64_t>(row) * p.q_stride + col, h[i][k], pack2(inverse, inverse), live ? valid_at<VEC>(col, p.cols) : 0);
    }
    const int col = col_of(i);
    if (t % kGroupLanes == 0 && live && col < p.cols) p.scales[static_cast<uint64_t>(row) * p.scales_stride + col / kGroup] = static_cast<uint8_t>(byte);
  }
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

int dtype_size(int32_t dtype) { return dtype == CAKE_DTYPE_F32 ? 4 : 2; }

bool known_dtype(int32_t dtype) { return dtype == CAKE_DTYPE_F32 || dtype == CAKE_DTYPE_BF16 || dtype == CAKE_DTYPE_F16; }

// Programmatic serialization: the kernel's launch overlaps its predecessor's tail; it waits on the
// device before it reads anything.
template <typename P>
int32_t launch(void (*kernel)(P), const P& p, unsigned grid, unsigned threads, void* stream) {
  cudaLaunchAttribute overlap;
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.stream = static_cast<cudaStream_t>(stream);
  config.attrs = &overlap;
  config.numAttrs = 1;
  CAKE_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, p));
  return CAKE_OK;
}

// What the two entry points check alike.
int32_t check_output(const char* who, const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t x_stride, int64_t x_cols,
                     const void* q, int64_t q_stride, const void* scales, int64_t scales_stride) {
  if (rows < 0 || rows > INT32_MAX) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: rows must be 0 to 2^31 - 1, got %lld", who, (long long)rows);
  if (!known_dtype(dtype)) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: dtype must be CAKE_DTYPE_F32, _BF16 or _F16", who);
  if (rows == 0) return CAKE_OK;
  if (!x || !q || !scales) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: null argument", who);
  if (!aligned(x, dtype_size(dtype))) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: x is not aligned to its elements", who);
  if (rows > 1 && (x_stride < x_cols || q_stride < cols || scales_stride < (cols + kGroup - 1) / kGroup))
    return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: a row stride is shorter than its row", who);
  if (rows > 1 && (x_stride > UINT32_MAX || q_stride > UINT32_MAX || scales_stride > UINT32_MAX))
    return fail(CAKE_ERR_UNSUPPORTED, "%s: row strides must be below 2^32", who);
  return CAKE_OK;
}

template <typename T>
int32_t launch_quantize(const QuantizeParams& p, bool gate, bool vec, void* stream) {
  const int64_t per_block = ((sizeof(T) == 4 || gate) ? 2 : 4) * (kQuantThreads / kGroupLanes);
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(p.items) + per_block - 1) / per_block);
  void (*kernel)(QuantizeParams) = gate ? (vec ? cake_quantize_rows_sm100<T, true, true> : cake_quantize_rows_sm100<T, true, false>)
                                        : (vec ? cake_quantize_rows_sm100<T, false, true> : cake_quantize_rows_sm100<T, false, false>);
  return launch(kernel, p, grid, kQuantThreads, stream);
}

template <typename T, typename W, int THREADS, int UNITS, bool VEC>
int32_t launch_norm_as(const NormParams& p, void* stream) {
  constexpr unsigned kRows = norm_rows(THREADS);
  return launch(cake_rms_norm_quantize_sm100<T, W, THREADS, UNITS, VEC>, p, (p.rows + kRows - 1) / kRows, THREADS * kRows, stream);
}

template <typename T, typename W, bool VEC>
int32_t launch_norm_vec(const NormParams& p, void* stream) {
  const int units = (p.cols + kGroup - 1) / kGroup * kGroupLanes;
  if (units <= 32) return launch_norm_as<T, W, 32, 1, VEC>(p, stream);
  if (units <= 64) return launch_norm_as<T, W, 64, 1, VEC>(p, stream);
  if (units <= 128) return launch_norm_as<T, W, 128, 1, VEC>(p, stream);
  if (units <= 256) return launch_norm_as<T, W, 256, 1, VEC>(p, stream);
  if (units <= 320) return launch_norm_as<T, W, 160, 2, VEC>(p, stream);
  if (units <= 512) return launch_norm_as<T, W, 256, 2, VEC>(p, stream);
  if (units <= 768) return launch_norm_as<T, W, 384, 2, VEC>(p, stream);
  if (units <= 1024) return launch_norm_as<T, W, 512, 2, VEC>(p, stream);
  return launch_norm_as<T, W, 1024, 2, VEC>(p, stream);
}

template <typename T>
int32_t launch_norm(const NormParams& p, bool same_weight, bool vec, void* stream) {
  if (same_weight) return vec ? launch_norm_vec<T, T, true>(p, stream) : launch_norm_vec<T, T, false>(p, stream);
  return vec ? launch_norm_vec<T, float, true>(p, stream) : launch_norm_vec<T, float, false>(p, stream);
}

}  // namespace
}  // namespace cake

using cake::fail;

extern "C" {

int32_t cake_quantize_rows_enqueue(const void* x, int32_t dtype, int64_t x_row_stride, int32_t gate, int64_t rows, int64_t cols,
                                   void* q, int64_t q_row_stride, void* scales, int64_t scales_row_stride, void* stream) {
  using namespace cake;
  const char* who = "cake_quantize_rows";
  if (cols < 1 || cols > INT32_MAX / 4) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: columns must be 1 to 2^29 - 1, got %lld", who, (long long)cols);
  if (gate != CAKE_GATE_NONE && gate != CAKE_GATE_SILU) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: unknown gate %d", who, gate);
  const int32_t rc = check_output(who, x, dtype, rows, cols, x_row_stride, gate ? 2 * cols : cols, q, q_row_stride, scales, scales_row_stride);
  if (rc || rows == 0) return rc;
  QuantizeParams p;
  p.x = x;
  p.q = static_cast<uint8_t*>(q);
  p.scales = static_cast<uint8_t*>(scales);
  p.x_stride = static_cast<uint32_t>(rows > 1 ? x_row_stride : 0);
  p.q_stride = static_cast<uint32_t>(rows > 1 ? q_row_stride : 0);
  p.scales_stride = static_cast<uint32_t>(rows > 1 ? scales_row_stride : 0);
  p.cols = static_cast<int32_t>(cols);
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  if (rows * groups > INT32_MAX)  // whose rows, two groups each or more, no memory of this GPU holds
    return fail(CAKE_ERR_UNSUPPORTED, "%s: rows times groups must be below 2^31, got %lld", who, (long long)(rows * groups));
  p.items = static_cast<uint32_t>(rows * groups);
  p.by_groups = fast_divisor(static_cast<uint32_t>(groups));
  const int size = dtype_size(dtype);
  const bool vec = cols % kVec == 0 && aligned(x, 16) && (rows == 1 || (x_row_stride * size % 16 == 0 && q_row_stride % 8 == 0)) &&
                   (!gate || cols * size % 16 == 0) && aligned(q, 8);
  if (dtype == CAKE_DTYPE_F32) return launch_quantize<float>(p, gate != 0, vec, stream);
  if (dtype == CAKE_DTYPE_BF16) return launch_quantize<__nv_bfloat16>(p, gate != 0, vec, stream);
  return launch_quantize<__half>(p, gate != 0, vec, stream);
}

int32_t cake_rms_norm_quantize_enqueue(const void* x, int32_t dtype, int64_t x_row_stride, const void* residual,
                                       int64_t residual_row_stride, void* residual_out, int64_t residual_out_row_stride,
                                       const void* weight, int32_t weight_dtype, float epsilon, int64_t rows, int64_t cols,
                                       void* q, int64_t q_row_stride, void* scales, int64_t scales_row_stride, void* stream) {
  using namespace cake;
  const char* who = "cake_rms_norm_quantize";
  if (cols < 1 || cols > CAKE_RMS_NORM_MAX_COLUMNS)
    return fail(CAKE_ERR_UNSUPPORTED, "%s: a row is held on chip, columns must be 1 to %d, got %lld", who, CAKE_RMS_NORM_MAX_COLUMNS, (long long)cols);
  if (weight_dtype != dtype && weight_dtype != CAKE_DTYPE_F32)
    return fail(CAKE_ERR_UNSUPPORTED, "%s: the weight has the type of x or is f32", who);
  if (!(epsilon >= 0.f)) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: epsilon must not be negative", who);
  const int32_t rc = check_output(who, x, dtype, rows, cols, x_row_stride, cols, q, q_row_stride, scales, scales_row_stride);
  if (rc || rows == 0) return rc;
  if (!weight) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: null argument", who);
  if ((residual == nullptr) != (residual_out == nullptr)) return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: residual and residual_out come together", who);
  const int size = dtype_size(dtype);
  if (!aligned(weight, dtype_size(weight_dtype)) || !aligned(residual, size) || !aligned(residual_out, size))
    return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: an operand is not aligned to its elements", who);
  if (residual && rows > 1 && (residual_row_stride < cols || residual_out_row_stride < cols))
    return fail(CAKE_ERR_INVALID_ARGUMENT, "%s: a row stride is shorter than its row", who);
  if (residual && rows > 1 && (residual_row_stride > UINT32_MAX || residual_out_row_stride > UINT32_MAX))
    return fail(CAKE_ERR_UNSUPPORTED, "%s: row strides must be below 2^32", who);
  NormParams p;
  p.x = x;
  p.residual = residual;
  p.residual_out = residual_out;
  p.weight = weight;
  p.q = static_cast<uint8_t*>(q);
  p.scales = static_cast<uint8_t*>(scales);
  p.x_stride = static_cast<uint32_t>(rows > 1 ? x_row_stride : 0);
  p.residual_stride = static_cast<uint32_t>(rows > 1 ? residual_row_stride : 0);
  p.residual_out_stride = static_cast<uint32_t>(rows > 1 ? residual_out_row_stride : 0);
  p.q_stride = static_cast<uint32_t>(rows > 1 ? q_row_stride : 0);
  p.scales_stride = static_cast<uint32_t>(rows > 1 ? scales_row_stride : 0);
  p.rows = static_cast<uint32_t>(rows);
  p.cols = static_cast<int32_t>(cols);
  p.epsilon = epsilon;
  p.inverse_cols = 1.0 / static_cast<double>(cols);
  const bool strides = rows == 1 || (x_row_stride * size % 16 == 0 && q_row_stride % 8 == 0 &&
                                     (!residual || (residual_row_stride * size % 16 == 0 && residual_out_row_stride * size % 16 == 0)));
  const bool vec = cols % kVec == 0 && strides && aligned(x, 16) && aligned(residual, 16) && aligned(residual_out, 16) && aligned(weight, 16) && aligned(q, 8);
  if (dtype == CAKE_DTYPE_F32) return launch_norm<float>(p, true, vec, stream);
  if (dtype == CAKE_DTYPE_BF16) return launch_norm<__nv_bfloat16>(p, weight_dtype == dtype, vec, stream);
  return launch_norm<__half>(p, weight_dtype == dtype, vec, stream);
}

}  // extern "C"
