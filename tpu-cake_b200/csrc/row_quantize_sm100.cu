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
// Both kernels are bound by HBM: one pass, every byte read and written once, 16 lanes per group with 8
// elements each (one 16-byte load of a 16-bit type), so a group's maximum is four shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cake_host.h"
#include "cake_ptx.cuh"

namespace cake {
namespace {

constexpr int kGroup = 128;  // columns that share a scale
constexpr int kVec = 8;      // elements of one lane
constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 4;  // groups in flight per half warp

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight elements as they lie in memory.
template <typename T>
struct Raw {
  static constexpr int kWords = kVec * static_cast<int>(sizeof(T)) / 16;
  uint4 w[kWords];
};

// Loads elements [0, valid) of the eight at `ptr`; the others are zero. VEC: all loads of whole vectors
// are 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(Raw<T>& r, const T* ptr, int valid) {
  if (VEC && valid >= kVec) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; ++i) r.w[i] = reinterpret_cast<const uint4*>(ptr)[i];
    return;
  }
  T e[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) e[i] = i < valid ? ptr[i] : from_f32<T>(0.f);
  memcpy(&r, e, sizeof(r));
}

template <typename T>
__device__ __forceinline__ void widen(float (&v)[kVec], const Raw<T>& r) {
  T e[kVec];
  memcpy(e, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = to_f32(e[i]);
}

// Stores elements [0, valid) of eight.
template <typename T, bool VEC>
__device__ __forceinline__ void store_as(T* ptr, const float (&v)[kVec], int valid) {
  T e[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) e[i] = from_f32<T>(v[i]);
  if (VEC && valid >= kVec) {
    Raw<T> r;
    memcpy(&r, e, sizeof(r));
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; ++i) reinterpret_cast<uint4*>(ptr)[i] = r.w[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (i < valid) ptr[i] = e[i];
}

// Magnitudes are compared as integers: that order is the magnitudes' own, with every NaN above infinity,
// so a NaN is never lost as it would be by a floating-point maximum.
__device__ __forceinline__ uint32_t largest_magnitude(const float (&v)[kVec]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return a;
}

// The maximum over the 16 lanes of a half warp.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t a) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, d));
  return a;
}

// Scale byte of a group whose largest magnitude has the bits `a`. With a = 1.m * 2^(E - 127) and
// 448 = 1.75 * 2^8 the exponent is E - 127 - 8, one more where 1.m > 1.75.
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
  if (a >= 0x7F800000u) return 255u;
  if (a == 0) return 127u;
  const int e = static_cast<int>(a >> 23) - 8 + ((a & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 0));
}

// The eight codes of a lane: v / 2^(byte - 127), rounded to nearest even.
__device__ __forceinline__ uint2 encode(const float (&v)[kVec], uint32_t byte) {
  if (byte == 255u) return make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
  const float inv = __uint_as_float((254u - byte) << 23);  // byte <= 247: a normal number
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// Stores codes [0, valid) of eight; whole vectors as one 8-byte store where VEC says they are aligned.
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* ptr, uint2 codes, int valid) {
  if (VEC && valid >= kVec) {
    *reinterpret_cast<uint2*>(ptr) = codes;
    return;
  }
  const uint64_t all = (static_cast<uint64_t>(codes.y) << 32) | codes.x;
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (i < valid) ptr[i] = static_cast<uint8_t>(all >> (8 * i));
}

// Division by a number known at launch, for dividends below 2^31: multiply, shift.
struct FastDivisor {
  uint32_t d, magic, shift;
};

__device__ __forceinline__ uint32_t divide(uint32_t n, const FastDivisor& f) {
  return (__umulhi(n, f.magic) + n) >> f.shift;
}

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
  int64_t x_stride, q_stride, scales_stride;  // elements (bytes) between rows
  int64_t items;                              // rows * groups
  int32_t cols, groups;
  FastDivisor by_groups;
};

// x / (1 + exp(-x)). For x below about -88 the exponential is infinite and the result -0.
__device__ __forceinline__ float silu(float x) { return x / (1.f + expf(-x)); }

// A half warp takes kQuantUnroll groups that are 16 apart, so that a block's groups lie next to each
// other and every lane has that many loads in flight.
template <typename T, bool GATE, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) cake_quantize_rows_sm100(const __grid_constant__ QuantizeParams p) {
  grid_dependency_wait();
  grid_dependency_trigger();
  const int lane = threadIdx.x & 15;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kQuantUnroll * (kQuantThreads / 16)) + (threadIdx.x >> 4);
  int64_t row[kQuantUnroll];
  int group[kQuantUnroll], valid[kQuantUnroll];
  Raw<T> x[kQuantUnroll], up[GATE ? kQuantUnroll : 1];
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    const int64_t item = first + u * (kQuantThreads / 16);
    if (p.items < (1ll << 31)) {
      const uint32_t r = divide(static_cast<uint32_t>(item), p.by_groups);  // item < items + 64: also below 2^31 + 64
      row[u] = r;
      group[u] = static_cast<int>(static_cast<uint32_t>(item) - r * p.by_groups.d);
    } else {
      row[u] = item / p.groups;
      group[u] = static_cast<int>(item - row[u] * p.groups);
    }
    // Items past the end have nothing valid: they load and store nothing.
    valid[u] = item < p.items ? min(max(p.cols - (group[u] * kGroup + lane * kVec), 0), kVec) : 0;
    const T* src = static_cast<const T*>(p.x) + row[u] * p.x_stride + group[u] * kGroup + lane * kVec;
    load_raw<T, VEC>(x[u], src, valid[u]);
    if (GATE) load_raw<T, VEC>(up[GATE ? u : 0], src + p.cols, valid[u]);
  }
#pragma unroll
  for (int u = 0; u < kQuantUnroll; ++u) {
    float v[kVec];
    widen<T>(v, x[u]);
    if (GATE) {
      float w[kVec];
      widen<T>(w, up[GATE ? u : 0]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = silu(v[i]) * w[i];
    }
    const uint32_t byte = scale_byte(half_warp_max(largest_magnitude(v)));
    if (valid[u] > 0) {
      store_codes<VEC>(p.q + row[u] * p.q_stride + group[u] * kGroup + lane * kVec, encode(v, byte), valid[u]);
      if (lane == 0) p.scales[row[u] * p.scales_stride + group[u]] = static_cast<uint8_t>(byte);
    }
  }
}

struct NormParams {
  const void* x;
  const void* residual;  // or null
  void* residual_out;    // with a residual only
  const void* weight;
  uint8_t* q;
  uint8_t* scales;
  int64_t x_stride, residual_stride, residual_out_stride, q_stride, scales_stride;
  int64_t rows;
  int32_t cols;
  float epsilon;
};

// THREADS threads hold one row in registers (VECS vectors of eight each, vector i of thread t being
// number i * THREADS + t of the row), so the sum x + residual is normalised as it is in 32 bits while its
// rounding is stored, and the stored sum may lie over x or over the residual. Blocks of 32 threads a row
// carry eight rows.
template <typename T, typename W, int THREADS, int VECS, bool VEC>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) cake_rms_norm_quantize_sm100(const __grid_constant__ NormParams p) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;  // rows of a block
  constexpr int kWarps = THREADS / 32;                      // warps of a row
  __shared__ float partial[kRows][kWarps];
  grid_dependency_wait();
  grid_dependency_trigger();
  const int t = threadIdx.x % THREADS;
  const int r = threadIdx.x / THREADS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + r;
  const bool live = row < p.rows;
  float h[VECS][kVec];
  Raw<W> weight[VECS];
  int valid[VECS];
  {
    Raw<T> x[VECS], add[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int col = (i * THREADS + t) * kVec;
      valid[i] = live ? min(max(p.cols - col, 0), kVec) : 0;
      load_raw<T, VEC>(x[i], static_cast<const T*>(p.x) + row * p.x_stride + col, valid[i]);
      if (p.residual) load_raw<T, VEC>(add[i], static_cast<const T*>(p.residual) + row * p.residual_stride + col, valid[i]);
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) load_raw<W, VEC>(weight[i], static_cast<const W*>(p.weight) + (i * THREADS + t) * kVec, valid[i]);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      widen<T>(h[i], x[i]);
      if (p.residual) {
        float a[kVec];
        widen<T>(a, add[i]);
#pragma unroll
        for (int e = 0; e < kVec; ++e) h[i][e] += a[e];
        store_as<T, VEC>(static_cast<T*>(p.residual_out) + row * p.residual_out_stride + (i * THREADS + t) * kVec, h[i], valid[i]);
      }
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; ++i)
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum = fmaf(h[i][e], h[i][e], sum);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (kWarps > 1) {
    if ((t & 31) == 0) partial[r][t / 32] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += partial[r][w];
  }
  const float scale = 1.f / sqrtf(sum / static_cast<float>(p.cols) + p.epsilon);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    float w[kVec];
    widen<W>(w, weight[i]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) h[i][e] = h[i][e] * scale * w[e];
    const uint32_t byte = scale_byte(half_warp_max(largest_magnitude(h[i])));
    if (valid[i] > 0) {
      const int vec = i * THREADS + t;
      store_codes<VEC>(p.q + row * p.q_stride + vec * kVec, encode(h[i], byte), valid[i]);
      if ((t & 15) == 0) p.scales[row * p.scales_stride + vec / 16] = static_cast<uint8_t>(byte);
    }
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
  return CAKE_OK;
}

template <typename T>
int32_t launch_quantize(const QuantizeParams& p, bool gate, bool vec, void* stream) {
  const int64_t per_block = kQuantUnroll * (kQuantThreads / 16);
  const unsigned grid = static_cast<unsigned>((p.items + per_block - 1) / per_block);
  void (*kernel)(QuantizeParams) = gate ? (vec ? cake_quantize_rows_sm100<T, true, true> : cake_quantize_rows_sm100<T, true, false>)
                                        : (vec ? cake_quantize_rows_sm100<T, false, true> : cake_quantize_rows_sm100<T, false, false>);
  return launch(kernel, p, grid, kQuantThreads, stream);
}

template <typename T, typename W, bool VEC>
int32_t launch_norm_vec(const NormParams& p, void* stream) {
  const int64_t vectors = (p.cols + kVec - 1) / kVec;
  if (vectors <= 32 * 4) return launch(cake_rms_norm_quantize_sm100<T, W, 32, 4, VEC>, p, static_cast<unsigned>((p.rows + 7) / 8), 256, stream);
  if (vectors <= 128 * 4) return launch(cake_rms_norm_quantize_sm100<T, W, 128, 4, VEC>, p, static_cast<unsigned>((p.rows + 1) / 2), 256, stream);
  if (vectors <= 256 * 4) return launch(cake_rms_norm_quantize_sm100<T, W, 256, 4, VEC>, p, static_cast<unsigned>(p.rows), 256, stream);
  if (vectors <= 512 * 4) return launch(cake_rms_norm_quantize_sm100<T, W, 512, 4, VEC>, p, static_cast<unsigned>(p.rows), 512, stream);
  return launch(cake_rms_norm_quantize_sm100<T, W, 1024, 4, VEC>, p, static_cast<unsigned>(p.rows), 1024, stream);
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
  p.x_stride = x_row_stride;
  p.q_stride = q_row_stride;
  p.scales_stride = scales_row_stride;
  p.cols = static_cast<int32_t>(cols);
  p.groups = static_cast<int32_t>((cols + kGroup - 1) / kGroup);
  p.items = rows * p.groups;
  p.by_groups = fast_divisor(static_cast<uint32_t>(p.groups));
  if (p.items > static_cast<int64_t>(INT32_MAX) * 64) return fail(CAKE_ERR_UNSUPPORTED, "%s: %lld groups are more than one launch covers", who, (long long)p.items);
  const int size = dtype_size(dtype);
  const bool vec = aligned(x, 16) && (rows == 1 || (x_row_stride * size % 16 == 0 && q_row_stride % 8 == 0)) &&
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
  NormParams p;
  p.x = x;
  p.residual = residual;
  p.residual_out = residual_out;
  p.weight = weight;
  p.q = static_cast<uint8_t*>(q);
  p.scales = static_cast<uint8_t*>(scales);
  p.x_stride = x_row_stride;
  p.residual_stride = residual_row_stride;
  p.residual_out_stride = residual_out_row_stride;
  p.q_stride = q_row_stride;
  p.scales_stride = scales_row_stride;
  p.rows = rows;
  p.cols = static_cast<int32_t>(cols);
  p.epsilon = epsilon;
  const bool strides = rows == 1 || (x_row_stride * size % 16 == 0 && q_row_stride % 8 == 0 &&
                                     (!residual || (residual_row_stride * size % 16 == 0 && residual_out_row_stride * size % 16 == 0)));
  const bool vec = strides && aligned(x, 16) && aligned(residual, 16) && aligned(residual_out, 16) && aligned(weight, 16) && aligned(q, 8);
  if (dtype == CAKE_DTYPE_F32) return launch_norm<float>(p, true, vec, stream);
  if (dtype == CAKE_DTYPE_BF16) return launch_norm<__nv_bfloat16>(p, weight_dtype == dtype, vec, stream);
  return launch_norm<__half>(p, weight_dtype == dtype, vec, stream);
}

}  // extern "C"
