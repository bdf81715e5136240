// Matrices held in MXFP4 - 32 consecutive values of a row as 4-bit floats (e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) under one
// power of two (e8m0), the OCP microscaling format - and their products on gfx950's scaled matrix instructions: a fully connected head
// served from, or attacked through, four-bit weights (the heads of dynamic_vehicles/Model.py:15-34, a detector's RoI head).
//
//   quantise  e = clamp(floor(log2 max|x|) - 2, -127, 127) per block, code = nearest-even(x / 2^e), saturated at 6; scale byte = e + 127.
//             A block that holds a NaN or an infinity is NaN as a whole (scale byte 255); an all-zero block has scale byte 0.
//   linear    y = relu?(Q(x) . W^T + b): a product of two blocks' codes and scales is exact in the matrix instruction, sums are float32
//   dgrad     gx = (gy where the ReLU let it pass) . W: W's values are exact in bfloat16, and gy goes in as the exact sum of bfloat16 terms
//             (three for float32, two for half, one for bfloat16) - the contraction runs across W's blocks, which the scaled instruction
//             cannot do
//
// Layout ("panels" of 256 columns): codes [panel][row][128 bytes], low nibble first; scales [panel][row][8].  What a workgroup reads of a
// panel - some rows - is one contiguous piece, a lane's scale bytes for four matrix instructions are one aligned dword, and a panel is
// padded with zero codes, so no kernel has a tail in the contraction.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "adv_internal.h"
#include "advengine.h"
#include "lowp.h"

namespace {

constexpr int kBlock = 256;
constexpr int kPanel = 256;                // columns of a panel: 128 code bytes, 8 scale bytes a row
typedef int Int8 __attribute__((ext_vector_type(8)));
typedef float Float16 __attribute__((ext_vector_type(16)));
typedef float Float2 __attribute__((ext_vector_type(2)));
typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t Uint4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int64_t panels_of(int64_t cols) { return (cols + kPanel - 1) / kPanel; }

// ---- quantise / dequantise.  V elements (16 bytes) a lane, kPanel / V lanes a panel's row; a wave walks rows of one panel, so that what it
//      writes is contiguous.  Bound by memory: 4.5 bytes moved a float32 value against ~6 instructions a lane's V values.
constexpr int kRowsPerWave = 4;            // row groups a wave takes

template <class T>
__global__ __launch_bounds__(kBlock) void mx4_quantize(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows,
                                                       int64_t cols) {
  constexpr int V = 16 / sizeof(T), kLanes = kPanel / V, kGroup = 64 / kLanes;      // lanes a row, rows a wave takes at once
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t panel = blockIdx.y;
  const int in_row = lane % kLanes;
  const int64_t col = panel * kPanel + in_row * V;
  const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(V), cols - col)));
  const int64_t row0 = ((static_cast<int64_t>(blockIdx.x) * (kBlock / 64) + wave) * kRowsPerWave) * kGroup + lane / kLanes;
#pragma unroll
  for (int k = 0; k < kRowsPerWave; ++k) {
    const int64_t row = row0 + k * kGroup;
    if (row >= rows) continue;               // (whole rows of lanes leave together: the exchanges below stay within one)
    float v[V];
    if (left == V) lowp::load<T, V>(x + row * cols + col, v);
    else lowp::load_some<T, V>(x + row * cols + col, v, left);
    uint32_t top = 0;                        // the largest magnitude's bits: NaN and infinities come out on top
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < 32 / V; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
    const bool none = top >= 0x7f800000u;
    const int ex = static_cast<int>(top >> 23) - 2;
    const uint32_t scale = none ? 255u : static_cast<uint32_t>(max(ex, 0));
    const float unit = __uint_as_float(max(scale << 23, 0x00400000u));                 // 2^-127 is a subnormal
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], unit, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], unit, 1);
    if (V == 8) {
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[V - 4], v[V - 3], unit, 2);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[V - 2], v[V - 1], unit, 3);
    }
    if (none) q = 0;
    uint8_t* c = codes + (panel * rows + row) * (kPanel / 2) + in_row * (V / 2);
    if (V == 8) *reinterpret_cast<uint32_t*>(c) = q;
    else *reinterpret_cast<uint16_t*>(c) = static_cast<uint16_t>(q);
    if (in_row % (32 / V) == 0) scales[(panel * rows + row) * 8 + in_row / (32 / V)] = static_cast<uint8_t>(scale);
  }
}

template <class T>
__global__ __launch_bounds__(kBlock) void mx4_dequantize(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ x,
                                                         int64_t rows, int64_t cols) {
  constexpr int V = 16 / sizeof(T), kLanes = kPanel / V, kGroup = 64 / kLanes;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t panel = blockIdx.y;
  const int in_row = lane % kLanes;
  const int64_t col = panel * kPanel + in_row * V;
  const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(V), cols - col)));
  if (left == 0) return;
  const int64_t row0 = ((static_cast<int64_t>(blockIdx.x) * (kBlock / 64) + wave) * kRowsPerWave) * kGroup + lane / kLanes;
#pragma unroll
  for (int k = 0; k < kRowsPerWave; ++k) {
    const int64_t row = row0 + k * kGroup;
    if (row >= rows) continue;
    const uint8_t* c = codes + (panel * rows + row) * (kPanel / 2) + in_row * (V / 2);
    const uint32_t q = V == 8 ? *reinterpret_cast<const uint32_t*>(c) : *reinterpret_cast<const uint16_t*>(c);
    const float unit = __uint_as_float(static_cast<uint32_t>(scales[(panel * rows + row) * 8 + in_row / (32 / V)]) << 23);
    float v[V];
    Float2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, unit, 0);
    v[0] = p.x, v[1] = p.y;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, unit, 1);
    v[2] = p.x, v[3] = p.y;
    if (V == 8) {
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, unit, 2);
      v[V - 4] = p.x, v[V - 3] = p.y;
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, unit, 3);
      v[V - 2] = p.x, v[V - 1] = p.y;
    }
    if (left == V) lowp::store<T, V>(x + row * cols + col, v);
    else lowp::store_some<T, V>(x + row * cols + col, v, left);
  }
}

// ---- the product.  v_mfma_scale_f32_32x32x64_f8f6f4 with both operands e2m1: lane l holds 32 consecutive values of row l % 32 of A (or B), the
//      first half of the wave the lower and the second the upper 32 of the 64, and their scale byte.  Which columns those are is free as long
//      as A and B agree: here the lower half takes the first four blocks of a panel in turn, the upper half the last four.
struct Operand {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows;
};

__device__ __forceinline__ Int8 widen(Uint4 v) {
  return Int8{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
}

template <int SEL>
__device__ __forceinline__ Float16 mfma(Uint4 a, Uint4 b, Float16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(a), widen(b), c, 4, 4, SEL, static_cast<int>(sa), SEL, static_cast<int>(sb));
}

template <class T>
__device__ __forceinline__ float finish(float v, const T* bias, int64_t n, int relu) {
  if (bias) v += static_cast<float>(bias[n]);
  return relu && v < 0.0f ? 0.0f : v;      // (a NaN stays)
}

// One 32 x 32 tile of y a workgroup, its four waves taking the panels in turn and joining their sums in LDS.
template <class T>
__global__ __launch_bounds__(kBlock) void mx4_linear(Operand x, Operand w, const T* __restrict__ bias, T* __restrict__ y, int64_t panels, int relu) {
  __shared__ float s_sum[3][16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 32, n0 = static_cast<int64_t>(blockIdx.x) * 32;
  const int64_t m = min(m0 + (lane & 31), x.rows - 1), n = min(n0 + (lane & 31), w.rows - 1);      // rows behind the last one are computed, not stored
  Float16 acc = {};
  for (int64_t p = wave; p < panels; p += 4) {
    const Uint4* xa = reinterpret_cast<const Uint4*>(x.codes + (p * x.rows + m) * 128 + half * 64);
    const Uint4* wb = reinterpret_cast<const Uint4*>(w.codes + (p * w.rows + n) * 128 + half * 64);
    const uint32_t sx = *reinterpret_cast<const uint32_t*>(x.scales + (p * x.rows + m) * 8 + half * 4);
    const uint32_t sw = *reinterpret_cast<const uint32_t*>(w.scales + (p * w.rows + n) * 8 + half * 4);
    acc = mfma<0>(xa[0], wb[0], acc, sx, sw);
    acc = mfma<1>(xa[1], wb[1], acc, sx, sw);
    acc = mfma<2>(xa[2], wb[2], acc, sx, sw);
    acc = mfma<3>(xa[3], wb[3], acc, sx, sw);
  }
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s_sum[wave - 1][i][lane] = acc[i];
  }
  __syncthreads();
  if (wave > 0) return;
  const int64_t nn = n0 + (lane & 31);
  if (nn >= w.rows) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t mm = m0 + 8 * (i / 4) + 4 * half + i % 4;
    const float v = acc[i] + s_sum[0][i][lane] + s_sum[1][i][lane] + s_sum[2][i][lane];
    if (mm < x.rows) y[mm * w.rows + nn] = static_cast<T>(finish<T>(v, bias, nn, relu));
  }
}

// ---- the input gradient.  A workgroup owns kGradRows rows x one panel of gx and walks W's rows 64 at a time: their codes become bfloat16
//      values in LDS, turned so that a lane's eight values along the contraction are 16 bytes; gy goes there as its bfloat16 terms.
constexpr int kGradRows = 64, kChunk = 64;

template <class T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kTerms<__bf16> = 1;

// v as the exact sum of N bfloat16 (cut, not rounded: what is left always fits the next ones, and a finite v stays finite)
template <int N>
__device__ __forceinline__ void split(float v, uint32_t (&t)[N]) {
  const uint32_t u = __float_as_uint(v);
  const bool finite = (u & 0x7f800000u) != 0x7f800000u;
  t[0] = v != v ? 0x7fc0u : u >> 16;
#pragma unroll
  for (int k = 1; k < N; ++k) {
    v -= __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    t[k] = finite ? __float_as_uint(v) >> 16 : 0u;
  }
}

// 16-byte chunk c of a 128-byte row r lies at chunk c ^ (r % 8): eight rows' equal chunks are in eight different places
__device__ __forceinline__ int swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

template <class T>
__global__ __launch_bounds__(kBlock) void mx4_dgrad(const T* __restrict__ gy, const T* __restrict__ mask, Operand w, T* __restrict__ gx, int64_t rows,
                                                    int64_t cols) {
  constexpr int N = kTerms<T>;
  __shared__ __attribute__((aligned(16))) uint8_t s_w[kPanel * 128];
  __shared__ __attribute__((aligned(16))) uint8_t s_g[N][kGradRows * 128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, half = lane >> 5;
  const int64_t panel = blockIdx.x, m0 = static_cast<int64_t>(blockIdx.y) * kGradRows, nw = w.rows;
  Float16 acc[2][2] = {};
  for (int64_t n0 = 0; n0 < nw; n0 += kChunk) {
    __syncthreads();
    {  // eight rows (n) x eight columns of W a thread
      const int o = t & 7, u = t >> 3;
      uint32_t q[8];
      float unit[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t n = n0 + 8 * o + j;
        const bool in = n < nw;
        const int64_t at = panel * nw + (in ? n : nw - 1);
        const uint32_t code = *reinterpret_cast<const uint32_t*>(w.codes + at * 128 + 4 * u);
        const uint32_t scale = w.scales[at * 8 + u / 4];
        q[j] = in ? code : 0u;
        unit[j] = __uint_as_float((in ? scale : 127u) << 23);
      }
      uint32_t v[8][4];                      // [row][pair of columns]
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[j], unit[j], 0));
        v[j][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[j], unit[j], 1));
        v[j][2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[j], unit[j], 2));
        v[j][3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[j], unit[j], 3));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {          // column 8u + k: its eight rows' values
        Uint4 out;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a = v[2 * j][k / 2], b = v[2 * j + 1][k / 2];
          out[j] = k & 1 ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
        }
        *reinterpret_cast<Uint4*>(s_w + swizzled(8 * u + k, o)) = out;
      }
    }
    for (int unit = t; unit < kGradRows * (kChunk / 8); unit += kBlock) {      // eight consecutive n of a row of gy
      const int r = unit >> 3, c = unit & 7;
      const int64_t m = m0 + r, n = n0 + 8 * c;
      float g[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = 0.0f;
      if (m < rows) {
        const T* p = gy + m * nw + n;
        const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(8), nw - n)));
        lowp::load_some<T, 8>(p, g, left);
        if (mask) {
          float o[8];
          lowp::load_some<T, 8>(mask + m * nw + n, o, left);
#pragma unroll
          for (int k = 0; k < 8; ++k) g[k] = o[k] <= 0.0f ? 0.0f : g[k];
        }
      }
      Uint4 out[N];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a[N], b[N];
        split<N>(g[2 * k], a);
        split<N>(g[2 * k + 1], b);
#pragma unroll
        for (int s = 0; s < N; ++s) out[s][k] = a[s] | b[s] << 16;
      }
#pragma unroll
      for (int s = 0; s < N; ++s) *reinterpret_cast<Uint4*>(s_g[s] + swizzled(r, c)) = out[s];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kChunk / 16; ++k) {  // 16 of the contraction a matrix instruction: lane half h has chunk 2k + h
      Bf16x8 b[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) b[j] = *reinterpret_cast<const Bf16x8*>(s_w + swizzled(wave * 64 + j * 32 + (lane & 31), 2 * k + half));
#pragma unroll
      for (int s = 0; s < N; ++s) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const Bf16x8 a = *reinterpret_cast<const Bf16x8*>(s_g[s] + swizzled(i * 32 + (lane & 31), 2 * k + half));
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t col = panel * kPanel + wave * 64 + j * 32 + (lane & 31);
      if (col >= cols) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t m = m0 + i * 32 + 8 * (e / 4) + 4 * half + e % 4;
        if (m < rows) gx[m * cols + col] = static_cast<T>(acc[i][j][e]);
      }
    }
  }
}

// sizes: every product of two of them fits an int64, every grid dimension its limit
constexpr int64_t kMostRows = int64_t{1} << 20, kMostCols = int64_t{1} << 22;

bool sizes_ok(int64_t rows, int64_t cols) { return rows >= 1 && cols >= 1 && rows <= kMostRows && cols <= kMostCols; }
int64_t code_bytes(int64_t rows, int64_t cols) { return panels_of(cols) * rows * (kPanel / 2); }
int64_t scale_bytes(int64_t rows, int64_t cols) { return panels_of(cols) * rows * 8; }

template <class T>
dim3 panel_grid(int64_t rows, int64_t cols) {
  const int64_t per = static_cast<int64_t>(kBlock / 64) * kRowsPerWave * (64 / (kPanel / (16 / static_cast<int>(sizeof(T)))));
  return dim3(static_cast<unsigned>((rows + per - 1) / per), static_cast<unsigned>(panels_of(cols)));
}

template <class T>
int run_quantize(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, hipStream_t st) {
  mx4_quantize<T><<<panel_grid<T>(rows, cols), kBlock, 0, st>>>(static_cast<const T*>(x), codes, scales, rows, cols);
  return adv_internal_finish_launch();
}
template <class T>
int run_dequantize(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int64_t cols, hipStream_t st) {
  mx4_dequantize<T><<<panel_grid<T>(rows, cols), kBlock, 0, st>>>(codes, scales, static_cast<T*>(x), rows, cols);
  return adv_internal_finish_launch();
}
template <class T>
int run_linear(Operand x, Operand w, const void* bias, void* y, int64_t k, int relu, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((w.rows + 31) / 32), static_cast<unsigned>((x.rows + 31) / 32));
  mx4_linear<T><<<grid, kBlock, 0, st>>>(x, w, static_cast<const T*>(bias), static_cast<T*>(y), panels_of(k), relu);
  return adv_internal_finish_launch();
}
template <class T>
int run_dgrad(const void* gy, const void* mask, Operand w, void* gx, int64_t m, int64_t k, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(panels_of(k)), static_cast<unsigned>((m + kGradRows - 1) / kGradRows));
  mx4_dgrad<T><<<grid, kBlock, 0, st>>>(static_cast<const T*>(gy), static_cast<const T*>(mask), w, static_cast<T*>(gx), m, k);
  return adv_internal_finish_launch();
}

}  // namespace

extern "C" {

int64_t adv_mx4_code_bytes(int64_t rows, int64_t cols) {
  if (rows == 0 && cols >= 1 && cols <= kMostCols) return 0;
  return sizes_ok(rows, cols) ? code_bytes(rows, cols) : ADV_EINVAL;
}

int adv_mx4_quantize(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, int dtype, adv_stream_t stream) {
  if (!x || !codes || !scales || !sizes_ok(rows, cols) || !lowp::known(dtype)) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  if (!lowp::aligned(x, e) || !lowp::aligned(codes, 16) || !lowp::aligned(scales, 8)) return ADV_EALIGN;
  const int64_t cb = code_bytes(rows, cols), sb = scale_bytes(rows, cols), xb = rows * cols * e;
  if (lowp::overlap(x, xb, codes, cb) || lowp::overlap(x, xb, scales, sb) || lowp::overlap(codes, cb, scales, sb)) return ADV_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ADV_F32) return run_quantize<float>(x, codes, scales, rows, cols, st);
  if (dtype == ADV_BF16) return run_quantize<__bf16>(x, codes, scales, rows, cols, st);
  return run_quantize<_Float16>(x, codes, scales, rows, cols, st);
}

int adv_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* x, int64_t rows, int64_t cols, int dtype, adv_stream_t stream) {
  if (!x || !codes || !scales || !sizes_ok(rows, cols) || !lowp::known(dtype)) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  if (!lowp::aligned(x, e) || !lowp::aligned(codes, 16) || !lowp::aligned(scales, 8)) return ADV_EALIGN;
  const int64_t xb = rows * cols * e;
  if (lowp::overlap(x, xb, codes, code_bytes(rows, cols)) || lowp::overlap(x, xb, scales, scale_bytes(rows, cols))) return ADV_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ADV_F32) return run_dequantize<float>(codes, scales, x, rows, cols, st);
  if (dtype == ADV_BF16) return run_dequantize<__bf16>(codes, scales, x, rows, cols, st);
  return run_dequantize<_Float16>(codes, scales, x, rows, cols, st);
}

int adv_mx4_linear(const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales, const void* bias, void* y, int64_t m,
                   int64_t n, int64_t k, int dtype, int relu, adv_stream_t stream) {
  if (!x_codes || !x_scales || !w_codes || !w_scales || !y || !sizes_ok(m, k) || !sizes_ok(n, k) || !lowp::known(dtype)) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  if (!lowp::aligned(x_codes, 16) || !lowp::aligned(w_codes, 16) || !lowp::aligned(x_scales, 8) || !lowp::aligned(w_scales, 8) || !lowp::aligned(y, e) ||
      !lowp::aligned(bias, e))
    return ADV_EALIGN;
  const int64_t yb = m * n * e;
  if (lowp::overlap(y, yb, x_codes, code_bytes(m, k)) || lowp::overlap(y, yb, x_scales, scale_bytes(m, k)) || lowp::overlap(y, yb, w_codes, code_bytes(n, k)) ||
      lowp::overlap(y, yb, w_scales, scale_bytes(n, k)) || (bias && lowp::overlap(y, yb, bias, n * e)))
    return ADV_EINVAL;
  const Operand x{x_codes, x_scales, m}, w{w_codes, w_scales, n};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ADV_F32) return run_linear<float>(x, w, bias, y, k, relu, st);
  if (dtype == ADV_BF16) return run_linear<__bf16>(x, w, bias, y, k, relu, st);
  return run_linear<_Float16>(x, w, bias, y, k, relu, st);
}

int adv_mx4_linear_dgrad(const void* gy, const void* mask, const uint8_t* w_codes, const uint8_t* w_scales, void* gx, int64_t m, int64_t n, int64_t k, int dtype,
                         adv_stream_t stream) {
  if (!gy || !w_codes || !w_scales || !gx || !sizes_ok(m, k) || !sizes_ok(n, k) || !lowp::known(dtype)) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  if (!lowp::aligned(gy, e) || !lowp::aligned(mask, e) || !lowp::aligned(gx, e) || !lowp::aligned(w_codes, 16) || !lowp::aligned(w_scales, 8)) return ADV_EALIGN;
  const int64_t xb = m * k * e, gb = m * n * e;
  if (lowp::overlap(gx, xb, gy, gb) || (mask && lowp::overlap(gx, xb, mask, gb)) || lowp::overlap(gx, xb, w_codes, code_bytes(n, k)) ||
      lowp::overlap(gx, xb, w_scales, scale_bytes(n, k)))
    return ADV_EINVAL;
  const Operand w{w_codes, w_scales, n};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ADV_F32) return run_dgrad<float>(gy, mask, w, gx, m, k, st);
  if (dtype == ADV_BF16) return run_dgrad<__bf16>(gy, mask, w, gx, m, k, st);
  return run_dgrad<_Float16>(gy, mask, w, gx, m, k, st);
}

}  // extern "C"
