// Matrices held in MXFP4 - 32 consecutive values of a row as 4-bit floats (e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) under one
// power of two (e8m0), the OCP microscaling format - and their products on gfx950's scaled matrix instructions: a fully connected head
// served from, or attacked through, four-bit weights (the heads of dynamic_vehicles/Model.py:15-34, a detector's RoI head).
//
//   quantise  e = clamp(floor(log2 max|x|) - 2, -127, 127) per block, code = nearest-even(x / 2^e), saturated at 6; scale byte = e + 127.
//             A block that holds a NaN or an infinity is NaN as a whole (scale byte 255); an all-zero block has scale byte 0.
//   linear    y = relu?(Q(x) . W^T + b): a product of two blocks' codes and scales is exact in the matrix instruction, sums are float32
//   dgrad     gx = (gy where the ReLU let it pass) . W: W's values are exact in bfloat16, and gy goes in as the exact sum of bfloat16 terms
//             (three for float32, two for half, one for bfloat16; of a float32 below 2^-110 what lies under 2^-133, bfloat16's last bit, is
//             cut) - the contraction runs across W's blocks, which the scaled instruction cannot do
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
typedef float Float4 __attribute__((ext_vector_type(4)));
typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t Uint4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int64_t panels_of(int64_t cols) { return (cols + kPanel - 1) / kPanel; }

struct Coded {
  uint32_t code, scale;
};
// V consecutive values of a lane, 32 / V neighbouring lanes a block: their codes and the block's scale byte
template <int V>
__device__ __forceinline__ Coded encode(const float (&v)[V]) {
  uint32_t top = 0;                        // the largest magnitude's bits: NaN and infinities come out on top
#pragma unroll
  for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < 32 / V; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
  const bool none = top >= 0x7f800000u;
  const uint32_t scale = none ? 255u : static_cast<uint32_t>(max(static_cast<int>(top >> 23) - 2, 0));
  const float unit = __uint_as_float(max(scale << 23, 0x00400000u));                 // 2^-127 is a subnormal
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], unit, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], unit, 1);
  if (V == 8) {
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[V - 4], v[V - 3], unit, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[V - 2], v[V - 1], unit, 3);
  }
  return {none ? 0u : q, scale};
}

// ---- quantise / dequantise.  V elements (16 bytes) a lane, kPanel / V lanes a panel's row; a wave walks rows of one panel, so that what it
//      writes is contiguous.  Bound by memory: 4.5 bytes moved a float32 value against ~6 instructions a lane's V values.  4096 x 25088 float32:
//      81 us to the codes, 79 back (5.7 TB/s; a copy of 1 GiB reaches 5.05, the codes come from the last-level cache).
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
  float v[kRowsPerWave][V];                  // every row's values are asked for before the first is used
#pragma unroll
  for (int k = 0; k < kRowsPerWave; ++k) {
    const int64_t row = min(row0 + k * kGroup, rows - 1);
    if (left == V) lowp::load<T, V>(x + row * cols + col, v[k]);
    else lowp::load_some<T, V>(x + row * cols + col, v[k], left);
  }
#pragma unroll
  for (int k = 0; k < kRowsPerWave; ++k) {
    const int64_t row = row0 + k * kGroup;
    if (row >= rows) break;                  // (whole rows of lanes leave together: the exchanges in encode() stay within one)
    const Coded q = encode<V>(v[k]);
    uint8_t* c = codes + (panel * rows + row) * (kPanel / 2) + in_row * (V / 2);
    if (V == 8) *reinterpret_cast<uint32_t*>(c) = q.code;
    else *reinterpret_cast<uint16_t*>(c) = static_cast<uint16_t>(q.code);
    if (in_row % (32 / V) == 0) scales[(panel * rows + row) * 8 + in_row / (32 / V)] = static_cast<uint8_t>(q.scale);
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
  uint32_t q[kRowsPerWave], scale[kRowsPerWave];
#pragma unroll
  for (int k = 0; k < kRowsPerWave; ++k) {
    const int64_t at = panel * rows + min(row0 + k * kGroup, rows - 1);
    const uint8_t* c = codes + at * (kPanel / 2) + in_row * (V / 2);
    q[k] = V == 8 ? *reinterpret_cast<const uint32_t*>(c) : *reinterpret_cast<const uint16_t*>(c);
    scale[k] = scales[at * 8 + in_row / (32 / V)];
  }
#pragma unroll
  for (int k = 0; k < kRowsPerWave; ++k) {
    const int64_t row = row0 + k * kGroup;
    if (row >= rows) break;
    const float unit = __uint_as_float(scale[k] << 23);
    float v[V];
    Float2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k], unit, 0);
    v[0] = p.x, v[1] = p.y;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k], unit, 1);
    v[2] = p.x, v[3] = p.y;
    if (V == 8) {
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k], unit, 2);
      v[V - 4] = p.x, v[V - 3] = p.y;
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k], unit, 3);
      v[V - 2] = p.x, v[V - 1] = p.y;
    }
    if (left == V) lowp::store<T, V>(x + row * cols + col, v);
    else lowp::store_some<T, V>(x + row * cols + col, v, left);
  }
}

// ---- the product.  v_mfma_scale_f32_*_f8f6f4 with both operands e2m1: a lane holds 32 consecutive values of one row of A (or B) - one block -
//      and that block's scale byte.  Which columns they are is free as long as A and B agree, so a lane takes neighbouring blocks of its row
//      for successive instructions: its codes are one contiguous piece of the panel and its scale bytes one aligned word, whose byte the
//      instruction selects.
struct Operand {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows;
};

__device__ __forceinline__ Int8 widen(Uint4 v) {
  return Int8{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
}

template <class T>
__device__ __forceinline__ float finish(float v, const T* bias, int64_t n, int relu) {
  if (bias) v += static_cast<float>(bias[n]);
  return relu && v < 0.0f ? 0.0f : v;      // (a NaN stays)
}

// Workgroup ids are dealt to the eight XCDs in turn, each with its own L2: give neighbouring tiles to one XCD.  (A remainder of ids keeps its
// place.)
__device__ __forceinline__ int by_xcd(int id, int total) {
  const int whole = total & ~7;
  return id < whole ? (id & 7) * (whole >> 3) + (id >> 3) : id;
}

typedef __attribute__((address_space(3))) void LdsVoid;

// A panel of a matrix as a buffer resource, and a request for 16 bytes a lane of it straight into LDS (lanes in order from ``lds``)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t panel_of(const uint8_t* base, int p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + static_cast<int64_t>(p) * bytes), 0, static_cast<int>(bytes), 0x00020000);
}
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t from, uint32_t at, uint8_t* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (LdsVoid*)lds, 16, static_cast<int>(at), 0, 0, 0);
}

// 16-byte chunk c of a 128-byte row r lies at chunk c ^ (r / 2 % 8): two rows fill the 64 banks, so the equal chunks of any sixteen neighbouring
// rows - what a 16-byte read serves at a time - are in sixteen different places
__device__ __forceinline__ int swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row >> 1 & 7)) << 4); }
// the chunk that lane ``lane`` of wave ``wave`` fetches so that it lands there (rows of a request: 8 * wave + lane / 8, plus multiples of 32)
__device__ __forceinline__ uint32_t staged_chunk(int wave, int lane) { return static_cast<uint32_t>((lane & 7) ^ ((4 * wave + (lane >> 4)) & 7)) << 4; }

// Where a workgroup stores its tile: a resource over the tile's real rows (row pitch ``pitch`` bytes), so that rows behind the last one are dropped by
// its range check; a column behind the last one is given kNowhere.
constexpr uint32_t kNowhere = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rows(void* base, int64_t m0, int64_t rows, int bm, int64_t pitch) {
  const int64_t bytes = min(static_cast<int64_t>(bm), rows - m0) * pitch;
  return __builtin_amdgcn_make_buffer_rsrc(static_cast<char*>(base) + m0 * pitch, 0, static_cast<int>(bytes), 0x00020000);
}
template <class T>
__device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t to, uint32_t at, float v) {
  if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), to, static_cast<int>(at), 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, static_cast<T>(v)), to, static_cast<int>(at), 0, 0);
}
// One 32 x 32 accumulator: lane l holds column l % 32, rows 8 (e / 4) + 4 (l / 32) + e % 4
template <class T>
__device__ __forceinline__ void put_tile(__amdgpu_buffer_rsrc_t to, const Float16& acc, int row, int half, int64_t col, int64_t cols, float bias, int relu) {
  const uint32_t pitch = static_cast<uint32_t>(cols * sizeof(T)), at = col < cols ? static_cast<uint32_t>(row + 4 * half) * pitch + static_cast<uint32_t>(col * sizeof(T)) : kNowhere;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float v = acc[e] + bias;
    if (relu && v < 0.0f) v = 0.0f;                    // (a NaN stays)
    put<T>(to, at == kNowhere ? at : at + (8 * (e / 4) + e % 4) * pitch, v);
  }
}

// Few rows of x: bound by reading W once.  16 rows of W (A) x 16 * MT rows of x (B) a workgroup on 16x16x128 instructions, operands straight
// from memory to registers (a panel's 16 rows are 2 KB in one piece); the waves share the panels out and join their sums in LDS, in order.
// RAW: x comes as values (few of them: thin_raw); every workgroup quantises them for itself into LDS while its first piece of W is on its way - a second
// reading of x from the L2 for every 16 rows of W, against a launch of its own: one row of 25088 x 4096 18.1 -> 15.3 us, of 4096 x 1000 12.1 -> 9.9.
template <int V>
constexpr int kThinBatch = V == 4 ? 7 : 4;             // pieces of a panel's row (two rows, 16-bit) that a wave has on their way together
template <class T, int MT, bool RAW>
__global__ __launch_bounds__(512) void mx4_linear_thin(Operand x, const T* __restrict__ values, int64_t cols, Operand w, const T* __restrict__ bias, T* __restrict__ y,
                                                       int panels, int relu) {
  extern __shared__ __attribute__((aligned(16))) uint8_t s_thin[];     // sums [wave][MT][4][64]; RAW: codes [panel][row][128], scales [panel][row][8]
  float* s_sum = reinterpret_cast<float*>(s_thin);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, quarter = lane >> 4;
  uint8_t* s_codes = s_thin + waves * MT * 1024;
  uint8_t* s_scales = s_codes + panels * static_cast<int>(RAW ? x.rows : 0) * 128;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const int64_t n = min(n0 + (lane & 15), w.rows - 1);                 // rows behind the last one are computed, not stored
  int64_t m[MT];
  Float4 acc[MT] = {};
#pragma unroll
  for (int i = 0; i < MT; ++i) m[i] = min(m0 + 16 * i + (lane & 15), x.rows - 1);
  constexpr int U = 2;                                                 // panels whose operands are on their way together (4: 5.9 us for 4.3 with 4096 x 4096)
  Uint4 a[U][2];
  uint32_t sa[U];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t p = min(p0 + u * waves, panels - 1);
      const Uint4* at = reinterpret_cast<const Uint4*>(w.codes + (p * w.rows + n) * 128 + quarter * 32);
      a[u][0] = at[0], a[u][1] = at[1];
      sa[u] = *reinterpret_cast<const uint16_t*>(w.scales + (p * w.rows + n) * 8 + quarter * 2);
    }
  };
  fetch(wave);
  if constexpr (RAW) {
    constexpr int V = 16 / sizeof(T), kLanes = kPanel / V, kGroup = 64 / kLanes;      // lanes a panel's row, rows a wave takes at once
    constexpr int kBatch = kThinBatch<V>;
    const int pieces = panels * static_cast<int>(x.rows), rows = static_cast<int>(x.rows), in_row = lane % kLanes, step = waves * kGroup;
    for (int i0 = wave * kGroup + lane / kLanes; i0 < pieces; i0 += kBatch * step) {
      float v[kBatch][V];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = min(i0 + k * step, pieces - 1), p = i / rows, row = i - p * rows;
        const int64_t col = static_cast<int64_t>(p) * kPanel + in_row * V;
        const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(V), cols - col)));
        if (left == V) lowp::load<T, V, false>(values + row * cols + col, v[k]);
        else lowp::load_some<T, V>(values + row * cols + col, v[k], left);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = i0 + k * step;
        if (i >= pieces) break;                                        // (whole rows of lanes leave together)
        const Coded q = encode<V>(v[k]);
        if (V == 8) *reinterpret_cast<uint32_t*>(s_codes + i * 128 + in_row * 4) = q.code;
        else *reinterpret_cast<uint16_t*>(s_codes + i * 128 + in_row * 2) = static_cast<uint16_t>(q.code);
        if (in_row % (32 / V) == 0) s_scales[i * 8 + in_row / (32 / V)] = static_cast<uint8_t>(q.scale);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");    // (__syncthreads would also wait for W)
  }
  for (int p0 = wave; p0 < panels;) {
    Uint4 b[U][MT][2];
    uint32_t sb[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t p = min(p0 + u * waves, panels - 1);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int64_t row = p * x.rows + m[i];
        const Uint4* bt = reinterpret_cast<const Uint4*>((RAW ? s_codes : x.codes) + row * 128 + quarter * 32);
        b[u][i][0] = bt[0], b[u][i][1] = bt[1];
        sb[u][i] = *reinterpret_cast<const uint16_t*>((RAW ? s_scales : x.scales) + row * 8 + quarter * 2);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + u * waves < panels) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(a[u][0]), widen(b[u][i][0]), acc[i], 4, 4, 0, static_cast<int>(sa[u]), 0,
                                                                    static_cast<int>(sb[u][i]));
          acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(a[u][1]), widen(b[u][i][1]), acc[i], 4, 4, 1, static_cast<int>(sa[u]), 1,
                                                                    static_cast<int>(sb[u][i]));
        }
      }
    }
    p0 += waves * U;
    if (p0 < panels) fetch(p0);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s_sum[((wave * MT + i) * 4 + e) * 64 + lane] = acc[i][e];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 256; o += blockDim.x) {           // (m, n) of the tile, n fastest; a lane held row n = 4 (lane / 16) + e, column m = lane % 16
    const int i = o >> 8, mm = (o >> 4) & 15, nn = o & 15;
    const int at = (i * 4 + (nn & 3)) * 64 + (nn >> 2) * 16 + mm;
    float v = s_sum[at];
    for (int k = 1; k < waves; ++k) v += s_sum[k * MT * 256 + at];
    if (m0 + 16 * i + mm < x.rows && n0 + nn < w.rows) y[(m0 + 16 * i + mm) * w.rows + n0 + nn] = static_cast<T>(finish<T>(v, bias, n0 + nn, relu));
  }
}

template <int SEL>
__device__ __forceinline__ Float16 mfma(Uint4 a, Uint4 b, Float16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(a), widen(b), c, 4, 4, SEL, static_cast<int>(sa), SEL, static_cast<int>(sb));
}

// Many rows: BM x BN of y a workgroup of four waves (2 x 2, or side by side over 32 rows), 32x32x64 instructions; panels go to LDS by direct copies,
// two (256 x 256) or three buffers, one barrier a panel.  A panel is four steps of 64 columns; the operands of a step are read while the step before is
// multiplied, and the barrier stands before a panel's last step, whose operands are in registers by then - its products cover the first reads of the next
// panel.  4096 x 25088 x 4096: 178 us in a kernel trace (median of 12, least 175): 4.7 PFLOP/s of the 7.0 - 7.6 that the bare instruction reaches, the matrix
// pipe 0.76 busy; among other calls 166, the call's time less the quantisation's.  The smaller tiles are bound by how long a panel takes to come: with the
// third buffer 128 x 4096 x 4104 takes 15.1 us for 17.9, 32 x 25088 x 4096 17.5 for 19.7 (calls).
template <int BM, int BN>
constexpr int kTileStages = BM > 128 ? 2 : 3;
template <int BM, int BN>
constexpr int kTileStage = (BM + BN) * 128 + ((BM > 128 ? BM : 128) + BN) * 8;      // (x's scale bytes come 1 KB at a time)

template <class T, int BM, int BN>
__global__ __launch_bounds__(kBlock, BM < 128 ? 2 : 1) void mx4_linear_tile(Operand x, Operand w, const T* __restrict__ bias, T* __restrict__ y,
                                                                               float* __restrict__ partial, int panels, int splits, int relu) {
  constexpr int WM = BM == 32 ? 1 : 2, WN = 4 / WM, TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int kStage = kTileStage<BM, BN>, kScales = (BM + BN) * 128, kRowsX = BM > 128 ? BM : 128;
  constexpr int kStages = kTileStages<BM, BN>;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_tile[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int tm = static_cast<int>((x.rows + BM - 1) / BM), tn = static_cast<int>((w.rows + BN - 1) / BN);
  int id = by_xcd(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
  const int part = id / (tm * tn);
  id -= part * tm * tn;
  const int group = 4 * tn, first = id / group * 4, high = min(4, tm - first);      // four rows of tiles at a time: both operands stay in the L2
  const int64_t m0 = static_cast<int64_t>(first + id % group % high) * BM, n0 = static_cast<int64_t>(id % group / high) * BN;
  const int begin = static_cast<int>(static_cast<int64_t>(part) * panels / splits), end = static_cast<int>(static_cast<int64_t>(part + 1) * panels / splits);

  uint32_t at_x[BM / 32], at_w[BN / 32];
  const uint32_t chunk = staged_chunk(wave, lane);
#pragma unroll
  for (int j = 0; j < BM / 32; ++j) at_x[j] = static_cast<uint32_t>(min(m0 + j * 32 + wave * 8 + (lane >> 3), x.rows - 1)) * 128u + chunk;
#pragma unroll
  for (int j = 0; j < BN / 32; ++j) at_w[j] = static_cast<uint32_t>(min(n0 + j * 32 + wave * 8 + (lane >> 3), w.rows - 1)) * 128u + chunk;
  const uint32_t x_bytes = static_cast<uint32_t>(x.rows) * 128u, w_bytes = static_cast<uint32_t>(w.rows) * 128u;
  const int wm = wave / WN * (TM * 32), wn = wave % WN * (TN * 32);
  int frag[4];                                         // this lane's chunk of a row in each of the four steps
#pragma unroll
  for (int k = 0; k < 4; ++k) frag[k] = swizzled(lane & 31, half * 4 + k);

  // the tile's scale bytes of a panel are one piece of BM (BN) * 8 bytes: 1 KB a wave (128 x 128 tiles have two: two waves copy each)
  const int piece = wave % ((kRowsX + BN) / 128);
  const bool for_x = piece < kRowsX / 128;
  const uint32_t at_scale = static_cast<uint32_t>((for_x ? m0 + piece * 128 : n0 + (piece - kRowsX / 128) * 128) * 8) + lane * 16;
  const int to_scale = kScales + piece * 1024;
  const uint8_t* scales = for_x ? x.scales : w.scales;
  const uint32_t scale_bytes = (for_x ? x_bytes : w_bytes) >> 4;
  // copy k of a panel: 32 rows of x's (W's) tile, 8 of them a wave
  constexpr int kX = BM / 32, kW = BN / 32;
  uint8_t* const to_x = s_tile + wave * 1024;
  uint8_t* const to_w = s_tile + BM * 128 + wave * 1024;
  auto copy_scales = [&](int p, int buf) { copy16(panel_of(scales, p, scale_bytes), at_scale, s_tile + buf * kStage + to_scale); };
  auto request_x = [&](int p, int buf) {
    const __amdgpu_buffer_rsrc_t r = panel_of(x.codes, p, x_bytes);
#pragma unroll
    for (int k = 0; k < kX; ++k) copy16(r, at_x[k], to_x + buf * kStage + k * 4096);
  };
  auto request_w = [&](int p, int buf) {
    const __amdgpu_buffer_rsrc_t r = panel_of(w.codes, p, w_bytes);
#pragma unroll
    for (int k = 0; k < kW; ++k) copy16(r, at_w[k], to_w + buf * kStage + k * 4096);
    copy_scales(p, buf);
  };
  Uint4 fa[2][TM], fb[2][TN];
  // operand piece i of step k
  auto read = [&](int buf, int k, int to, int i) {
    if (i < TM) fa[to][i] = *reinterpret_cast<const Uint4*>(s_tile + buf * kStage + wm * 128 + frag[k] + i * 4096);
    else fb[to][i - TM] = *reinterpret_cast<const Uint4*>(s_tile + buf * kStage + (BM + wn) * 128 + frag[k] + (i - TM) * 4096);
  };
  uint32_t sx[2][TM], sw[2][TN];
  auto scale_words = [&](int buf, int to) {
    const uint8_t* a = s_tile + buf * kStage + kScales + (wm + (lane & 31)) * 8 + half * 4;
    const uint8_t* b = s_tile + buf * kStage + kScales + (kRowsX + wn + (lane & 31)) * 8 + half * 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[to][i] = *reinterpret_cast<const uint32_t*>(a + i * 256);
#pragma unroll
    for (int j = 0; j < TN; ++j) sw[to][j] = *reinterpret_cast<const uint32_t*>(b + j * 256);
  };
  Float16 acc[TM][TN] = {};
  // One step's products, ALSO behind product k.  A wave issues in order, a product holds the next one back for its 32 cycles, and a copy or a read
  // that the memory pipes cannot take yet holds back everything behind it: what a step has to ask for goes one by one between its products.
#define MX4_STEP(SEL, FROM, ALSO)                                                                       \
  _Pragma("unroll") for (int k = 0; k < TM * TN; ++k) {                                                \
    acc[k / TN][k % TN] = mfma<SEL>(fa[FROM][k / TN], fb[FROM][k % TN], acc[k / TN][k % TN], sx[0][k / TN], sw[0][k % TN]); \
    ALSO;                                                                                              \
    __builtin_amdgcn_sched_barrier(0);                                                                 \
  }
  // behind the even products a piece of the next step's operands, behind the odd ones a copy (all of them, should there be fewer products)
#define READ_NEXT(STEP, TO)                                                                             \
  _Pragma("unroll") for (int i = 0; i < kReads; ++i)                                                   \
      if (TM * TN >= 2 * kReads ? i * 2 == k : i * TM * TN / kReads == k) read(buf, STEP, TO, i)
#define COPY_BETWEEN(COUNT, FROM, AT, TO, BUF)                                                          \
  _Pragma("unroll") for (int i = 0; i < COUNT; ++i)                                                    \
      if (TM * TN >= 2 * COUNT ? i * 2 + 1 == k : i * TM * TN / COUNT == k) copy16(FROM, AT[i], TO + (BUF) * kStage + i * 4096)
  constexpr int kReads = TM + TN;
  // (the tail's requests beyond the last panel ask for that one again, into buffers nobody reads: one loop body, no branches)
  const int last = end - 1;
  constexpr int kAhead = (kStages - 2) * (kX + kW + 1);      // a wave's copies of the panels behind the next one: not waited for
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    request_x(min(begin + s, last), s);
    request_w(min(begin + s, last), s);
    __builtin_amdgcn_sched_barrier(0);
  }
  request_x(min(begin + kStages - 1, last), kStages - 1);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kAhead + kX) : "memory");
#pragma unroll
  for (int i = 0; i < kReads; ++i) read(0, 0, 0, i);
  scale_words(0, 0);
  int buf = 0, free = kStages - 1;                     // this panel's buffer, the one of the panel before
  for (int p = begin; p < end; ++p) {
    // x's part of the panel kStages - 1 further on was asked for in the last step of the one before, W's part is in this step: the copies come evenly
    const __amdgpu_buffer_rsrc_t rw = panel_of(w.codes, min(p + kStages - 1, last), w_bytes), rx = panel_of(x.codes, min(p + kStages, last), x_bytes);
    MX4_STEP(0, 0, {
      READ_NEXT(1, 1);
      COPY_BETWEEN(kW, rw, at_w, to_w, free);
      if (k == TM * TN - 1) copy_scales(min(p + kStages - 1, last), free);
    });
    MX4_STEP(1, 1, { READ_NEXT(2, 0); });
    MX4_STEP(2, 0, { READ_NEXT(3, 1); });
    // every wave has this panel's operands in registers, and its copies of the next panel have landed
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kAhead) : "memory");
    __builtin_amdgcn_sched_barrier(0);
    free = buf;
    buf = buf == kStages - 1 ? 0 : buf + 1;
    MX4_STEP(3, 1, {
      if (k == 0) scale_words(buf, 1);
      READ_NEXT(0, 0);
      COPY_BETWEEN(kX, rx, at_x, to_x, free);
    });
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[0][i] = sx[1][i];
#pragma unroll
    for (int j = 0; j < TN; ++j) sw[0][j] = sw[1][j];
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // no copy may land in an LDS that is another workgroup's by then
#undef MX4_STEP
#undef READ_NEXT
#undef COPY_BETWEEN
  float* to = partial + static_cast<int64_t>(part) * x.rows * w.rows;
  const __amdgpu_buffer_rsrc_t out = splits > 1 ? tile_rows(to, m0, x.rows, BM, w.rows * 4) : tile_rows(y, m0, x.rows, BM, w.rows * static_cast<int64_t>(sizeof(T)));
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int64_t n = n0 + wn + j * 32 + (lane & 31);
    const float b = bias && splits == 1 ? static_cast<float>(bias[min(n, w.rows - 1)]) : 0.0f;
    if (splits > 1) {
#pragma unroll
      for (int i = 0; i < TM; ++i) put_tile<float>(out, acc[i][j], wm + i * 32, half, n, w.rows, 0.0f, 0);
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) put_tile<T>(out, acc[i][j], wm + i * 32, half, n, w.rows, b, relu);
    }
  }
}

// y = relu?(part 0 + part 1 + ... + bias), in that order; four elements a thread.  Five parts of 301 x 2048: 5 us, latency (12 MB, from the caches)
template <class T>
__global__ __launch_bounds__(kBlock) void mx4_join(const float* __restrict__ partial, const T* __restrict__ bias, T* __restrict__ y, int64_t n, int64_t cols,
                                                   int parts, int relu) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * 4;
  const int left = static_cast<int>(min(static_cast<int64_t>(4), n - i));
  if (left <= 0) return;
  float v[4];
  if (left == 4) {
    lowp::load<float, 4, false>(partial + i, v);
    for (int k = 1; k < parts; ++k) {
      float p[4];
      lowp::load<float, 4, false>(partial + k * n + i, p);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += p[j];
    }
  } else {
    lowp::load_some<float, 4>(partial + i, v, left);
    for (int k = 1; k < parts; ++k) {
      float p[4];
      lowp::load_some<float, 4>(partial + k * n + i, p, left);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += p[j];
    }
  }
  int64_t c = bias ? static_cast<int64_t>(static_cast<uint32_t>(i) % static_cast<uint32_t>(cols)) : 0;      // (a result in parts has at most 2^24 elements: plan_linear, plan_dgrad)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j >= left) break;
    float t = v[j];
    if (bias) {
      t += static_cast<float>(bias[c]);
      c = c + 1 == cols ? 0 : c + 1;
    }
    y[i + j] = static_cast<T>(relu && t < 0.0f ? 0.0f : t);      // (a NaN stays)
  }
}

// ---- the input gradient.  First gy, 0 where the ReLU stopped it, becomes planes of bfloat16 terms [term][row][n padded to 128] - once, not in
//      every workgroup that needs it.  Then a workgroup owns BM rows x one panel of gx and walks W's rows 32 at a time: their codes become
//      bfloat16 values in LDS, turned so that a lane's eight values along the contraction are 16 bytes; the terms are copied there.
constexpr int kChunk = 32;

template <class T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kTerms<__bf16> = 1;

// v as the sum of N bfloat16, exact but for bits under 2^-133 (cut, not rounded: what is left always fits the next ones, and a finite v stays finite)
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

// a thread: eight consecutive n of a row.  512 x 2048 float32: 7 us, latency (4 MB in, 6 MB out)
template <class T>
__global__ __launch_bounds__(kBlock) void mx4_grad_terms(const T* __restrict__ gy, const T* __restrict__ mask, uint8_t* __restrict__ planes, int64_t rows, int64_t n,
                                                         int64_t padded) {
  constexpr int N = kTerms<T>;
  const int64_t per_row = padded / 8, unit = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kBlock + threadIdx.x;
  if (unit >= rows * per_row) return;
  const int64_t m = unit / per_row, c = (unit - m * per_row) * 8;
  const int left = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(8), n - c)));
  float g[8], o[8];
  lowp::load_eight<T>(gy + m * n + c, g, left);
  if (mask) {
    lowp::load_eight<T>(mask + m * n + c, o, left);
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = o[k] <= 0.0f ? 0.0f : g[k];
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
  for (int s = 0; s < N; ++s) *reinterpret_cast<Uint4*>(planes + ((s * rows + m) * padded + c) * 2) = out[s];
}

// LDS places of a stage.  Terms: rows of 64 bytes (32 of the contraction); four of them fill the banks, so chunk c of row r lies at c ^ (r / 4 % 4).
// W: rows (n) of 512 bytes (a panel's 256 columns), in units of 16 bytes; what is written together - two rows, eight blocks of columns, the same unit
// of each - and what a transposing read takes together - four rows, four neighbouring units - must lie in different banks.  (By sixteen lanes they do;
// the counters still show a third of the LDS cycles of 64-row tiles in bank conflicts, which this does not explain.)
__device__ __forceinline__ int short_row(int row, int chunk) { return row * 64 + ((chunk ^ (row >> 2 & 3)) << 4); }
__device__ __forceinline__ int wide_row(int row, int unit) { return row * 512 + ((unit ^ (row & 3) << 2 ^ (unit >> 4 & 1) ^ (row & 1) << 1) << 4); }

// ds_read_b64_tr_b16: sixteen lanes read 8 bytes each - lane 4r + s four columns of row r - and lane i gets column i of the four rows
typedef __bf16 Bf16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Bf16x4 read_turned(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) Bf16x4*)p);
}

template <int N, int BM>
constexpr int kGradLds = 2 * (kPanel + N * BM) * 64;

// Everything is doubled: while chunk c is multiplied, chunk c + 1 of W is taken from registers to LDS, the copies of its terms land, and the next kHeld
// chunks of W are on their way to registers (one 16-byte and one byte load a thread and chunk: what a load instruction costs hardly depends on its
// width).  One barrier a chunk.  The matrix instruction wants eight n of one column in a lane; the codes come along the columns: they are stored as
// bfloat16 rows and turned by the transposing LDS read.  512 x 2048 to 25088 columns: 132 us in float32 in a kernel trace (median of 12, least 129; three
// terms: 1.2 PFLOP/s; the matrix pipe of a busy CU 0.78 busy, 392 workgroups on 512 places); among other calls 118, the call's time less the terms'.
// 37 x 4096 bfloat16: 22 us, bound by W's conversion.
constexpr int kHeld = 4;
template <class T, int BM>
__global__ __launch_bounds__(kBlock, BM == 128 ? 2 : 3) void mx4_dgrad(const uint8_t* __restrict__ planes, Operand w, T* __restrict__ gx, float* __restrict__ partial,
                                                                      int64_t rows, int64_t cols, int64_t padded, int splits) {
  constexpr int N = kTerms<T>, WM = BM == 128 ? 2 : 1, WK = 4 / WM, TI = BM / WM / 32, TJ = kPanel / WK / 32;
  constexpr int kCopies = BM >= 64 ? BM / 64 : 1, kTermBytes = BM * 64;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_grad[];      // [2][column][64 bytes], [2][term][row][64 bytes]
  uint8_t* s_g = s_grad + 2 * kPanel * 64;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = lane >> 5;
  const int tiles_m = static_cast<int>((rows + BM - 1) / BM), panels = static_cast<int>(panels_of(cols));
  int id = by_xcd(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
  const int part = id / (tiles_m * panels);
  id -= part * tiles_m * panels;
  const int64_t panel = id / tiles_m, m0 = static_cast<int64_t>(id % tiles_m) * BM, nw = w.rows;
  const int fours = static_cast<int>(padded / (kHeld * kChunk));
  const int begin = static_cast<int>(static_cast<int64_t>(part) * fours / splits) * kHeld, end = static_cast<int>(static_cast<int64_t>(part + 1) * fours / splits) * kHeld;
  const int last = end - 1;
  const int wm = wave / WK * (TI * 32), wk = wave % WK * (TJ * 32);

  // a copy request is 16 rows of 64 bytes a wave (with 32 rows two waves ask for each)
  uint32_t at[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int row = j * 64 + (BM >= 64 ? wave : wave & 1) * 16 + (lane >> 2);
    at[j] = static_cast<uint32_t>(min(static_cast<int64_t>(row), rows - 1 - m0) * padded * 2) + (static_cast<uint32_t>((lane & 3) ^ (row >> 2 & 3)) << 4);
  }
  const uint8_t* plane0 = planes + m0 * padded * 2;
  const uint32_t tile_bytes = static_cast<uint32_t>(min(static_cast<int64_t>(BM), rows - m0) * padded * 2);
  auto copy = [&](int c, int buf, int e) {             // copy e of a chunk: kCopies of each term
    const int s = e / kCopies, j = e % kCopies;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(plane0 + s * rows * padded * 2 + static_cast<int64_t>(c) * (kChunk * 2)), 0,
                                                                       static_cast<int>(tile_bytes - static_cast<uint32_t>(c) * (kChunk * 2)), 0x00020000);
    copy16(r, at[j], s_g + (buf * N + s) * kTermBytes + j * 4096 + (BM >= 64 ? wave : wave & 1) * 1024);
  };

  // 32 columns - one block - of one row of W a thread; rows behind the last one read as zeros (the resource ends there): the value 0 under the scale 2^-127
  struct Held {
    Uint4 code;
    uint32_t scale;
  };
  const uint8_t* codes = w.codes + panel * nw * 128;
  const uint8_t* scales = w.scales + panel * nw * 8;
  const int slab = static_cast<int>(nw);
  auto fetch = [&](int c, Held& h) {
    const uint32_t left = max(slab - c * kChunk, 0);
    const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(codes + static_cast<int64_t>(c) * (kChunk * 128)), 0, static_cast<int>(left * 128u), 0x00020000);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(scales + static_cast<int64_t>(c) * (kChunk * 8)), 0, static_cast<int>(left * 8u), 0x00020000);
    h.code = __builtin_bit_cast(Uint4, __builtin_amdgcn_raw_buffer_load_b128(rc, t * 16, 0, 0));
    h.scale = __builtin_amdgcn_raw_buffer_load_b8(rs, t, 0, 0);
  };
  const uint32_t put_at = static_cast<uint32_t>(wide_row(t >> 3, (t & 7) * 4));
  auto turn = [&](const Held& h, int buf, int k) {     // a quarter of it: eight columns
    const float f = __uint_as_float(h.scale << 23);
    {
      Uint4 out;
      out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(h.code[k], f, 0));
      out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(h.code[k], f, 1));
      out[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(h.code[k], f, 2));
      out[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(h.code[k], f, 3));
      *reinterpret_cast<Uint4*>(s_grad + (put_at ^ static_cast<uint32_t>(k << 4)) + buf * (kPanel * 64)) = out;
    }
  };
  Float16 acc[TI][TJ] = {};
  const uint8_t* const read_g = s_g + wm * 64;
  const uint32_t place_g = static_cast<uint32_t>(short_row(lane & 31, half));
  uint32_t place_w[TJ];                                // lane 16g + 4r + s: row r (+ 8 for the upper half of the wave), columns 16 (g % 2) + 4s ..
#pragma unroll
  for (int j = 0; j < TJ; ++j)
    place_w[j] = static_cast<uint32_t>(half * 4096 + wide_row(lane >> 2 & 3, (wk + j * 32) / 8 + (lane >> 4 & 1) * 2 + (lane >> 1 & 1)) + (lane & 1) * 8);
  constexpr int K = kChunk / 16;                       // 16 of the contraction a matrix instruction: lane half h has eight, 16k + 8h ..
  auto read = [&](int buf, Bf16x8 (&b)[K][TJ]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const uint8_t* p = s_grad + place_w[j] + buf * (kPanel * 64) + k * 8192;
        b[k][j] = __builtin_shufflevector(read_turned(p), read_turned(p + 2048), 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  };
  constexpr int kFrags = K * N * TI;                   // gy's operands of a chunk, in order of use: k, term, row block
  auto frag = [&](int buf, int e) {
    const int k = e / (N * TI), s = e / TI % N, i = e % TI;
    return *reinterpret_cast<const Bf16x8*>(read_g + (place_g ^ static_cast<uint32_t>(k * 32)) + (buf * N + s) * kTermBytes + i * 2048);
  };

  Held held[kHeld];                                    // chunk c is in held[c % kHeld]
#pragma unroll
  for (int e = 0; e < N * kCopies; ++e) copy(begin, 0, e);
  __builtin_amdgcn_sched_barrier(0);                   // (the copies must be older than the two loads that step() leaves on their way)
#pragma unroll
  for (int k = 0; k < kHeld; ++k) fetch(min(begin + k, last), held[k]);
#pragma unroll
  for (int k = 0; k < 4; ++k) turn(held[0], 0, k);
  fetch(min(begin + kHeld, last), held[0]);
  // h: holds chunk c + 1, is given chunk c + 1 + kHeld.  Everything a step asks for or converts goes between its products, in a fixed order: gy's
  // operands two groups of products ahead, then the copies, then the four quarters of the next chunk of W, then its loads.
  constexpr int kExtras = N * kCopies + 5;
  auto step = [&](int c, Held& h, int buf) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // chunk c's copies have landed: only the two loads of chunk c + kHeld came after
    Bf16x8 b[K][TJ], g[kFrags];
    read(buf, b);                                      // before the next copies are asked for: the compiler takes a turned read to depend on every copy on its way
    g[0] = frag(buf, 0);
    if (kFrags > 1) g[1] = frag(buf, 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < kFrags; ++e) {
      if (e + 2 < kFrags) g[e + 2] = frag(buf, e + 2);
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[e % TI][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(g[e], b[e / (N * TI)][j], acc[e % TI][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < kExtras; ++x) {
        if (x * kFrags / kExtras != e) continue;
        if (x < N * kCopies) copy(min(c + 1, last), buf ^ 1, x);
        else if (x < N * kCopies + 4) turn(h, buf ^ 1, x - N * kCopies);
        else fetch(min(c + 1 + kHeld, last), h);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  for (int c = begin; c < end; c += kHeld) {           // (chunks come in fours: the planes are padded to them)
#pragma unroll
    for (int k = 0; k < kHeld; ++k) step(c + k, held[(k + 1) % kHeld], k & 1);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // no copy may land in an LDS that is another workgroup's by then
  float* to = partial + static_cast<int64_t>(part) * rows * cols;
  const __amdgpu_buffer_rsrc_t out = splits > 1 ? tile_rows(to, m0, rows, BM, cols * 4) : tile_rows(gx, m0, rows, BM, cols * static_cast<int64_t>(sizeof(T)));
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    const int64_t col = panel * kPanel + wk + j * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      if (splits > 1) put_tile<float>(out, acc[i][j], wm + i * 32, half, col, cols, 0.0f, 0);
      else put_tile<T>(out, acc[i][j], wm + i * 32, half, col, cols, 0.0f, 0);
    }
  }
}

// sizes: every product of two of them fits an int64, every grid dimension its limit
constexpr int64_t kMostRows = int64_t{1} << 20, kMostCols = int64_t{1} << 20;      // 256 rows of a result: at most 2^30 bytes

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
constexpr int64_t kAlign = 256;
int64_t padded(int64_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }

// How a product is cut.
//   thin   one launch, but every 16 rows of W read all of x again: up to 16 rows of up to 56 panels (8 rows of 8192 x 4096: 7.7 against 9.2 us, of
//          12544 x 2048 9.3 against 9.5, of 25088 x 4096 17.0 against 13.9), a single row of up to 112, which is quantised in there (25088: 15.5 against
//          17.5), and up to 64 rows of 1024 panels together under a small weight (32 of 6400 x 1024: 7.6 against 7.7, 64 of them 11.4 against 8.6).
//   big    256 x 256 tiles, whole or with their panels dealt to two workgroups, or 128 x 128, of which 64 or 32 rows where x has no more: what is estimated
//          to take less.  A round of 256 workgroups takes, for each panel, 0.94 - 1.68 us (big; more once they crowd) or 0.27 - 0.55 (128 rows), and 11.5
//          or 5.1 us for its start and end; a part 1.2 us per million sums to join.  x quantised before, bfloat16, 25088 -> 4096: 2048 rows big in two parts
//          113 us, whole 132, 128 rows 117; 2049 to 4096 rows big 131 .. 178, 128 rows 156 .. 241, in two parts 166 .. 219; 4097 rows 128 rows 270,
//          big 283; 1500 rows big in two parts 95, 128 rows 105.  4096 -> 4096: 2048 rows 128 rows 28, big 33, in two parts 43.  Up to 128 rows of x never
//          fill half of a big tile: 20 of 25088 -> 32768 take 70 us in tiles of 32 rows, 153 (in two parts 109) in big ones, 128 of them 83 and 156.
//   splits the panels are dealt to several workgroups a tile where tiles alone do not fill the chip: the number with the least estimated time, from
//          what a panel takes (128 rows: 0.26 us up to 64 workgroups, 0.45 at one a CU; fewer rows 0.14 and 0.33), three panels' time for a workgroup's
//          start and end, and the joining pass.  Fitted to 8 .. 512 rows of nine weights.
struct LinearPlan {
  int thin, big, splits;
};
// us for ``groups`` workgroups of ``panels`` panels each, a panel taking ``first`` us + ``more`` for every workgroup at work, + ``crowd`` for each beyond 144
double estimate_rounds(int64_t groups, int64_t panels, double first, double more, double crowd, double ends) {
  auto round = [&](int64_t at_work) {
    return ends + static_cast<double>(panels) * (first + more * static_cast<double>(at_work) + crowd * static_cast<double>(at_work > 144 ? at_work - 144 : 0));
  };
  return static_cast<double>(groups / 256) * round(256) + (groups % 256 ? round(groups % 256) : 0.0);
}
double estimate_join(int64_t m, int64_t n, int64_t splits) { return splits > 1 ? 1.0 + 1.2e-6 * static_cast<double>(splits * m * n) : 0.0; }
LinearPlan plan_linear(int64_t m, int64_t n, int64_t k) {
  const int64_t panels = panels_of(k);
  if (m * panels <= 112 || (m <= 16 ? panels <= 56 : m <= 64 && m * panels <= 1024 && n <= 4096)) return {1, 0, 1};
  const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), small = ((m + 127) / 128) * ((n + 127) / 128);
  int best = 1;
  double least = 0.0;
  for (int64_t s = 1; s <= 32 && (s == 1 || (s <= panels / 4 && small <= 1024)); ++s) {
    const int64_t groups = small * s;
    const double panel = (m <= 64 ? 0.14 : 0.26) + 0.001 * static_cast<double>(groups <= 64 ? 0 : (groups < 256 ? groups - 64 : 192));
    const double t = panel * static_cast<double>(((panels + s - 1) / s + 3) * ((groups + 255) / 256)) + estimate_join(m, n, s);
    if (s == 1 || t < least) best = static_cast<int>(s), least = t;
  }
  if (m <= 128) return {0, 0, best};
  const double with_small = estimate_rounds(small * best, (panels + best - 1) / best, 0.27, 0.00108, 0.0, 5.1) + estimate_join(m, n, best);
  auto with_big = [&](int64_t s) { return estimate_rounds(big * s, (panels + s - 1) / s, 0.93, 0.002, 0.0021, 11.5) + estimate_join(m, n, s); };
  const int parts = panels >= 8 && big <= 256 && with_big(2) < with_big(1) ? 2 : 1;
  return with_small < 0.97 * with_big(parts) ? LinearPlan{0, 0, best} : LinearPlan{0, 1, parts};      // (the estimates are good to a few per cent)
}
int64_t linear_partial_bytes(int64_t m, int64_t n, int64_t k) {
  const LinearPlan p = plan_linear(m, n, k);
  return p.splits > 1 ? padded(4LL * p.splits * m * n) : 0;
}

template <class T>
void run_join(const float* partial, const void* bias, void* y, int64_t rows, int64_t cols, int parts, int relu, hipStream_t st) {
  const int64_t n = rows * cols, blocks = (n + 4 * kBlock - 1) / (4 * kBlock);
  mx4_join<T><<<dim3(static_cast<unsigned>(blocks)), kBlock, 0, st>>>(partial, static_cast<const T*>(bias), static_cast<T*>(y), n, cols, parts,
                                                                                         relu);
}

int thin_waves(int64_t panels) { return panels >= 16 ? 8 : (panels >= 4 ? 4 : 1); }
// x is quantised inside the thin product where its values come in two rounds of loads or less - another round costs what the launch does that it saves
// (float32, one round: a row of 4096 4.5 against 6.3 us; two: a row of 25088 15.5 against 17.6, 4 rows of 4096 6.8 against 7.0; three: 4 rows of 8192
// 11.9 against 10.4)
bool thin_raw(int64_t m, int64_t k, int bytes) {
  const int64_t panels = panels_of(k);
  return m <= 16 && m * panels <= 2 * thin_waves(panels) * (bytes == 4 ? kThinBatch<4> : 2 * kThinBatch<8>);
}

template <class T, int MT, bool RAW>
int run_thin(Operand x, const void* values, int64_t k, Operand w, const void* bias, void* y, int relu, hipStream_t st) {
  const int panels = static_cast<int>(panels_of(k)), waves = thin_waves(panels);
  const int lds = waves * MT * 1024 + (RAW ? panels * static_cast<int>(x.rows) * 136 : 0);
  const dim3 grid(static_cast<unsigned>((w.rows + 15) / 16), static_cast<unsigned>((x.rows + 16 * MT - 1) / (16 * MT)));
  mx4_linear_thin<T, MT, RAW><<<grid, waves * 64, lds, st>>>(x, static_cast<const T*>(values), k, w, static_cast<const T*>(bias), static_cast<T*>(y), panels, relu);
  return adv_internal_finish_launch();
}

template <class T, int BM, int BN>
int run_tile(Operand x, Operand w, const void* bias, void* y, float* partial, int panels, int splits, int relu, hipStream_t st) {
  const int64_t tiles = ((x.rows + BM - 1) / BM) * ((w.rows + BN - 1) / BN) * splits;
  if (!adv_internal_lds_limit<mx4_linear_tile<T, BM, BN>>(kTileStages<BM, BN> * kTileStage<BM, BN>)) return ADV_ELAUNCH;
  mx4_linear_tile<T, BM, BN><<<dim3(static_cast<unsigned>(tiles)), kBlock, kTileStages<BM, BN> * kTileStage<BM, BN>, st>>>(x, w, static_cast<const T*>(bias), static_cast<T*>(y), partial, panels,
                                                                                                  splits, relu);
  if (splits > 1) run_join<T>(partial, bias, y, x.rows, w.rows, splits, relu, st);
  return adv_internal_finish_launch();
}

// x: codes and scales, or - x.codes NULL - ``values``, which are quantised into ``ws``
template <class T>
int run_linear(Operand x, const void* values, Operand w, const void* bias, void* y, uint8_t* ws, int64_t k, int relu, hipStream_t st) {
  const LinearPlan p = plan_linear(x.rows, w.rows, k);
  if (!x.codes && p.thin && thin_raw(x.rows, k, static_cast<int>(sizeof(T)))) return run_thin<T, 1, true>(x, values, k, w, bias, y, relu, st);
  const int64_t cb = padded(code_bytes(x.rows, k)), sb = padded(scale_bytes(x.rows, k));
  if (!x.codes) {
    const int bad = run_quantize<T>(values, ws, ws + cb, x.rows, k, st);
    if (bad) return bad;
    x.codes = ws, x.scales = ws + cb;
  }
  if (p.thin) {
    if (x.rows <= 16) return run_thin<T, 1, false>(x, nullptr, k, w, bias, y, relu, st);
    if (x.rows <= 32) return run_thin<T, 2, false>(x, nullptr, k, w, bias, y, relu, st);
    return run_thin<T, 4, false>(x, nullptr, k, w, bias, y, relu, st);
  }
  float* partial = reinterpret_cast<float*>(ws + cb + sb);
  const int panels = static_cast<int>(panels_of(k));
  if (p.big) return run_tile<T, 256, 256>(x, w, bias, y, partial, panels, p.splits, relu, st);
  if (x.rows <= 32) return run_tile<T, 32, 128>(x, w, bias, y, partial, panels, p.splits, relu, st);
  if (x.rows <= 64) return run_tile<T, 64, 128>(x, w, bias, y, partial, panels, p.splits, relu, st);
  return run_tile<T, 128, 128>(x, w, bias, y, partial, panels, p.splits, relu, st);
}

// The input gradient: the contraction is dealt to several workgroups where panels x row tiles do not fill two workgroups a CU.  (Row tiles go by m alone,
// and a part's joining has no price here: 301 rows of 4096 -> 25088, 294 workgroups, take 232 us where 512 take 250; 128 rows, in five parts, 81.)
struct GradPlan {
  int bm, splits;
  int64_t padded_n;
};
GradPlan plan_dgrad(int64_t m, int64_t n, int64_t k) {
  const int bm = m <= 32 ? 32 : (m <= 64 ? 64 : 128);
  const int64_t fours = (n + kHeld * kChunk - 1) / (kHeld * kChunk), tiles = panels_of(k) * ((m + bm - 1) / bm);
  int64_t s = 512 / tiles;
  if (s > fours / 2) s = fours / 2;
  if (s < 1) s = 1;
  return {bm, static_cast<int>(s), fours * kHeld * kChunk};
}
int terms_of(int dtype) { return dtype == ADV_F32 ? 3 : (dtype == ADV_F16 ? 2 : 1); }
int64_t plane_bytes(int64_t m, int64_t n, int dtype) { return padded(terms_of(dtype) * m * plan_dgrad(m, n, 1).padded_n * 2); }

template <class T, int BM>
int run_dgrad_tile(const uint8_t* planes, Operand w, void* gx, float* partial, int64_t m, int64_t k, const GradPlan& p, hipStream_t st) {
  const int64_t blocks = panels_of(k) * ((m + BM - 1) / BM) * p.splits;
  constexpr int lds = kGradLds<kTerms<T>, BM>;
  if (!adv_internal_lds_limit<mx4_dgrad<T, BM>>(lds)) return ADV_ELAUNCH;
  mx4_dgrad<T, BM><<<dim3(static_cast<unsigned>(blocks)), kBlock, lds, st>>>(planes, w, static_cast<T*>(gx), partial, m, k, p.padded_n, p.splits);
  if (p.splits > 1) run_join<T>(partial, nullptr, gx, m, k, p.splits, 0, st);
  return adv_internal_finish_launch();
}

constexpr int64_t kAcross = 1 << 16;       // a launch's x dimension has fewer than 2^32 threads: a long list of blocks goes over y as well
template <class T>
int run_dgrad(const void* gy, const void* mask, Operand w, void* gx, uint8_t* ws, int64_t m, int64_t k, int dtype, hipStream_t st) {
  const GradPlan p = plan_dgrad(m, w.rows, k);
  const int64_t units = m * (p.padded_n / 8);
  const int64_t blocks = (units + kBlock - 1) / kBlock, across = blocks < kAcross ? blocks : kAcross;
  mx4_grad_terms<T><<<dim3(static_cast<unsigned>(across), static_cast<unsigned>((blocks + across - 1) / across)), kBlock, 0, st>>>(
      static_cast<const T*>(gy), static_cast<const T*>(mask), ws, m, w.rows, p.padded_n);
  float* partial = reinterpret_cast<float*>(ws + plane_bytes(m, w.rows, dtype));
  if (p.bm == 32) return run_dgrad_tile<T, 32>(ws, w, gx, partial, m, k, p, st);
  if (p.bm == 64) return run_dgrad_tile<T, 64>(ws, w, gx, partial, m, k, p, st);
  return run_dgrad_tile<T, 128>(ws, w, gx, partial, m, k, p, st);
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

int64_t adv_mx4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (!sizes_ok(m, k) || !sizes_ok(n, k)) return ADV_EINVAL;
  return padded(code_bytes(m, k)) + padded(scale_bytes(m, k)) + linear_partial_bytes(m, n, k);
}

int adv_mx4_linear(const void* x, const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales, const void* bias, void* y,
                   void* workspace, int64_t m, int64_t n, int64_t k, int dtype, int relu, adv_stream_t stream) {
  if (!w_codes || !w_scales || !y || !workspace || !sizes_ok(m, k) || !sizes_ok(n, k) || !lowp::known(dtype)) return ADV_EINVAL;
  if (x ? (x_codes || x_scales) : (!x_codes || !x_scales)) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  if (!lowp::aligned(x_codes, 16) || !lowp::aligned(w_codes, 16) || !lowp::aligned(x_scales, 8) || !lowp::aligned(w_scales, 8) || !lowp::aligned(y, e) ||
      !lowp::aligned(bias, e) || !lowp::aligned(x, e) || !lowp::aligned(workspace, kAlign))
    return ADV_EALIGN;
  const struct { const void* at; int64_t bytes; } in[] = {{x, m * k * e}, {x_codes, code_bytes(m, k)}, {x_scales, scale_bytes(m, k)}, {w_codes, code_bytes(n, k)},
                                                          {w_scales, scale_bytes(n, k)}, {bias, n * e}};
  const int64_t yb = m * n * e, wb = adv_mx4_linear_workspace_bytes(m, n, k);
  if (lowp::overlap(y, yb, workspace, wb)) return ADV_EINVAL;
  for (const auto& b : in)
    if (b.at && (lowp::overlap(y, yb, b.at, b.bytes) || lowp::overlap(workspace, wb, b.at, b.bytes))) return ADV_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const Operand xo{x_codes, x_scales, m}, wo{w_codes, w_scales, n};
  if (dtype == ADV_F32) return run_linear<float>(xo, x, wo, bias, y, ws, k, relu, st);
  if (dtype == ADV_BF16) return run_linear<__bf16>(xo, x, wo, bias, y, ws, k, relu, st);
  return run_linear<_Float16>(xo, x, wo, bias, y, ws, k, relu, st);
}

int64_t adv_mx4_linear_dgrad_workspace_bytes(int64_t m, int64_t n, int64_t k, int dtype) {
  if (!sizes_ok(m, k) || !sizes_ok(n, k) || !lowp::known(dtype)) return ADV_EINVAL;
  const GradPlan p = plan_dgrad(m, n, k);
  return plane_bytes(m, n, dtype) + (p.splits > 1 ? padded(4LL * p.splits * m * k) : 0);
}

int adv_mx4_linear_dgrad(const void* gy, const void* mask, const uint8_t* w_codes, const uint8_t* w_scales, void* gx, void* workspace, int64_t m, int64_t n, int64_t k,
                         int dtype, adv_stream_t stream) {
  if (!gy || !w_codes || !w_scales || !gx || !workspace || !sizes_ok(m, k) || !sizes_ok(n, k) || !lowp::known(dtype)) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  if (!lowp::aligned(gy, e) || !lowp::aligned(mask, e) || !lowp::aligned(gx, e) || !lowp::aligned(w_codes, 16) || !lowp::aligned(w_scales, 8) ||
      !lowp::aligned(workspace, kAlign))
    return ADV_EALIGN;
  const struct { const void* at; int64_t bytes; } in[] = {{gy, m * n * e}, {mask, m * n * e}, {w_codes, code_bytes(n, k)}, {w_scales, scale_bytes(n, k)}};
  const int64_t xb = m * k * e, wb = adv_mx4_linear_dgrad_workspace_bytes(m, n, k, dtype);
  if (lowp::overlap(gx, xb, workspace, wb)) return ADV_EINVAL;
  for (const auto& b : in)
    if (b.at && (lowp::overlap(gx, xb, b.at, b.bytes) || lowp::overlap(workspace, wb, b.at, b.bytes))) return ADV_EINVAL;
  const Operand w{w_codes, w_scales, n};
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (dtype == ADV_F32) return run_dgrad<float>(gy, mask, w, gx, ws, m, k, dtype, st);
  if (dtype == ADV_BF16) return run_dgrad<__bf16>(gy, mask, w, gx, ws, m, k, dtype, st);
  return run_dgrad<_Float16>(gy, mask, w, gx, ws, m, k, dtype, st);
}

}  // extern "C"
