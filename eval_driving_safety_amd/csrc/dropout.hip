// Dropout of a fully connected head (the reference's heads: dynamic_vehicles/Model.py:15-34 Linear - Dropout - ReLU, driving_constraint/
// Model.py:15-30 Linear - Dropout) from a counter-based generator: the mask of element i at step s under a seed is a pure function of
// (i, s, seed), so it is never stored - the backward pass computes it again - and two processes draw the same one.
//
//   word(i) = Philox4x32 with seven rounds, counter (i / 4, s), key seed, output i % 4           (Salmon, Moraes, Dror, Shaw, SC'11)
//   kept(i) = word(i) >= t,  t = round(p * 2^32): the rate is met to 2^-33
//   y  = relu?( kept ? (x + b[i % cols]) * (1 / (1 - p)) : 0 )       float32 arithmetic, one rounding to the tensor's type
//   gx = kept && !(relu && y <= 0) ? gy * (1 / (1 - p)) : 0;  gb = sum over rows of gx before its rounding, float32, fixed order
// A dropped element is 0 whatever x holds there (a select, not a product: an infinity does not turn into NaN); a kept NaN stays one.
//
// Seven rounds are the fewest that pass BigCrush (table 2 of the paper); ten would cost 43 % more of what bounds the 16-bit types.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "adv_internal.h"
#include "advengine.h"
#include "lowp.h"

namespace {

constexpr int kBlock = 256;
constexpr int kRounds = 7;

struct Rng {
  uint64_t seed;
  const int64_t* step_at;      // NULL: the step is ``step``
  uint64_t step;
  uint32_t threshold;          // kept: word >= threshold
  int all;                     // p = 1 (a threshold of 2^32): nothing is kept
};

__device__ __forceinline__ void philox(uint64_t i4, uint64_t step, uint64_t seed, uint32_t (&w)[4]) {
  uint32_t a = static_cast<uint32_t>(i4), b = static_cast<uint32_t>(i4 >> 32), c = static_cast<uint32_t>(step), d = static_cast<uint32_t>(step >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint64_t p = static_cast<uint64_t>(0xD2511F53u) * a, q = static_cast<uint64_t>(0xCD9E8D57u) * c;
    a = static_cast<uint32_t>(q >> 32) ^ b ^ k0;
    b = static_cast<uint32_t>(q);
    c = static_cast<uint32_t>(p >> 32) ^ d ^ k1;
    d = static_cast<uint32_t>(p);
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  w[0] = a, w[1] = b, w[2] = c, w[3] = d;
}

// bit j: element first + j is kept.  V / 4 counters where first is a multiple of four, one more where it is not (rows of odd length)
template <int V>
__device__ __forceinline__ uint32_t kept_bits(uint64_t first, uint64_t step, const Rng& g) {
  uint64_t i4 = first >> 2;
  const int off = static_cast<int>(first & 3);
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < V / 4; ++k, ++i4) {
    uint32_t w[4];
    philox(i4, step, g.seed, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) bits |= (w[j] >= g.threshold ? 1u : 0u) << (4 * k + j);
  }
  if (off) {
    uint32_t w[4];
    philox(i4, step, g.seed, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) bits |= (w[j] >= g.threshold ? 1u : 0u) << (V + j);
    bits >>= off;
  }
  return g.all ? 0u : bits;
}

// How the elements are dealt to threads: a thread owns V consecutive columns and walks rows; tx threads (a power of two) stand side by
// side over the columns, kBlock / tx below each other over the rows; block (x, y) has rows [y * chunk, (y + 1) * chunk).  Without a bias the
// tensor is one line, folded into rows of kBlock * V (``n`` ends the last one).
struct Shape {
  int64_t rows, cols, n;       // n = elements: cols * rows, or less in the folded line's last row
  int tx_log2;
  int64_t chunk;
};

// One pass, bound by memory: 4096 x 25088 float32 with a bias 168 us (4.9 TB/s of the 5.05 that a copy of 1 GiB reaches), 512 x 25088 bfloat16 12.2 us
// (4.2 TB/s, out of the last-level cache); 16 x 4096 3 us, latency.  23 vector instructions an element, most of them the generator, under the loads.
template <class T, int V, bool BIAS, bool RELU>
__global__ __launch_bounds__(kBlock) void dropout_fwd(const T* x, const T* __restrict__ bias, T* y, Shape s, Rng g, float scale) {
  const int tx = threadIdx.x & ((1 << s.tx_log2) - 1), ty = threadIdx.x >> s.tx_log2, ny = kBlock >> s.tx_log2;
  const int64_t col = ((static_cast<int64_t>(blockIdx.x) << s.tx_log2) + tx) * V;
  if (col >= s.cols) return;
  const uint64_t step = g.step_at ? static_cast<uint64_t>(*g.step_at) : g.step;
  const int64_t row_end = min(s.rows, (static_cast<int64_t>(blockIdx.y) + 1) * s.chunk);
  const int own = static_cast<int>(min(static_cast<int64_t>(V), s.cols - col));
  float b[V];
  if (BIAS) lowp::load_some<T, V>(bias + col, b, own);
  for (int64_t r = blockIdx.y * s.chunk + ty; r < row_end; r += ny) {
    const int64_t i = r * s.cols + col;
    const int64_t left = s.n - i;
    if (left <= 0) return;
    const int k = static_cast<int>(min(static_cast<int64_t>(own), left));
    float v[V];
    if (k == V) lowp::load<T, V>(x + i, v);
    else lowp::load_some<T, V>(x + i, v, k);
    const uint32_t keep = (g.threshold || g.all) ? kept_bits<V>(static_cast<uint64_t>(i), step, g) : ~0u;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float t = v[j];
      if (BIAS) t += b[j];
      t = (keep >> j & 1u) ? t * scale : 0.0f;
      if (RELU) t = t < 0.0f ? 0.0f : t;      // (a NaN stays)
      v[j] = t;
    }
    if (k == V) lowp::store<T, V>(y + i, v);
    else lowp::store_some<T, V>(y + i, v, k);
  }
}

// RELU: the mask is y > 0 already (a dropped element's y is 0), no generator needed.  SUM: this block's share of the bias gradient goes to
// partial[blockIdx.y][cols], or - the only block of its columns - to gbias.  4096 x 25088 float32 with its bias's gradient 168 + 5 us.
template <class T, int V, bool RELU, bool SUM>
__global__ __launch_bounds__(kBlock) void dropout_bwd(const T* gy, const T* __restrict__ y, T* gx, float* __restrict__ partial, T* __restrict__ gbias,
                                                      Shape s, Rng g, float scale) {
  __shared__ float s_sum[SUM ? kBlock * V : 1];
  const int tx = threadIdx.x & ((1 << s.tx_log2) - 1), ty = threadIdx.x >> s.tx_log2, ny = kBlock >> s.tx_log2;
  const int64_t col = ((static_cast<int64_t>(blockIdx.x) << s.tx_log2) + tx) * V;
  const uint64_t step = RELU ? 0 : (g.step_at ? static_cast<uint64_t>(*g.step_at) : g.step);
  const int64_t row_end = min(s.rows, (static_cast<int64_t>(blockIdx.y) + 1) * s.chunk);
  const int own = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(V), s.cols - col)));
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  for (int64_t r = blockIdx.y * s.chunk + ty; r < row_end && own > 0; r += ny) {
    const int64_t i = r * s.cols + col;
    const int64_t left = s.n - i;
    if (left <= 0) break;
    const int k = static_cast<int>(min(static_cast<int64_t>(own), left));
    float v[V], o[V];
    if (k == V) lowp::load<T, V>(gy + i, v);
    else lowp::load_some<T, V>(gy + i, v, k);
    uint32_t keep = ~0u;
    if (RELU) {
      if (k == V) lowp::load<T, V>(y + i, o);
      else lowp::load_some<T, V>(y + i, o, k);
    } else if (g.threshold || g.all) {
      keep = kept_bits<V>(static_cast<uint64_t>(i), step, g);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool pass = RELU ? !(o[j] <= 0.0f) : (keep >> j & 1u) != 0;
      v[j] = pass ? v[j] * scale : 0.0f;
      if (SUM) sum[j] += v[j];
    }
    if (k == V) lowp::store<T, V>(gx + i, v);
    else lowp::store_some<T, V>(gx + i, v, k);
  }
  if (SUM) {
#pragma unroll
    for (int j = 0; j < V; ++j) s_sum[j * kBlock + threadIdx.x] = sum[j];
    __syncthreads();
    if (ty == 0) {
      const int used = static_cast<int>(min(static_cast<int64_t>(ny), row_end - blockIdx.y * s.chunk));      // threads below each other that had a row
      for (int t = 1; t < used; ++t) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += s_sum[j * kBlock + (t << s.tx_log2) + tx];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j >= own) break;
        if (gridDim.y == 1) gbias[col + j] = static_cast<T>(sum[j]);
        else partial[blockIdx.y * s.cols + col + j] = sum[j];
      }
    }
  }
}

// gbias[c] = partial[0][c] + partial[1][c] + ... : four threads a column, each a quarter of the parts, joined in order
template <class T>
__global__ __launch_bounds__(kBlock) void dropout_bias_sum(const float* __restrict__ partial, T* __restrict__ gbias, int64_t cols, int parts) {
  __shared__ float s_sum[kBlock];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + tx;
  float sum = 0.0f;
  if (c < cols) {
    const int per = (parts + 3) / 4, end = min(parts, (ty + 1) * per);
#pragma unroll 8
    for (int k = ty * per; k < end; ++k) sum += partial[k * cols + c];
  }
  s_sum[threadIdx.x] = sum;
  __syncthreads();
  if (ty == 0 && c < cols) gbias[c] = static_cast<T>(s_sum[tx] + s_sum[64 + tx] + s_sum[128 + tx] + s_sum[192 + tx]);
}

int make_rng(double p, uint64_t seed, const int64_t* step_at, int64_t step, Rng* g, float* scale) {
  if (!(p >= 0.0 && p <= 1.0) || step < 0 || !lowp::aligned(step_at, 8)) return ADV_EINVAL;
  const double t = p * 4294967296.0 + 0.5;
  *g = Rng{seed, step_at, static_cast<uint64_t>(step), t >= 4294967296.0 ? 0u : static_cast<uint32_t>(t), t >= 4294967296.0 ? 1 : 0};
  *scale = g->all ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
  return ADV_OK;
}

// How many threads stand side by side, and how the rows are dealt.  A small tensor is spread over the chip first: fewer columns a block, more rows side
// by side in it, until there are 256 blocks or a thread has one row (16 x 4096: 7.9 -> 2 us a pass against sixteen rows one behind the other).  A
// large one gets about kBlocks blocks.  The bias gradient needs a second launch only where several blocks share a column.
constexpr int64_t kBlocks = 2048;
Shape make_shape(int64_t rows, int64_t cols, int v, bool by_column, bool sums, dim3* grid) {
  Shape s{rows, cols, rows * cols, 8, 1};
  if (!by_column) {
    s.cols = static_cast<int64_t>(kBlock) * v;
    s.rows = (s.n + s.cols - 1) / s.cols;
  }
  auto blocks = [&] { return (s.cols + (static_cast<int64_t>(v) << s.tx_log2) - 1) / (static_cast<int64_t>(v) << s.tx_log2); };
  while (s.tx_log2 > 0 && (static_cast<int64_t>(v) << (s.tx_log2 - 1)) >= s.cols) --s.tx_log2;
  while (by_column && s.tx_log2 > 3 && blocks() < 256 && (kBlock >> s.tx_log2) < s.rows) --s.tx_log2;
  const int64_t gx = blocks(), ny = kBlock >> s.tx_log2;
  int64_t gy = (kBlocks + gx - 1) / gx;
  const int64_t most = sums ? s.rows / (16 * ny) : (s.rows + ny - 1) / ny;
  if (gy > most) gy = most;
  if (gy < 1) gy = 1;
  s.chunk = (s.rows + gy - 1) / gy;
  gy = (s.rows + s.chunk - 1) / s.chunk;
  *grid = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  return s;
}

template <class T>
constexpr int kVec = 16 / sizeof(T);

template <class T>
int run_fwd(const void* x, const void* bias, void* y, int64_t rows, int64_t cols, const Rng& g, float scale, int relu, hipStream_t st) {
  constexpr int V = kVec<T>;
  dim3 grid;
  const Shape s = make_shape(rows, cols, V, bias != nullptr, false, &grid);
  const T* xp = static_cast<const T*>(x);
  const T* bp = static_cast<const T*>(bias);
  T* yp = static_cast<T*>(y);
  if (bias && relu) dropout_fwd<T, V, true, true><<<grid, kBlock, 0, st>>>(xp, bp, yp, s, g, scale);
  else if (bias) dropout_fwd<T, V, true, false><<<grid, kBlock, 0, st>>>(xp, bp, yp, s, g, scale);
  else if (relu) dropout_fwd<T, V, false, true><<<grid, kBlock, 0, st>>>(xp, bp, yp, s, g, scale);
  else dropout_fwd<T, V, false, false><<<grid, kBlock, 0, st>>>(xp, bp, yp, s, g, scale);
  return adv_internal_finish_launch();
}

template <class T>
int run_bwd(const void* gy, const void* y, void* gx, void* gbias, float* partial, int64_t rows, int64_t cols, const Rng& g, float scale, hipStream_t st) {
  constexpr int V = kVec<T>;
  dim3 grid;
  const Shape s = make_shape(rows, cols, V, gbias != nullptr, gbias != nullptr, &grid);
  const T* gp = static_cast<const T*>(gy);
  const T* yp = static_cast<const T*>(y);
  T* op = static_cast<T*>(gx);
  T* bp = static_cast<T*>(gbias);
  if (y && gbias) dropout_bwd<T, V, true, true><<<grid, kBlock, 0, st>>>(gp, yp, op, partial, bp, s, g, scale);
  else if (y) dropout_bwd<T, V, true, false><<<grid, kBlock, 0, st>>>(gp, yp, op, partial, bp, s, g, scale);
  else if (gbias) dropout_bwd<T, V, false, true><<<grid, kBlock, 0, st>>>(gp, yp, op, partial, bp, s, g, scale);
  else dropout_bwd<T, V, false, false><<<grid, kBlock, 0, st>>>(gp, yp, op, partial, bp, s, g, scale);
  if (gbias && grid.y > 1)
    dropout_bias_sum<T><<<dim3(static_cast<unsigned>((cols + 63) / 64)), kBlock, 0, st>>>(partial, bp, cols, static_cast<int>(grid.y));
  return adv_internal_finish_launch();
}

constexpr int64_t kMost = int64_t{1} << 40;      // elements: row and column counts below it keep every product and the grid in range

}  // namespace

extern "C" {

int adv_dropout_fwd(const void* x, const void* bias, void* y, int64_t rows, int64_t cols, int dtype, double p, uint64_t seed, const int64_t* step_at,
                    int64_t step, int relu, adv_stream_t stream) {
  if (!x || !y || rows < 0 || cols < 0 || !lowp::known(dtype)) return ADV_EINVAL;
  Rng g;
  float scale;
  const int bad = make_rng(p, seed, step_at, step, &g, &scale);
  if (bad) return bad;
  if (rows == 0 || cols == 0) return ADV_OK;
  if (rows > kMost / cols) return ADV_EINVAL;
  const int e = lowp::size_of(dtype);
  const int64_t bytes = rows * cols * e;
  if (!lowp::aligned(x, e) || !lowp::aligned(y, e) || !lowp::aligned(bias, e)) return ADV_EALIGN;
  if ((x != y && lowp::overlap(x, bytes, y, bytes)) || (bias && lowp::overlap(bias, cols * e, y, bytes))) return ADV_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ADV_F32) return run_fwd<float>(x, bias, y, rows, cols, g, scale, relu, st);
  if (dtype == ADV_BF16) return run_fwd<__bf16>(x, bias, y, rows, cols, g, scale, relu, st);
  return run_fwd<_Float16>(x, bias, y, rows, cols, g, scale, relu, st);
}

int64_t adv_dropout_bwd_workspace_floats(int64_t rows, int64_t cols, int dtype) {
  if (rows < 0 || cols < 0 || !lowp::known(dtype) || (cols > 0 && rows > kMost / cols)) return ADV_EINVAL;
  if (rows == 0 || cols == 0) return 0;
  dim3 grid;
  make_shape(rows, cols, 16 / lowp::size_of(dtype), true, true, &grid);
  return grid.y > 1 ? static_cast<int64_t>(grid.y) * cols : 0;
}

int adv_dropout_bwd(const void* gy, const void* y, void* gx, void* gbias, float* workspace, int64_t rows, int64_t cols, int dtype, double p, uint64_t seed,
                    const int64_t* step_at, int64_t step, adv_stream_t stream) {
  if (!gy || !gx || rows < 1 || cols < 1 || !lowp::known(dtype) || rows > kMost / cols) return ADV_EINVAL;
  Rng g;
  float scale;
  const int bad = make_rng(p, seed, step_at, step, &g, &scale);
  if (bad) return bad;
  const int e = lowp::size_of(dtype);
  const int64_t bytes = rows * cols * e, ws = gbias ? 4 * adv_dropout_bwd_workspace_floats(rows, cols, dtype) : 0;
  if (ws && !workspace) return ADV_EINVAL;
  if (!lowp::aligned(gy, e) || !lowp::aligned(gx, e) || !lowp::aligned(y, e) || !lowp::aligned(gbias, e) || !lowp::aligned(workspace, 4)) return ADV_EALIGN;
  if ((gy != gx && lowp::overlap(gy, bytes, gx, bytes)) || (y && lowp::overlap(y, bytes, gx, bytes))) return ADV_EINVAL;
  if (gbias && (lowp::overlap(gbias, cols * e, gx, bytes) || lowp::overlap(gbias, cols * e, gy, bytes) || (y && lowp::overlap(gbias, cols * e, y, bytes))))
    return ADV_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == ADV_F32) return run_bwd<float>(gy, y, gx, gbias, workspace, rows, cols, g, scale, st);
  if (dtype == ADV_BF16) return run_bwd<__bf16>(gy, y, gx, gbias, workspace, rows, cols, g, scale, st);
  return run_bwd<_Float16>(gy, y, gx, gbias, workspace, rows, cols, g, scale, st);
}

}  // extern "C"
