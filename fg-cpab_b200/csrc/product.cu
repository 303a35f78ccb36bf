// Projections in 8 bits: matrices as e4m3 codes with an e8m0 scale (a power of
// two) for each 128 of them along the summed axis, and their products.
//
//   s = 2^ceil(log2(max|x| / 448)) >= 2^-126,   q = e4m3(x / s)
//   y[m, n] = sum_k xq[m, k] xs[m, k / 128] wq[n, k] ws[n, k / 128] + bias[n]
//
// The scales are powers of two, so x / s is exact and the codes are those of one
// rounding; the tensor cores apply them (block-scaled instructions) and sum in
// float32.
#include <cuda_fp8.h>

#include <algorithm>
#include <mutex>

#include "product_core.cuh"
#include "sequence.cuh"

namespace cpab {

bool make_tile_map(CUtensorMap *map, bool halves, const void *base, int64_t columns, int64_t rows, int64_t batch,
                   int64_t pitch, int64_t plane, int box_rows) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      encode = reinterpret_cast<Encode>(f);
  });
  if (encode == nullptr) return false;
  const int e = halves ? 2 : 1;
  const cuuint64_t dims[3] = {(cuuint64_t)columns, (cuuint64_t)rows, (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch, (cuuint64_t)plane};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / e), (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
  return encode(map, halves ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3,
                const_cast<void *>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kBlock = 128;  // codes to a scale

// ---- codes -------------------------------------------------------------------

// The scale's exponent + 127 of a block whose largest magnitude has these bits:
// 448 = 1.75 * 2^8, so a mantissa over 1.75 takes the next power.  A block that
// holds an infinity or a NaN has the scale NaN (255).
__device__ __forceinline__ uint32_t scale_exponent(uint32_t most) {
  if (most >= 0x7F800000u) return 255u;
  const uint32_t e = (most + 0x1FFFFFu) >> 23;
  return e > 9u ? e - 8u : 1u;
}
// 1 / scale (NaN for the scale NaN).
__device__ __forceinline__ float inverse_scale(uint32_t exponent) {
  return __uint_as_float(exponent == 255u ? 0x7FC00000u : (254u - exponent) << 23);
}
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

struct QuantizeArgs {
  const void *x;
  int64_t x_row, rows, columns;
  uint8_t *q, *scale;      // by rows, or null
  int64_t q_row, scale_row;
  uint8_t *qt, *scale_t;   // of the transposed matrix, or null
  int64_t qt_row, scale_t_row;
  float *sums;             // [ceil(rows / 128), columns]: columns' sums over each tile, or null
};

// A block takes a tile of 128 x 128; a thread 8 rows x 8 columns of it, so that a
// row's block is 16 threads' (half a warp's) and a column's 8 codes are one word
// pair of the transposed codes.
template <typename T, bool VEC, bool ROWS, bool COLUMNS, bool SUMS>
__global__ void __launch_bounds__(256) k_quantize(const QuantizeArgs a) {
  __shared__ uint32_t most_of[COLUMNS ? 16 : 1][COLUMNS ? 128 : 1];
  __shared__ float sum_of[SUMS ? 16 : 1][SUMS ? 128 : 1];
  __shared__ uint2 turned[COLUMNS ? 128 * 16 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane & 15, band = 2 * warp + (lane >> 4);  // this thread's columns 8 l.., rows 8 band..
  const int64_t tiles_x = (a.columns + 127) / 128;
  const int64_t ty = blockIdx.x / tiles_x, tx = blockIdx.x % tiles_x;
  const int64_t c0 = tx * 128 + 8 * l, r0 = ty * 128 + 8 * band;
  const T *x = static_cast<const T *>(a.x) + r0 * a.x_row + c0;

  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = r0 + i < a.rows;
    if (VEC) {
      constexpr int N = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8; j += N) {
        Pack<T, N> p;
        if (in && c0 + j + N <= a.columns) {
          p = *reinterpret_cast<const Pack<T, N> *>(x + i * a.x_row + j);
#pragma unroll
          for (int k = 0; k < N; ++k) v[i][j + k] = to_f32(p.v[k]);
        } else {  // (nothing is read past a row's end)
#pragma unroll
          for (int k = 0; k < N; ++k)
            v[i][j + k] = in && c0 + j + k < a.columns ? to_f32(x[i * a.x_row + j + k]) : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = in && c0 + j < a.columns ? to_f32(x[i * a.x_row + j]) : 0.f;
    }
  }

  if (COLUMNS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
      most_of[band][8 * l + j] = most;
    }
  }
  if (SUMS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i][j];
      sum_of[band][8 * l + j] = s;
    }
  }
  if (ROWS) {
    const uint32_t half = 0xFFFFu << (lane & 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
      const uint32_t e = scale_exponent(__reduce_max_sync(half, most));
      const float r = inverse_scale(e);
      uint2 w;
      w.x = codes_of(v[i][0] * r, v[i][1] * r, v[i][2] * r, v[i][3] * r);
      w.y = codes_of(v[i][4] * r, v[i][5] * r, v[i][6] * r, v[i][7] * r);
      if (r0 + i < a.rows) {
        // (rows are padded to multiples of 16 codes)
        if (c0 < a.columns) *reinterpret_cast<uint2 *>(a.q + (r0 + i) * a.q_row + c0) = w;
        if (l == 0) a.scale[(r0 + i) * a.scale_row + tx] = (uint8_t)e;
      }
    }
  }
  if (!COLUMNS && !SUMS) return;
  __syncthreads();
  if (COLUMNS) {
    // (all bands' threads of a column find its maximum, of which they keep the scale)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t most = 0;
#pragma unroll
      for (int b = 0; b < 16; ++b) most = max(most, most_of[b][8 * l + j]);
      const uint32_t e = scale_exponent(most);
      const float r = inverse_scale(e);
      uint2 w;
      w.x = codes_of(v[0][j] * r, v[1][j] * r, v[2][j] * r, v[3][j] * r);
      w.y = codes_of(v[4][j] * r, v[5][j] * r, v[6][j] * r, v[7][j] * r);
      turned[(8 * l + j) * 16 + (band ^ l)] = w;  // (so that half a warp's words lie in different banks)
      if (band == 0 && c0 + j < a.columns) a.scale_t[(c0 + j) * a.scale_t_row + ty] = (uint8_t)e;
    }
  }
  if (SUMS && threadIdx.x < 128 && tx * 128 + threadIdx.x < a.columns) {
    float s = 0.f;
#pragma unroll
    for (int b = 0; b < 16; ++b) s += sum_of[b][threadIdx.x];
    a.sums[ty * a.columns + tx * 128 + threadIdx.x] = s;
  }
  if (!COLUMNS) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = i * 16 + (threadIdx.x >> 4), k = threadIdx.x & 15;
    const int64_t column = tx * 128 + c, row = ty * 128 + 8 * k;
    if (column < a.columns && row < a.rows)
      *reinterpret_cast<uint2 *>(a.qt + column * a.qt_row + row) = turned[c * 16 + (k ^ (c >> 3))];
  }
}

// Columns' sums over the tiles, in order.
template <typename T>
__global__ void __launch_bounds__(256) k_sum_tiles(const float *sums, int64_t tiles, int64_t columns, T *out) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= columns) return;
  float s = 0.f;
  for (int64_t t = 0; t < tiles; ++t) s += sums[t * columns + c];
  out[c] = from_f32<T>(s);
}

template <typename T, bool VEC>
void launch_quantize_as(const QuantizeArgs &a, unsigned grid, cudaStream_t s) {
  const bool rows = a.q != nullptr, columns = a.qt != nullptr;
  if (a.sums != nullptr) {
    if (rows && columns) k_quantize<T, VEC, true, true, true><<<grid, 256, 0, s>>>(a);
    else if (rows) k_quantize<T, VEC, true, false, true><<<grid, 256, 0, s>>>(a);
    else if (columns) k_quantize<T, VEC, false, true, true><<<grid, 256, 0, s>>>(a);
    else k_quantize<T, VEC, false, false, true><<<grid, 256, 0, s>>>(a);
  } else if (rows && columns) k_quantize<T, VEC, true, true, false><<<grid, 256, 0, s>>>(a);
  else if (rows) k_quantize<T, VEC, true, false, false><<<grid, 256, 0, s>>>(a);
  else k_quantize<T, VEC, false, true, false><<<grid, 256, 0, s>>>(a);
}

template <typename T>
void launch_quantize(const QuantizeArgs &a, unsigned grid, cudaStream_t s) {
  if (aligned_to(a.x, a.x_row, sizeof(T), 16)) launch_quantize_as<T, true>(a, grid, s);
  else launch_quantize_as<T, false>(a, grid, s);
}

// ---- products ------------------------------------------------------------------

struct Scales {
  const uint8_t *bytes;  // e8m0 [rows, row], or null: all 1
  int64_t row;
  int words;             // rows begin on multiples of 4 bytes and hold whole words
};

struct ProductArgs {
  CUtensorMap a, b;
  Scales sa, sb;
  const float *ra, *rb;  // float32 scales of rows of A, of B, or null
  const void *bias;
  void *y;
  int64_t y_row;
  int M, N, steps;
  int tiles_m, tiles_n;
  int wide;              // y's rows begin on 32 bytes
};

__device__ __forceinline__ uint32_t scale_word(const Scales &s, int row, int rows, int group, int blocks) {
  if (s.bytes == nullptr || row >= rows) return 0x7F7F7F7Fu;
  const uint8_t *p = s.bytes + (int64_t)row * s.row + 4 * group;
  if (s.words) return __ldg(reinterpret_cast<const uint32_t *>(p));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * group + i < blocks) w |= (uint32_t)__ldg(p + i) << (8 * i);
  return w;
}

// y = A B^T in tiles of 128 CTAS x BN.
template <typename T, typename TB, int CTAS, int BN>
struct Product {
  static constexpr int kCtas = CTAS, kBN = BN, kAcc = BN * 2 + 16 <= 512 ? 2 : 1, kParts = 1, kSegment = 0;
  static constexpr bool kScaled = true, kBMn = false;
  // A tile's columns' scales and bias; the next tile's are written while slow warps
  // still read this one's.
  struct alignas(16) Shared {
    float scale[2][BN], bias[2][BN];
  };
  struct Tile {
    int m0, n0, steps, slot;
  };
  const ProductArgs &a;

  __device__ int tiles() const { return a.tiles_m * a.tiles_n; }
  // Bands of 8 rows of tiles, column by column, so that tiles at work together
  // share operands in L2.
  __device__ Tile tile(int i) const {
    const int band = i / (8 * a.tiles_n), top = band * 8, high = min(8, a.tiles_m - top);
    const int in = i - band * 8 * a.tiles_n;
    return {(top + in % high) * 128 * CTAS, in / high * BN, a.steps, (i / (int)(gridDim.x / CTAS)) & 1};
  }
  __device__ void load(const Tile &t, int k, uint32_t sa, uint32_t sb, uint32_t bar, uint32_t rank) const {
    tc::tile_load<CTAS>(sa, &a.a, bar, k * 128, t.m0 + rank * 128, 0);
    tc::tile_load<CTAS>(sb, &a.b, bar, k * 128, t.n0 + rank * (BN / CTAS), 0);
  }
  __device__ uint32_t scale_words_a(const Tile &t, uint32_t rank, int row, int g) const {
    return scale_word(a.sa, t.m0 + rank * 128 + row, a.M, g, a.steps);
  }
  __device__ uint32_t scale_words_b(const Tile &t, int row, int g) const {
    return scale_word(a.sb, t.n0 + row, a.N, g, a.steps);
  }
  __device__ void begin(const Tile &t, Shared &sh, int thread) const {
    if (a.rb == nullptr && a.bias == nullptr) return;
    if (thread < BN) {
      const int n = t.n0 + thread;
      const bool in = n < a.N;
      sh.scale[t.slot][thread] = in && a.rb != nullptr ? a.rb[n] : 1.f;
      sh.bias[t.slot][thread] = in && a.bias != nullptr ? to_f32(static_cast<const TB *>(a.bias)[n]) : 0.f;
    }
    tc::epilogue_sync();
  }
  __device__ void store(const Tile &t, const Shared &sh, int row, int c, const float *acc) const {
    const int col = t.n0 + c;
    if (row >= a.M || col >= a.N) return;
    float v[16];
    const float ra = a.ra != nullptr ? a.ra[row] : 1.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = acc[j] * ra;
    if (a.rb != nullptr || a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = fmaf(v[j], sh.scale[t.slot][c + j], sh.bias[t.slot][c + j]);
    }
    T *y = static_cast<T *>(a.y) + (int64_t)row * a.y_row + col;
    if (a.wide && col + 16 <= a.N) {
      uint32_t w[8];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = pack_pair<T>(v[2 * j], v[2 * j + 1]);
        tc::store_sector(y, w);
      } else {
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[h + j]);
          tc::store_sector(y + h, w);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (col + j < a.N) y[j] = from_f32<T>(v[j]);
    }
  }
};

template <typename T, typename TB, int CTAS, int BN>
__global__ void __launch_bounds__(tc::kCoreThreads, 1) k_product(const __grid_constant__ ProductArgs a) {
  tc::core(Product<T, TB, CTAS, BN>{a});
}

template <typename T, typename TB, int CTAS, int BN>
cudaError_t launch_product_as(ProductArgs &a, cudaStream_t s) {
  using S = tc::CoreShape<Product<T, TB, CTAS, BN>>;
  auto *kernel = k_product<T, TB, CTAS, BN>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (e != cudaSuccess) return e;
  a.tiles_m = (a.M + 128 * CTAS - 1) / (128 * CTAS);
  a.tiles_n = (a.N + BN - 1) / BN;
  const int tiles = a.tiles_m * a.tiles_n, groups = device_info().sm_count / CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CTAS * std::min(tiles, groups)));
  cfg.blockDim = dim3(tc::kCoreThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {CTAS, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, typename TB>
cudaError_t launch_product(ProductArgs &a, cudaStream_t s) {
  return a.M > 128 && a.N > 128 ? launch_product_as<T, TB, 2, 256>(a, s) : launch_product_as<T, TB, 1, 128>(a, s);
}

// What an operand lacks, or null; fills the map and scales.
const char *operand(const cpab_quantized &o, int64_t rows, int64_t K, int box_rows, CUtensorMap *map, Scales *blocks,
                    const float **per_row) {
  if (o.codes == nullptr || o.scale == nullptr) return "null codes or scales";
  if (reinterpret_cast<uintptr_t>(o.codes) % 16 || o.row % 16 || o.row < K)
    return "codes must begin on 16 bytes, each row on a multiple of 16 that holds it";
  *per_row = nullptr, *blocks = {nullptr, 0, 0};
  if (o.scale_row == 0) {
    if (reinterpret_cast<uintptr_t>(o.scale) % 4) return "float32 scales must begin on 4 bytes";
    *per_row = static_cast<const float *>(o.scale);
  } else {
    const int64_t n = (K + kBlock - 1) / kBlock;
    if (o.scale_row < n) return "a row of scales must hold one for each 128 codes";
    const bool words = reinterpret_cast<uintptr_t>(o.scale) % 4 == 0 && o.scale_row % 4 == 0;
    *blocks = {static_cast<const uint8_t *>(o.scale), o.scale_row, words};
  }
  if (!make_tile_map(map, false, o.codes, K, rows, 1, o.row, o.row * rows, box_rows)) return "no tensor map for the codes";
  return nullptr;
}

}  // namespace
}  // namespace cpab

using namespace cpab;

extern "C" int64_t cpab_b200_quantize_blocks_workspace(int64_t rows, int64_t columns) {
  return rows < 0 || columns < 0 ? 0 : (rows + 127) / 128 * columns;
}

extern "C" int cpab_b200_quantize_blocks(int dtype, const void *x, int64_t x_row, int64_t rows, int64_t columns,
                                         uint8_t *q, int64_t q_row, uint8_t *scale, int64_t scale_row, uint8_t *qt,
                                         int64_t qt_row, uint8_t *scale_t, int64_t scale_t_row, int sum_dtype,
                                         void *column_sum, float *workspace, cpab_stream_t stream) {
  if (!dtype_ok(dtype) || (column_sum != nullptr && !dtype_ok(sum_dtype)))
    return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: unknown element type");
  if (rows < 0 || columns < 0 || x_row < 0) return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: negative size");
  const int64_t tiles_y = (rows + 127) / 128, tiles_x = (columns + 127) / 128;
  if (rows >= int64_t(1) << 31 || columns >= int64_t(1) << 31 || tiles_x * tiles_y >= int64_t(1) << 31)
    return report_error(CPAB_ERR_SIZE, "%s", "quantize_blocks: too many elements");
  if (q == nullptr && qt == nullptr && column_sum == nullptr)
    return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: nothing to write");
  if (rows > 0 && columns > 0) {
    if (x == nullptr) return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: null x");
    if (q != nullptr && (scale == nullptr || reinterpret_cast<uintptr_t>(q) % 16 || q_row % 16 || q_row < columns ||
                         scale_row < tiles_x))
      return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: codes' rows must begin on multiples of 16 bytes that "
                          "hold them, scales' rows hold one for each 128 codes");
    if (qt != nullptr && (scale_t == nullptr || reinterpret_cast<uintptr_t>(qt) % 16 || qt_row % 16 || qt_row < rows ||
                          scale_t_row < tiles_y))
      return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: transposed codes' rows must begin on multiples of 16 "
                          "bytes that hold them, scales' rows hold one for each 128 codes");
    if (column_sum != nullptr && workspace == nullptr)
      return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: column sums need a workspace");
  }
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows > 0 && columns > 0) {
    const QuantizeArgs a = {x, x_row, rows, columns, q, scale, q_row, scale_row, qt, scale_t, qt_row, scale_t_row,
                            column_sum != nullptr ? workspace : nullptr};
    const unsigned grid = (unsigned)(tiles_x * tiles_y);
    if (dtype == CPAB_F32) launch_quantize<float>(a, grid, s);
    else if (dtype == CPAB_F16) launch_quantize<__half>(a, grid, s);
    else launch_quantize<__nv_bfloat16>(a, grid, s);
  }
  if (column_sum != nullptr && columns > 0) {
    const unsigned grid = (unsigned)((columns + 255) / 256);
    const int64_t n = rows > 0 ? tiles_y : 0;
    if (sum_dtype == CPAB_F32) k_sum_tiles<<<grid, 256, 0, s>>>(workspace, n, columns, static_cast<float *>(column_sum));
    else if (sum_dtype == CPAB_F16) k_sum_tiles<<<grid, 256, 0, s>>>(workspace, n, columns, static_cast<__half *>(column_sum));
    else k_sum_tiles<<<grid, 256, 0, s>>>(workspace, n, columns, static_cast<__nv_bfloat16 *>(column_sum));
  }
  return launch_status(cudaGetLastError(), "quantize_blocks");
}

extern "C" int cpab_b200_matmul_quantized(int dtype, const cpab_quantized *x, const cpab_quantized *weight, int64_t M,
                                          int64_t N, int64_t K, int bias_dtype, const void *bias, void *y,
                                          int64_t y_row, cpab_stream_t stream) {
  if (!dtype_ok(dtype) || (bias != nullptr && bias_dtype != CPAB_F32 && bias_dtype != dtype))
    return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: unknown element type, or a bias of neither y's nor float32");
  if (x == nullptr || weight == nullptr) return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: null operand");
  if (M < 0 || N < 0 || K < 1 || y_row < N) return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: sizes out of range");
  constexpr int64_t kMost = (int64_t(1) << 31) - 512;
  if (M > kMost || N > kMost || K > kMost || (M + 127) / 128 * ((N + 127) / 128) >= kMost)
    return report_error(CPAB_ERR_SIZE, "%s", "matmul_quantized: sizes too large");
  if (M == 0 || N == 0) return report_error(CPAB_OK, "%s", "");
  if (y == nullptr) return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: null y");
  ProductArgs a = {};
  const char *why = operand(*x, M, K, 128, &a.a, &a.sa, &a.ra);
  if (why == nullptr) why = operand(*weight, N, K, 128, &a.b, &a.sb, &a.rb);
  if (why != nullptr) return report_error(CPAB_ERR_ARG, "matmul_quantized: %s", why);
  a.bias = bias, a.y = y, a.y_row = y_row, a.M = (int)M, a.N = (int)N, a.steps = (int)((K + kBlock - 1) / kBlock);
  a.wide = aligned_to(y, y_row, dtype_size(dtype), 32);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == CPAB_F32) e = launch_product<float, float>(a, s);
  else if (dtype == CPAB_F16)
    e = bias_dtype == CPAB_F32 ? launch_product<__half, float>(a, s) : launch_product<__half, __half>(a, s);
  else e = bias_dtype == CPAB_F32 ? launch_product<__nv_bfloat16, float>(a, s)
                                  : launch_product<__nv_bfloat16, __nv_bfloat16>(a, s);
  return launch_status(e, "matmul_quantized");
}
