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
#include <atomic>
#include <mutex>
#include <type_traits>

#include "product_core.cuh"
#include "sequence.cuh"

namespace cpab {

namespace {

constexpr int kDevices = 64;
std::atomic<int64_t> g_longest{2000000000};
std::atomic<int *> g_words[kDevices];  // a page that host and device share, for each device
std::mutex g_words_mutex;

std::atomic<int *> *word_of_device() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && device >= 0 && device < kDevices ? &g_words[device] : nullptr;
}

}  // namespace

tc::Waits tc::waits() {
  std::atomic<int *> *word = word_of_device();
  if (word != nullptr && word->load() == nullptr) {
    std::lock_guard<std::mutex> lock(g_words_mutex);
    if (word->load() == nullptr) {
      // (the first call may be one of a capture)
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaThreadExchangeStreamCaptureMode(&mode);
      void *p = nullptr;
      if (cudaHostAlloc(&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable) == cudaSuccess) {
        *static_cast<int *>(p) = 0;
        word->store(static_cast<int *>(p));
      } else {
        (void)cudaGetLastError();
      }
      cudaThreadExchangeStreamCaptureMode(&mode);
    }
  }
  return {(uint64_t)g_longest.load(), word != nullptr ? word->load() : nullptr};
}
bool tc::gave_up() {
  std::atomic<int *> *word = word_of_device();
  volatile int *p = word != nullptr ? word->load() : nullptr;
  if (p == nullptr || *p == 0) return false;
  *p = 0;
  return true;
}
int tc::report_gave_up(const char *what) {
  return report_error(CPAB_ERR_WAIT, "%s: not begun: a matrix product before it gave up waiting, and its results are NaN",
                      what);
}

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
constexpr int64_t kMostSize = (int64_t(1) << 31) - 512;

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

// The eight elements of a row that a thread holds, as read: magnitudes, their maximum
// and float32 values.  Magnitudes of 16-bit types are compared two at a time, as
// whole numbers.
template <typename T>
struct Eight {
  uint32_t w[4];
  __device__ float2 pair(int k) const { return unpack_pair<T>(w[k]); }
  // Bits of the larger magnitude of two words each, element by element.
  static __device__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  __device__ uint32_t magnitude(int k) const { return w[k] & 0x7FFF7FFFu; }
  __device__ uint32_t most() const {
    const uint32_t m = larger(larger(magnitude(0), magnitude(1)), larger(magnitude(2), magnitude(3)));
    return max(m & 0xFFFFu, m >> 16);
  }
  static constexpr int kWords = 4;
  // float32 bits of the element's magnitude
  static __device__ uint32_t bits(uint32_t m) {
    if constexpr (sizeof(T) == 4) return m;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
    else return __float_as_uint(__half2float(__ushort_as_half((uint16_t)m)));
  }
};
template <>
struct Eight<float> {
  uint32_t w[8];
  __device__ float2 pair(int k) const { return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1])); }
  static __device__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ uint32_t magnitude(int k) const { return w[k] & 0x7FFFFFFFu; }
  __device__ uint32_t most() const {
    uint32_t m = magnitude(0);
#pragma unroll
    for (int k = 1; k < 8; ++k) m = max(m, magnitude(k));
    return m;
  }
  static constexpr int kWords = 8;
  static __device__ uint32_t bits(uint32_t m) { return m; }
};

// A block takes a tile of 128 x 128; a thread 8 rows x 8 columns of it, so that a
// row's block is 16 threads' (half a warp's) and a column's 8 codes are one word
// pair of the transposed codes, which cross through shared memory.
template <typename T, bool COLUMNS, bool SUMS>
struct QuantizeShared {
  uint2 turned[COLUMNS ? 128 * 16 : 1];
  uint32_t most_of[COLUMNS ? 8 : 1][COLUMNS ? 16 * Eight<T>::kWords : 1];
  float inverse[COLUMNS ? 128 : 1];
  float sum_of[SUMS ? 8 : 1][SUMS ? 128 : 1];
};

// FULL: the tile lies inside the matrix (16384 x 4096 both ways without this form: 67 us).
template <typename T, bool VEC, bool ROWS, bool COLUMNS, bool SUMS, bool FULL>
__device__ __forceinline__ void quantize_tile(const QuantizeArgs &a, QuantizeShared<T, COLUMNS, SUMS> &sh, int64_t tx,
                                              int64_t ty) {
  using E = Eight<T>;
  constexpr int W = E::kWords;
  auto &most_of = sh.most_of;
  auto &inverse = sh.inverse;
  auto &sum_of = sh.sum_of;
  auto &turned = sh.turned;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane & 15, band = 2 * warp + (lane >> 4);  // this thread's columns 8 l.., rows 8 band..
  const int64_t c0 = tx * 128 + 8 * l, r0 = ty * 128 + 8 * band;
  const T *x = static_cast<const T *>(a.x) + r0 * a.x_row + c0;

  E v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = FULL || r0 + i < a.rows;
    if (VEC && in && (FULL || c0 + 8 <= a.columns)) {
#pragma unroll
      for (int k = 0; k < W; k += 4)
        *reinterpret_cast<uint4 *>(v[i].w + k) =
            *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(x + i * a.x_row) + k);
    } else {  // (nothing is read past a row's end)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e0 = in && (FULL || c0 + 2 * k < a.columns) ? to_f32(x[i * a.x_row + 2 * k]) : 0.f;
        const float e1 = in && (FULL || c0 + 2 * k + 1 < a.columns) ? to_f32(x[i * a.x_row + 2 * k + 1]) : 0.f;
        if constexpr (sizeof(T) == 2) v[i].w[k] = pack_pair<T>(e0, e1);
        else v[i].w[2 * k] = __float_as_uint(e0), v[i].w[2 * k + 1] = __float_as_uint(e1);
      }
    }
  }

  if (COLUMNS) {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      uint32_t most = v[0].magnitude(k);
#pragma unroll
      for (int i = 1; i < 8; ++i) most = E::larger(most, v[i].magnitude(k));
      most = E::larger(most, __shfl_xor_sync(~0u, most, 16));
      if (lane < 16) most_of[warp][l * W + k] = most;
    }
  }
  if (SUMS) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) s.x += v[i].pair(k).x, s.y += v[i].pair(k).y;
      s.x += __shfl_xor_sync(~0u, s.x, 16);
      s.y += __shfl_xor_sync(~0u, s.y, 16);
      if (lane < 16) *reinterpret_cast<float2 *>(&sum_of[warp][8 * l + 2 * k]) = s;
    }
  }
  if (ROWS) {
    const uint32_t half = 0xFFFFu << (lane & 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t e = scale_exponent(E::bits(__reduce_max_sync(half, v[i].most())));
      const float r = inverse_scale(e);
      const float2 p0 = v[i].pair(0), p1 = v[i].pair(1), p2 = v[i].pair(2), p3 = v[i].pair(3);
      uint2 w;
      w.x = codes_of(p0.x * r, p0.y * r, p1.x * r, p1.y * r);
      w.y = codes_of(p2.x * r, p2.y * r, p3.x * r, p3.y * r);
      if (FULL || r0 + i < a.rows) {
        // (rows are padded to multiples of 16 codes)
        if (FULL || c0 < a.columns) *reinterpret_cast<uint2 *>(a.q + (r0 + i) * a.q_row + c0) = w;
        if (l == 0) a.scale[(r0 + i) * a.scale_row + tx] = (uint8_t)e;
      }
    }
  }
  if (!COLUMNS && !SUMS) return;
  __syncthreads();
  if (threadIdx.x < 128) {
    const int c = threadIdx.x;
    const int64_t column = tx * 128 + c;
    if (COLUMNS) {
      uint32_t most = 0;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint32_t m = sizeof(T) == 2 ? most_of[b][c >> 1] >> (16 * (c & 1)) & 0xFFFFu : most_of[b][c];
        most = max(most, m);
      }
      const uint32_t e = scale_exponent(E::bits(most));
      inverse[c] = inverse_scale(e);
      if (FULL || column < a.columns) a.scale_t[column * a.scale_t_row + ty] = (uint8_t)e;
    }
    if (SUMS && (FULL || column < a.columns)) {
      float s = 0.f;
#pragma unroll
      for (int b = 0; b < 8; ++b) s += sum_of[b][c];
      a.sums[ty * a.columns + column] = s;
    }
  }
  if (!COLUMNS) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 r = *reinterpret_cast<const float2 *>(&inverse[8 * l + 2 * k]);
    float2 p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = v[i].pair(k);
    uint2 w;
    w.x = codes_of(p[0].x * r.x, p[1].x * r.x, p[2].x * r.x, p[3].x * r.x);
    w.y = codes_of(p[4].x * r.x, p[5].x * r.x, p[6].x * r.x, p[7].x * r.x);
    turned[(8 * l + 2 * k) * 16 + (band ^ l)] = w;  // (so that half a warp's words lie in different banks)
    w.x = codes_of(p[0].y * r.y, p[1].y * r.y, p[2].y * r.y, p[3].y * r.y);
    w.y = codes_of(p[4].y * r.y, p[5].y * r.y, p[6].y * r.y, p[7].y * r.y);
    turned[(8 * l + 2 * k + 1) * 16 + (band ^ l)] = w;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = i * 16 + (threadIdx.x >> 4), k = threadIdx.x & 15;
    const int64_t column = tx * 128 + c, row = ty * 128 + 8 * k;
    if (FULL || (column < a.columns && row < a.rows))
      *reinterpret_cast<uint2 *>(a.qt + column * a.qt_row + row) = turned[c * 16 + (k ^ (c >> 3))];
  }
}

template <typename T, bool VEC, bool ROWS, bool COLUMNS, bool SUMS>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && !SUMS ? 3 : 2) k_quantize(const QuantizeArgs a) {
  __shared__ QuantizeShared<T, COLUMNS, SUMS> sh;
  const int64_t tiles_x = (a.columns + 127) / 128;
  const int64_t ty = blockIdx.x / tiles_x, tx = blockIdx.x - ty * tiles_x;
  tc::dep_launch();
  tc::dep_wait();
  if (ty * 128 + 128 <= a.rows && tx * 128 + 128 <= a.columns)
    quantize_tile<T, VEC, ROWS, COLUMNS, SUMS, true>(a, sh, tx, ty);
  else
    quantize_tile<T, VEC, ROWS, COLUMNS, SUMS, false>(a, sh, tx, ty);
}

// Columns' sums over the tiles, in a fixed order: 32 columns a block, each by 8
// threads.
template <typename T>
__global__ void __launch_bounds__(256) k_sum_tiles(const float *sums, int64_t tiles, int64_t columns, T *out) {
  __shared__ float part[8][32];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + x;
  tc::dep_launch();
  tc::dep_wait();
  float s = 0.f;
  if (c < columns) {
#pragma unroll 8
    for (int64_t t = y; t < tiles; t += 8) s += sums[t * columns + c];
  }
  part[y][x] = s;
  __syncthreads();
  if (y == 0 && c < columns) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[k][x];
    out[c] = from_f32<T>(s);
  }
}

template <typename T, bool VEC>
cudaError_t launch_quantize_as(const QuantizeArgs &a, unsigned grid, cudaStream_t s) {
  const bool rows = a.q != nullptr, columns = a.qt != nullptr;
  auto go = [&](void (*kernel)(QuantizeArgs)) { return tc::launch(kernel, grid, 256, 0, 1, s, a); };
  if (a.sums != nullptr) {
    if (rows && columns) return go(k_quantize<T, VEC, true, true, true>);
    if (rows) return go(k_quantize<T, VEC, true, false, true>);
    if (columns) return go(k_quantize<T, VEC, false, true, true>);
    return go(k_quantize<T, VEC, false, false, true>);
  }
  if (rows && columns) return go(k_quantize<T, VEC, true, true, false>);
  if (rows) return go(k_quantize<T, VEC, true, false, false>);
  return go(k_quantize<T, VEC, false, true, false>);
}

template <typename T>
cudaError_t launch_quantize(const QuantizeArgs &a, unsigned grid, cudaStream_t s) {
  return aligned_to(a.x, a.x_row, sizeof(T), 16) ? launch_quantize_as<T, true>(a, grid, s)
                                                 : launch_quantize_as<T, false>(a, grid, s);
}

// ---- codes that lie otherwise ---------------------------------------------------

struct LayoutArgs {
  const uint8_t *src[2];
  uint8_t *dst[2];
  int64_t src_row[2], rows[2];
  int64_t K, groups;  // 16 codes to a group
};

// Rows of codes that begin anywhere, to rows that begin on 16 bytes; the codes of up
// to two matrices at once, 16 a thread.  (A product of 100 x 2000 x 1003 such codes takes
// 16 us, with torch's copies of both 23.)
__global__ void __launch_bounds__(256) k_lay_out(const __grid_constant__ LayoutArgs a) {
  tc::dep_launch();
  tc::dep_wait();
  const int m = blockIdx.y;
  const int64_t count = a.rows[m] * a.groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / a.groups, k = (i - row * a.groups) * 16;
    const uint8_t *from = a.src[m] + row * a.src_row[m] + k;
    uint32_t w[4] = {0, 0, 0, 0};
    if (k >= 4 && k + 20 <= a.K) {  // whole words around them lie in the row
      const uint32_t shift = 8 * (uint32_t)(reinterpret_cast<uintptr_t>(from) & 3);
      const uint32_t *words = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(from) & ~uintptr_t(3));
      uint32_t v[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) v[j] = words[j];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], shift);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k + j < a.K) w[j >> 2] |= (uint32_t)from[j] << (8 * (j & 3));
    }
    *reinterpret_cast<uint4 *>(a.dst[m] + row * a.groups * 16 + k) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- products ------------------------------------------------------------------

// An operand's scales: of blocks, or of rows.  A row's float32 scale is taken apart: its
// power of two goes to each of its blocks, so that the sums are within a factor 4 of the
// results and leave float32's range only where those do, and the rest (1 to 2) to the
// sum.  (As one factor of the sum, 1e30 and the other operand's 1e-33 came to infinity; a
// choice of the order for each element made 8192 x 8192 x 8192 547 us.)
struct Scales {
  const uint8_t *bytes;  // e8m0 [rows, row], or null
  int64_t row;
  int words;             // rows begin on multiples of 4 bytes
  const float *rows;     // float32 [rows], or null
};

// A row's scale as a byte's power of two (an infinity and a NaN have none), and the rest.
__device__ __forceinline__ uint32_t row_power(float r) {
  const uint32_t e = __float_as_uint(r) >> 23 & 255u;
  return e == 255u ? 127u : max(e, 1u);
}
__device__ __forceinline__ float row_rest(float r) {
  const uint32_t bits = __float_as_uint(r), e = bits & 0x7F800000u;
  if (e == 0u) return r * 0x1p126f;
  return e == 0x7F800000u ? r : __uint_as_float((bits & 0x807FFFFFu) | 0x3F800000u);
}
__device__ __forceinline__ float row_rest(const Scales &s, int64_t row) {
  return s.rows != nullptr ? row_rest(s.rows[row]) : 1.f;
}

struct ProductArgs {
  CUtensorMap a, b;
  Scales sa, sb;
  const void *bias;
  void *y;
  int64_t y_row;
  int M, N, steps;
  int tiles_m, tiles_n;
  int wide;              // y's rows begin on 16 bytes
  int a_rows;            // of A that a block loads: what M leaves of 128
  int splits, each;      // the sum in so many parts of `each` steps (a multiple of 8),
  float *parts;          // float32 [splits, M, pitch], where they are not one
  int64_t pitch;
  tc::Waits waits;
};

// A row's scales of 8 steps (of a row's one scale its bits, until all are asked for).
// Rows outside hold no codes: any scale but NaN.
__device__ __forceinline__ void scale_words(const Scales &s, int row, int rows, int group, int blocks, uint32_t (&w)[2]) {
  if (s.rows != nullptr) {
    w[0] = row < rows ? __float_as_uint(s.rows[row]) : 0x3F800000u;
    return;
  }
  if (row >= rows) {
#pragma unroll
    for (int q = 0; q < 2; ++q) w[q] = 0x7F7F7F7Fu;
    return;
  }
  const int first = 8 * group;
  const uint8_t *p = s.bytes + (int64_t)row * s.row + first;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    w[q] = 0;
    if (s.words && first + 4 * q + 4 <= blocks) {
      w[q] = reinterpret_cast<const uint32_t *>(p)[q];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (first + 4 * q + i < blocks) w[q] |= (uint32_t)p[4 * q + i] << (8 * i);
    }
  }
}

// Longer sums are cut into segments of so many steps, which are added in registers: what
// an accumulator cuts off has one sign, in the mean 2.2e-8 of the sum for each 32 codes
// of like signs.  Float32 results are at most 5.6e-6 off by it (in one piece 3.9e-5 at
// 32768 codes and 2.8e-4 at 131072), 16-bit ones 1.1e-5 (2^20 codes: 4e-3, a whole
// rounding to bfloat16).  A segment's end costs 1 us of its 26 (2048 x 2048 x 32768 in
// float32: 104 -> 108 us), segments of 16 steps 19% of the whole.
template <typename T>
constexpr int longest_sum() {
  return sizeof(T) == 4 ? 64 : 128;
}

// y = A B^T in tiles of 128 CTAS x BN.  LONG: with segments (kernels of their own: their
// registers made 16384 x 4096 x 2048 in float32 162 us, without 128).
template <typename T, typename TB, int CTAS, int BN, bool LONG>
struct Product {
  static constexpr int kCtas = CTAS, kBN = BN, kAcc = BN * 2 + 16 <= 512 ? 2 : 1, kParts = 1;
  static constexpr int kSegment = LONG ? longest_sum<T>() : 0;
  static constexpr int kChunk = 64 / sizeof(T);  // 64 bytes of a row at a time
  static constexpr bool kScaled = true, kBMn = false;
  // A tile's columns' scales and bias; the next tile's are written while slow warps
  // still read this one's.
  struct alignas(16) Shared {
    float scale[2][BN], bias[2][BN];
    // Each warp's 32 rows of 64 bytes (and 16 of padding, for the banks) on their way
    // out, so that four threads store a row's 64 bytes and not each thread its own
    // row's 32.
    uint4 rows[8][32][5];
  };
  struct Tile {
    int m0, n0, steps, slot, part;
  };
  const ProductArgs &a;

  __device__ const tc::Waits &waits() const { return a.waits; }
  __device__ int tiles() const { return a.tiles_m * a.tiles_n * a.splits; }
  // Bands of 8 rows of tiles, column by column, so that tiles at work together
  // share operands in L2.
  __device__ Tile tile(int i) const {
    const int slot = (i / (int)(gridDim.x / CTAS)) & 1, part = a.splits > 1 ? i / (a.tiles_m * a.tiles_n) : 0;
    i -= part * a.tiles_m * a.tiles_n;
    const int band = i / (8 * a.tiles_n), top = band * 8, high = min(8, a.tiles_m - top);
    const int in = i - band * 8 * a.tiles_n;
    return {(top + in % high) * 128 * CTAS, in / high * BN, min(a.each, a.steps - part * a.each), slot, part};
  }
  __device__ void warm(const Tile &) const {
    if (threadIdx.x == 0) tc::prefetch_map(&a.a), tc::prefetch_map(&a.b);
    tc::touch(a.sa.bytes), tc::touch(a.sb.bytes), tc::touch(a.y), tc::touch(a.bias), tc::touch(a.wide);
    tc::touch(a.sa.rows), tc::touch(a.sb.rows);
  }
  __device__ void load(const Tile &t, int k, uint32_t sa, uint32_t sb, uint32_t bar, uint32_t rank) const {
    const int at = (t.part * a.each + k) * 128;
    tc::tile_load<CTAS>(sa, &a.a, bar, at, t.m0 + rank * 128, 0);
    tc::tile_load<CTAS>(sb, &a.b, bar, at, t.n0 + rank * (BN / CTAS), 0);
  }
  // (Rows of A that are not loaded hold anything, and so do the sums that nobody
  // stores.  With all 128 loaded, as zeros, a row by 8192 x 8192 took 31 us.)
  __device__ uint32_t stage_bytes() const { return CTAS * 128 * (a.a_rows + BN / CTAS); }
  __device__ void scales_a(const Tile &t, uint32_t rank, int row, int g, uint32_t (&w)[2]) const {
    scale_words(a.sa, t.m0 + rank * 128 + row, a.M, t.part * (a.each / 8) + g, a.steps, w);
  }
  __device__ void scales_b(const Tile &t, int row, int g, uint32_t (&w)[2]) const {
    scale_words(a.sb, t.n0 + row, a.N, t.part * (a.each / 8) + g, a.steps, w);
  }
  __device__ bool one_a() const { return a.sa.rows != nullptr; }
  __device__ bool one_b() const { return a.sb.rows != nullptr; }
  __device__ void words_of_one(uint32_t (&w)[2]) const { w[0] = w[1] = 0x01010101u * row_power(__uint_as_float(w[0])); }
  __device__ void begin(const Tile &t, Shared &sh, int thread) const {
    if (a.splits > 1 || (a.sb.rows == nullptr && a.bias == nullptr)) return;
    if (thread < BN) {
      const int n = t.n0 + thread;
      const bool in = n < a.N;
      sh.scale[t.slot][thread] = in ? row_rest(a.sb, n) : 1.f;
      sh.bias[t.slot][thread] = in && a.bias != nullptr ? to_f32(static_cast<const TB *>(a.bias)[n]) : 0.f;
    }
    tc::epilogue_sync();
  }
  struct Ahead {};
  __device__ Ahead ahead(const Tile &, int, int) const { return {}; }
  __device__ void store(const Tile &t, Shared &sh, int row, int c, const float *acc, const Ahead &) const {
    const int col = t.n0 + c, lane = threadIdx.x & 31;
    if (col >= a.N) return;
    if (a.splits > 1) {
      if (row >= a.M) return;
      float *to = a.parts + ((int64_t)t.part * a.M + row) * a.pitch + col;
#pragma unroll
      for (int k = 0; k < kChunk; k += 8) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(acc[k + j]);
        if (col + k < a.N) tc::store_sector(to + k, w);  // (the pitch is a multiple of 8)
      }
      return;
    }
    uint4(&rows)[32][5] = sh.rows[(threadIdx.x >> 5) - 4];
    const float ra = row < a.M ? row_rest(a.sa, row) : 1.f;
    const bool columns = a.sb.rows != nullptr || a.bias != nullptr;
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 4; ++h) {  // 16 bytes
      constexpr int E = 16 / sizeof(T);
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        v[j] = acc[h * E + j] * ra;
        if (columns) v[j] = fmaf(v[j], sh.scale[t.slot][c + h * E + j], sh.bias[t.slot][c + h * E + j]);
      }
      uint4 w;
      if constexpr (sizeof(T) == 2)
        w = make_uint4(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]), pack_pair<T>(v[4], v[5]), pack_pair<T>(v[6], v[7]));
      else
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      rows[lane][h] = w;
    }
    __syncwarp();
    const int first = row - lane;  // of the warp's rows
    if (a.wide && col + kChunk <= a.N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        if (first + r < a.M)
          *reinterpret_cast<uint4 *>(static_cast<T *>(a.y) + (int64_t)(first + r) * a.y_row + col + (lane & 3) * (16 / sizeof(T))) =
              rows[r][lane & 3];
      }
    } else {  // rows that begin anywhere, or end here: element by element
      constexpr int R = 32 / kChunk;  // rows at a time
      const int x = lane % kChunk;
      T *y = static_cast<T *>(a.y) + col + x;
#pragma unroll 4
      for (int r = lane / kChunk; r < 32; r += R)
        if (first + r < a.M && col + x < a.N) y[(int64_t)(first + r) * a.y_row] = reinterpret_cast<const T *>(rows[r])[x];
    }
  }
};

// The parts of a sum, in order.
template <typename T, typename TB>
__global__ void __launch_bounds__(256) k_join_product(const __grid_constant__ ProductArgs a) {
  tc::dep_launch();
  tc::dep_wait();
  const int64_t count = (int64_t)a.M * a.N, plane = a.M * a.pitch;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / a.N, col = i - row * a.N;
    const float *from = a.parts + row * a.pitch + col;
    const float ra = row_rest(a.sa, row), rb = row_rest(a.sb, col);
    float v = 0.f;
#pragma unroll 8
    for (int k = 0; k < a.splits; ++k) v += from[k * plane];
    v *= ra, v *= rb;
    if (a.bias != nullptr) v += to_f32(static_cast<const TB *>(a.bias)[col]);
    static_cast<T *>(a.y)[row * a.y_row + col] = from_f32<T>(v);
  }
}

template <typename T, typename TB, int CTAS, int BN, bool LONG>
__global__ void __launch_bounds__(tc::kCoreThreads, 1) k_product(const __grid_constant__ ProductArgs a) {
  tc::core(Product<T, TB, CTAS, BN, LONG>{a});
}

template <typename T, typename TB, int CTAS, int BN>
cudaError_t launch_product_as(ProductArgs &a, cudaStream_t s) {
  using S = tc::CoreShape<Product<T, TB, CTAS, BN, false>>;  // (as large with segments)
  auto *kernel = a.each > longest_sum<T>() ? k_product<T, TB, CTAS, BN, true> : k_product<T, TB, CTAS, BN, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (e != cudaSuccess) return e;
  a.tiles_m = (a.M + 128 * CTAS - 1) / (128 * CTAS);
  a.tiles_n = (a.N + BN - 1) / BN;
  const int tiles = a.tiles_m * a.tiles_n * a.splits, groups = device_info().sm_count / CTAS;
  e = tc::launch(kernel, (unsigned)(CTAS * std::min(tiles, groups)), tc::kCoreThreads, S::kBytes, CTAS, s, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  const int64_t blocks = std::min<int64_t>(((int64_t)a.M * a.N + 255) / 256, 8 * device_info().sm_count);
  return tc::launch(k_join_product<T, TB>, (unsigned)blocks, 256, 0, 1, s, a);
}

// The tile of the least time: 128 x 64, 128 x 128, or 256 x 256 by a pair of blocks.
// Measured (us, bf16): a wave of tiles costs 0.3 + 0.26 s, 0.4 + 0.29 s and 1.5 + 0.40 s
// for s steps of 128, a launch 3, 3 and 4.8 more.  1024^3: 5.3, 6.1, 9.4 us; 2048^3:
// 20.7, 13.4, 12.8; 16384 x 4096 x 2048: 249, 144, 111.
int tile_of(int64_t M, int64_t N, int64_t steps) {
  const int64_t sms = device_info().sm_count;
  const float launch[3] = {3.f, 3.f, 4.8f}, wave[3] = {0.3f, 0.4f, 1.5f}, step[3] = {0.26f, 0.29f, 0.40f};
  const int64_t rows[3] = {128, 128, 256}, columns[3] = {64, 128, 256};
  int best = 0;
  float least = 0.f;
  for (int k = 0; k < 3; ++k) {
    const int64_t tiles = (M + rows[k] - 1) / rows[k] * ((N + columns[k] - 1) / columns[k]);
    const int64_t slots = std::max<int64_t>(1, k == 2 ? sms / 2 : sms), waves = (tiles + slots - 1) / slots;
    const float t = launch[k] + (float)waves * (wave[k] + step[k] * (float)steps);
    if (k == 0 || t < least) best = k, least = t;
  }
  return best;
}

// Parts that a long sum of few tiles is cut into, and their steps: as many parts as
// there are blocks for, of at least 16 steps (the joining launch costs 4 us, 16 steps).
// 256 x 128 x 131072, a narrow network's weight gradient: 18 us, where one part's 1024
// steps of 0.26 take 270; 16 x 361 x 6942 11 us, in one part 17.
struct Split {
  int splits, each;
};
Split split_of(int64_t M, int64_t N, int64_t steps) {
  const int tile = tile_of(M, N, steps);
  const int64_t rows = tile == 2 ? 256 : 128, columns = tile == 2 ? 256 : tile == 1 ? 128 : 64;
  const int64_t tiles = (M + rows - 1) / rows * ((N + columns - 1) / columns);
  const int64_t slots = tile == 2 ? device_info().sm_count / 2 : device_info().sm_count;
  const int64_t parts = std::min<int64_t>({64, slots / tiles, steps / 16});
  if (parts < 2) return {1, (int)steps};
  const int64_t each = ((steps + parts - 1) / parts + 7) / 8 * 8;
  return {(int)((steps + each - 1) / each), (int)each};
}

template <typename T, typename TB>
cudaError_t launch_product(ProductArgs &a, cudaStream_t s) {
  switch (tile_of(a.M, a.N, a.steps)) {
    case 2: return launch_product_as<T, TB, 2, 256>(a, s);
    case 1: return launch_product_as<T, TB, 1, 128>(a, s);
    default: return launch_product_as<T, TB, 1, 64>(a, s);
  }
}

// ---- few rows ----------------------------------------------------------------------
//
// A product of at most 16 rows is a pass over the weight: its codes go from memory to
// the registers of the warp that multiplies them (as halves, which hold them exactly),
// without a tile of 128 rows that would be empty.  A warp takes 16 of the weight's rows
// and an eighth of the sum, in blocks of 128; a block's eight warps are added in order.
// Any order of the summed index will do as long as both operands have it: a lane's 16
// neighbouring codes of a row are its share of four instructions.
// One row by 4096 x 2048: 4.3 us, by tiles 6.9; by 5000 x 6000 18.7 and 15.5; 16 rows by
// 4096 x 2048 7.5 and 6.9.

constexpr int kFewMost = 16;
constexpr int kFewWarps = 8;

struct FewArgs {
  const uint8_t *x, *w;
  int64_t x_row, w_row;
  Scales sx, sw;
  const void *bias;
  void *y;
  int64_t y_row;
  int M, N, K, blocks;
};

// 16 codes of a row from k on; 0 past its end.
__device__ __forceinline__ uint4 sixteen(const uint8_t *row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const uint4 *>(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Two codes (the low or high half of a word) as halves.
__device__ __forceinline__ uint32_t two_halves(uint32_t w, bool high) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(high ? w >> 16 : w & 0xFFFFu), __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
// The scale of an e8m0 byte (255: NaN; 2^-127 is subnormal).
__device__ __forceinline__ float power(uint32_t e) {
  return __uint_as_float(e == 255u ? 0x7FC00000u : e == 0u ? 0x00400000u : e << 23);
}
// Whether one is so far from 1 that a block's sum of products of codes (a multiple of
// 2^-18, at most 2^25) times it alone can leave float32's normal range.
__device__ __forceinline__ bool is_far(uint32_t e) { return e - 67u > 120u; }
// Such a sum times two of them, the smaller first (which is exact, down to 2^-145).
__device__ __forceinline__ float by_powers(float v, float a, float b) { return a < b ? v * a * b : v * b * a; }
// v (2^-18 to 2^51 or 0) times two rows' powers, half of their sum's at a time: only what
// ends as 0 or an infinity leaves float32's range between.
__device__ __forceinline__ float by_rows(float v, float a, float b) {
  const int e = (int)(row_power(a) + row_power(b)) - 254, p = e >> 1;
  return v * __uint_as_float((uint32_t)(p + 127) << 23) * __uint_as_float((uint32_t)(e - p + 127) << 23);
}

// KIND: both operands have scales of blocks; both of rows, whose sums are of codes alone;
// or one of each, where a row's power of two is that of each of its blocks.  (A row by
// 4096 x 2048, weights out of L2: 5.0, 4.4 and 5.3 us; with all of it in one kernel 5.3.)
enum FewScales { kBlocks, kRows, kMixed };
template <typename T, typename TB, int TILES, FewScales KIND>
__global__ void __launch_bounds__(32 * kFewWarps) k_few_rows(const __grid_constant__ FewArgs a) {
  extern __shared__ __align__(16) uint8_t few_smem[];  // x as halves, [M, pitch]
  __shared__ float part[kFewWarps][16][8 * TILES + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, pitch = a.blocks * 128 + 8;
  // (rows past the end are others' again, and not stored)
  const int r0 = min(n0 + g, a.N - 1), r1 = min(n0 + g + 8, a.N - 1);
  const uint8_t *w0 = a.w + r0 * a.w_row, *w1 = a.w + r1 * a.w_row;
  const uint4 *x[TILES];
#pragma unroll
  for (int i = 0; i < TILES; ++i)
    x[i] = reinterpret_cast<const uint4 *>(few_smem + (min(8 * i + g, a.M - 1) * pitch + 16 * t) * 2);
  tc::dep_launch();
  tc::dep_wait();
  float sum[TILES][4] = {};
  struct Block {
    uint4 p[2], q[2];
    uint32_t s0, s1, e0, e1;  // (e0, e1: x's of the first eight rows)
  };
  const int c0 = min(2 * t, a.M - 1), c1 = min(2 * t + 1, a.M - 1);
  const uint8_t *x0 = a.sx.bytes + c0 * a.sx.row, *x1 = a.sx.bytes + c1 * a.sx.row;
  auto fetch = [&](int b, Block &f) {
    if (b * 128 + 128 <= a.K) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = b * 128 + 64 * h + 16 * t;
        f.p[h] = *reinterpret_cast<const uint4 *>(w0 + k), f.q[h] = *reinterpret_cast<const uint4 *>(w1 + k);
      }
    } else if (b < a.blocks) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = b * 128 + 64 * h + 16 * t;
        f.p[h] = sixteen(w0, k, a.K), f.q[h] = sixteen(w1, k, a.K);
      }
    }
    if constexpr (KIND != kRows) {
      f.s0 = f.s1 = f.e0 = f.e1 = 127u;
      if ((KIND == kBlocks || a.sw.bytes != nullptr) && b < a.blocks)
        f.s0 = a.sw.bytes[r0 * a.sw.row + b], f.s1 = a.sw.bytes[r1 * a.sw.row + b];
      if ((KIND == kBlocks || a.sx.bytes != nullptr) && b < a.blocks) f.e0 = x0[b], f.e1 = x1[b];
    }
  };
  auto multiply = [&](int b, const Block &f) {
    float acc[TILES][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 u[TILES][2];
#pragma unroll
      for (int i = 0; i < TILES; ++i) u[i][0] = x[i][b * 16 + 8 * h], u[i][1] = x[i][b * 16 + 8 * h + 1];
      const uint32_t pw[4] = {f.p[h].x, f.p[h].y, f.p[h].z, f.p[h].w}, qw[4] = {f.q[h].x, f.q[h].y, f.q[h].z, f.q[h].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t m[4] = {two_halves(pw[k], false), two_halves(qw[k], false), two_halves(pw[k], true),
                               two_halves(qw[k], true)};
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const uint4 &c = u[i][k >> 1];
          const uint32_t c0 = k & 1 ? c.z : c.x, c1 = k & 1 ? c.w : c.y;
          asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
              "{%8, %9}, {%0, %1, %2, %3};"
              : "+f"(acc[i][0]), "+f"(acc[i][1]), "+f"(acc[i][2]), "+f"(acc[i][3])
              : "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3]), "r"(c0), "r"(c1));
        }
      }
    }
    if constexpr (KIND == kRows) {
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] += acc[i][j];
    } else {
      uint32_t u0 = f.s0, u1 = f.s1;
      if (KIND == kMixed && a.sw.rows != nullptr) u0 = row_power(a.sw.rows[r0]), u1 = row_power(a.sw.rows[r1]);
      const bool far = is_far(u0) || is_far(u1);
      const float s0 = power(u0), s1 = power(u1);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const int c0 = min(8 * i + 2 * t, a.M - 1), c1 = min(8 * i + 2 * t + 1, a.M - 1);
        uint32_t e0 = f.e0, e1 = f.e1;
        if (i > 0 && (KIND == kBlocks || a.sx.bytes != nullptr))
          e0 = a.sx.bytes[c0 * a.sx.row + b], e1 = a.sx.bytes[c1 * a.sx.row + b];
        if (KIND == kMixed && a.sx.rows != nullptr) e0 = row_power(a.sx.rows[c0]), e1 = row_power(a.sx.rows[c1]);
        const float y0 = power(e0), y1 = power(e1);
        if (!far) {
          sum[i][0] = fmaf(acc[i][0] * s0, y0, sum[i][0]), sum[i][1] = fmaf(acc[i][1] * s0, y1, sum[i][1]);
          sum[i][2] = fmaf(acc[i][2] * s1, y0, sum[i][2]), sum[i][3] = fmaf(acc[i][3] * s1, y1, sum[i][3]);
        } else {
          sum[i][0] += by_powers(acc[i][0], s0, y0), sum[i][1] += by_powers(acc[i][1], s0, y1);
          sum[i][2] += by_powers(acc[i][2], s1, y0), sum[i][3] += by_powers(acc[i][3], s1, y1);
        }
      }
    }
  };
  // Three blocks in flight.
  const int per = (a.blocks + kFewWarps - 1) / kFewWarps, end = min(a.blocks, (warp + 1) * per);
  int b = warp * per;
  Block f0, f1, f2;
  fetch(b, f0), fetch(b + 1, f1);
  for (int i = threadIdx.x; i < a.M * a.blocks * 8; i += 32 * kFewWarps) {
    const int row = i / (a.blocks * 8), k = i % (a.blocks * 8) * 16;
    const uint4 c = sixteen(a.x + row * a.x_row, k, a.K);
    uint4 *to = reinterpret_cast<uint4 *>(few_smem + (row * pitch + k) * 2);
    to[0] = make_uint4(two_halves(c.x, false), two_halves(c.x, true), two_halves(c.y, false), two_halves(c.y, true));
    to[1] = make_uint4(two_halves(c.z, false), two_halves(c.z, true), two_halves(c.w, false), two_halves(c.w, true));
  }
  __syncthreads();
  for (; b < end; b += 3) {
    fetch(b + 2, f2);
    multiply(b, f0);
    if (b + 1 >= end) break;
    fetch(b + 3, f0);
    multiply(b + 1, f1);
    if (b + 2 >= end) break;
    fetch(b + 4, f1);
    multiply(b + 2, f2);
  }
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    part[warp][g][8 * i + 2 * t] = sum[i][0], part[warp][g][8 * i + 2 * t + 1] = sum[i][1];
    part[warp][g + 8][8 * i + 2 * t] = sum[i][2], part[warp][g + 8][8 * i + 2 * t + 1] = sum[i][3];
  }
  const int r = threadIdx.x & 15, m = threadIdx.x >> 4;
  float rx = 1.f, rw = 1.f;
  if (KIND == kRows || (KIND == kMixed && a.sx.rows != nullptr)) rx = a.sx.rows[min(m, a.M - 1)];
  if (KIND == kRows || (KIND == kMixed && a.sw.rows != nullptr)) rw = a.sw.rows[min(n0 + r, a.N - 1)];
  __syncthreads();
  if (m >= 8 * TILES || m >= a.M || n0 + r >= a.N) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < kFewWarps; ++k) v += part[k][r][m];
  if constexpr (KIND != kBlocks) v = v * row_rest(rx) * row_rest(rw);
  if constexpr (KIND == kRows) v = by_rows(v, rx, rw);
  if (a.bias != nullptr) v += to_f32(static_cast<const TB *>(a.bias)[n0 + r]);
  static_cast<T *>(a.y)[m * a.y_row + n0 + r] = from_f32<T>(v);
}

// Bytes of x as halves; few rows whose x takes more are left to the tiles, and so are
// large weights, for whose codes this kernel's conversions are too many.
int64_t few_bytes(int64_t M, int64_t K) { return M * ((K + kBlock - 1) / kBlock * 128 + 8) * 2; }
bool is_few(int64_t M, int64_t N, int64_t K) {
  return M <= kFewMost && few_bytes(M, K) <= 72 * 1024 && N * K <= int64_t(1) << (M <= 8 ? 24 : 22);
}

template <typename T, typename TB, int TILES, FewScales KIND>
cudaError_t launch_few_as(const FewArgs &a, cudaStream_t s) {
  auto *kernel = k_few_rows<T, TB, TILES, KIND>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024);
  if (e != cudaSuccess) return e;
  return tc::launch(kernel, (unsigned)((a.N + 15) / 16), 32 * kFewWarps, (size_t)few_bytes(a.M, a.K), 1, s, a);
}
template <typename T, typename TB>
cudaError_t launch_few(const FewArgs &a, cudaStream_t s) {
  const bool one = a.M <= 8;
  if (a.sx.rows == nullptr && a.sw.rows == nullptr)
    return one ? launch_few_as<T, TB, 1, kBlocks>(a, s) : launch_few_as<T, TB, 2, kBlocks>(a, s);
  if (a.sx.rows != nullptr && a.sw.rows != nullptr)
    return one ? launch_few_as<T, TB, 1, kRows>(a, s) : launch_few_as<T, TB, 2, kRows>(a, s);
  return one ? launch_few_as<T, TB, 1, kMixed>(a, s) : launch_few_as<T, TB, 2, kMixed>(a, s);
}

// What an operand lacks, or null; fills its scales.
const char *operand(const cpab_quantized &o, int64_t K, Scales *scales) {
  if (o.codes == nullptr || o.scale == nullptr) return "null codes or scales";
  if (reinterpret_cast<uintptr_t>(o.codes) % 16 || o.row % 16 || o.row < K)
    return "codes must begin on 16 bytes, each row on a multiple of 16 that holds it";
  *scales = {};
  if (o.scale_row == 0) {
    if (reinterpret_cast<uintptr_t>(o.scale) % 4) return "float32 scales must begin on 4 bytes";
    scales->rows = static_cast<const float *>(o.scale);
  } else {
    const int64_t n = (K + kBlock - 1) / kBlock;
    if (o.scale_row < n) return "a row of scales must hold one for each 128 codes";
    const bool words = reinterpret_cast<uintptr_t>(o.scale) % 4 == 0 && o.scale_row % 4 == 0;
    *scales = {static_cast<const uint8_t *>(o.scale), o.scale_row, words, nullptr};
  }
  return nullptr;
}

}  // namespace
}  // namespace cpab

using namespace cpab;

extern "C" int cpab_b200_set_wait_limit(int64_t nanoseconds) {
  if (nanoseconds < 0) return report_error(CPAB_ERR_ARG, "%s", "set_wait_limit: negative time");
  g_longest.store(nanoseconds);
  return report_error(CPAB_OK, "%s", "");
}

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
  if (rows > 0 && columns > 0) {
    if (q == nullptr && qt == nullptr && column_sum == nullptr)
      return report_error(CPAB_ERR_ARG, "%s", "quantize_blocks: nothing to write");
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
  cudaError_t e = cudaSuccess;
  if (rows > 0 && columns > 0) {
    const QuantizeArgs a = {x, x_row, rows, columns, q, scale, q_row, scale_row, qt, scale_t, qt_row, scale_t_row,
                            column_sum != nullptr ? workspace : nullptr};
    const unsigned grid = (unsigned)(tiles_x * tiles_y);
    e = dtype == CPAB_F32   ? launch_quantize<float>(a, grid, s)
        : dtype == CPAB_F16 ? launch_quantize<__half>(a, grid, s)
                            : launch_quantize<__nv_bfloat16>(a, grid, s);
  }
  if (e == cudaSuccess && column_sum != nullptr && columns > 0) {
    const unsigned grid = (unsigned)((columns + 31) / 32);
    const int64_t n = rows > 0 ? tiles_y : 0;
    if (sum_dtype == CPAB_F32) e = tc::launch(k_sum_tiles<float>, grid, 256, 0, 1, s, static_cast<const float *>(workspace), n, columns, static_cast<float *>(column_sum));
    else if (sum_dtype == CPAB_F16) e = tc::launch(k_sum_tiles<__half>, grid, 256, 0, 1, s, static_cast<const float *>(workspace), n, columns, static_cast<__half *>(column_sum));
    else e = tc::launch(k_sum_tiles<__nv_bfloat16>, grid, 256, 0, 1, s, static_cast<const float *>(workspace), n, columns, static_cast<__nv_bfloat16 *>(column_sum));
  }
  return launch_status(e, "quantize_blocks");
}

extern "C" int cpab_b200_lay_out_codes(int count, const uint8_t *const *src, const int64_t *src_row,
                                       const int64_t *rows, uint8_t *const *dst, int64_t K, cpab_stream_t stream) {
  if (count < 0 || count > 2 || K < 1 || (count > 0 && (src == nullptr || src_row == nullptr || rows == nullptr || dst == nullptr)))
    return report_error(CPAB_ERR_ARG, "%s", "lay_out_codes: one or two matrices of rows of codes");
  LayoutArgs a = {};
  a.K = K, a.groups = (K + 15) / 16;
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 0 || src_row[i] < 0 || (rows[i] > 0 && (src[i] == nullptr || dst[i] == nullptr)) ||
        reinterpret_cast<uintptr_t>(dst[i]) % 16)
      return report_error(CPAB_ERR_ARG, "%s", "lay_out_codes: null codes, negative sizes, or a destination off 16 bytes");
    if (rows[i] > kMostSize || K > kMostSize) return report_error(CPAB_ERR_SIZE, "%s", "lay_out_codes: sizes too large");
    a.src[i] = src[i], a.dst[i] = dst[i], a.src_row[i] = src_row[i], a.rows[i] = rows[i];
    most = std::max(most, rows[i] * a.groups);
  }
  if (most == 0) return report_error(CPAB_OK, "%s", "");
  const int64_t blocks = std::min<int64_t>((most + 255) / 256, 16 * device_info().sm_count);
  return launch_status(tc::launch(k_lay_out, dim3((unsigned)blocks, (unsigned)count), 256, 0, 1,
                                  reinterpret_cast<cudaStream_t>(stream), a),
                       "lay_out_codes");
}

extern "C" int64_t cpab_b200_matmul_quantized_workspace(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1 || M > kMostSize || N > kMostSize || K > kMostSize || is_few(M, N, K)) return 0;
  const Split split = split_of(M, N, (K + kBlock - 1) / kBlock);
  return split.splits > 1 ? split.splits * M * ((N + 15) / 16 * 16) : 0;
}

extern "C" int cpab_b200_matmul_quantized(int dtype, const cpab_quantized *x, const cpab_quantized *weight, int64_t M,
                                          int64_t N, int64_t K, int bias_dtype, const void *bias, void *y,
                                          int64_t y_row, float *workspace, cpab_stream_t stream) {
  if (!dtype_ok(dtype) || (bias != nullptr && bias_dtype != CPAB_F32 && bias_dtype != dtype))
    return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: unknown element type, or a bias of neither y's nor float32");
  if (x == nullptr || weight == nullptr) return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: null operand");
  if (M < 0 || N < 0 || K < 1 || y_row < N) return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: sizes out of range");
  if (M > kMostSize || N > kMostSize || K > kMostSize || (M + 127) / 128 * ((N + 63) / 64) >= kMostSize)
    return report_error(CPAB_ERR_SIZE, "%s", "matmul_quantized: sizes too large");
  if (M == 0 || N == 0) return report_error(CPAB_OK, "%s", "");
  if (y == nullptr) return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: null y");
  ProductArgs a = {};
  const char *why = operand(*x, K, &a.sa);
  if (why == nullptr) why = operand(*weight, K, &a.sb);
  if (why == nullptr && !is_few(M, N, K)) {
    const int tile = tile_of(M, N, (K + kBlock - 1) / kBlock), columns = tile == 0 ? 64 : 128;  // of B a block loads
    a.a_rows = tile == 2 || M > 64 ? 128 : M > 32 ? 64 : M > 16 ? 32 : 16;
    if (!make_tile_map(&a.a, false, x->codes, K, M, 1, x->row, x->row * M, a.a_rows) ||
        !make_tile_map(&a.b, false, weight->codes, K, N, 1, weight->row, weight->row * N, columns))
      why = "no tensor map for the codes";
  }
  if (why != nullptr) return report_error(CPAB_ERR_ARG, "matmul_quantized: %s", why);
  a.bias = bias, a.y = y, a.y_row = y_row, a.M = (int)M, a.N = (int)N, a.steps = (int)((K + kBlock - 1) / kBlock);
  a.wide = aligned_to(y, y_row, dtype_size(dtype), 16);
  const Split split = split_of(M, N, a.steps);
  a.splits = split.splits, a.each = split.each, a.parts = workspace, a.pitch = (N + 15) / 16 * 16;
  if (!is_few(M, N, K) && a.splits > 1 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 32))
    return report_error(CPAB_ERR_ARG, "%s", "matmul_quantized: a null workspace, or one off 32 bytes");
  if (tc::gave_up()) return tc::report_gave_up("matmul_quantized");
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (is_few(M, N, K)) {
    const FewArgs f = {x->codes, weight->codes, x->row, weight->row, a.sa, a.sb, bias, y, y_row,
                       (int)M, (int)N, (int)K, a.steps};
    if (dtype == CPAB_F32) e = launch_few<float, float>(f, s);
    else if (dtype == CPAB_F16) e = bias_dtype == CPAB_F32 ? launch_few<__half, float>(f, s) : launch_few<__half, __half>(f, s);
    else e = bias_dtype == CPAB_F32 ? launch_few<__nv_bfloat16, float>(f, s)
                                    : launch_few<__nv_bfloat16, __nv_bfloat16>(f, s);
    return launch_status(e, "matmul_quantized");
  }
  a.waits = tc::waits();
  if (dtype == CPAB_F32) e = launch_product<float, float>(a, s);
  else if (dtype == CPAB_F16)
    e = bias_dtype == CPAB_F32 ? launch_product<__half, float>(a, s) : launch_product<__half, __half>(a, s);
  else e = bias_dtype == CPAB_F32 ? launch_product<__nv_bfloat16, float>(a, s)
                                  : launch_product<__nv_bfloat16, __nv_bfloat16>(a, s);
  return launch_status(e, "matmul_quantized");
}
