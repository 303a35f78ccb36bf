// Root-mean-square norm of a residual stream, its gradient, and its form with
// an 8-bit output.
//
//   s = x + residual (rounded to the stream's type, which is what is kept),
//   y = s r w,  r = (mean(s^2) + eps)^(-1/2)   per row of D columns
//
//   ds = gs + r (w dy - s r^2 mean(w dy s)),  dw = sum over rows of dy s r
//
// The 8-bit form gives e4m3 codes q and one scale per row: scale =
// max(max|y| / 448, 2^-126), q = y / scale rounded to nearest.
//
// A row is held in the registers of 1 to 512 threads between its one read and
// its one write; sums are float32, over lanes by shuffles and over warps in
// shared memory.  The weight's gradient is summed per thread over the rows a
// block visits, then over blocks in a second kernel in a fixed order (same
// result every run; no atomics).
#include <cuda_fp8.h>

#include "sequence.cuh"

namespace cpab {
namespace {

constexpr int kBlock = 256;        // threads of a block whose rows take fewer
constexpr int kMost = 512;         // threads of a row at most
constexpr int64_t kMaxWidth = 16384;
constexpr float kE4m3Max = 448.0f;

struct NormArgs {
  const void *x, *res;
  int64_t xs, rs;          // row strides of x and residual, in elements
  const void *w;
  int w_f32;               // the weight is float32 (else of x's type)
  int64_t rows, D;
  float eps;
  void *y, *s;             // [rows, D]; s null without a residual
  float *r;                // [rows] or null
  uint8_t *q;
  float *scale;
  // gradient
  const void *dy, *gs;     // [rows, D]; gs null when none flows into s
  void *dx, *dres;         // dres null when dx's type is the stream's
  float *partial;          // [blocks, D]
  int threads;             // of a row
};

// Sum (or maximum) over the `n` threads (a power of two) that share a row.
template <bool MAX>
__device__ __forceinline__ float over_row(float v, int n, float *shared) {
  const int width = n < 32 ? n : 32;
  for (int o = width / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(~0u, v, o);
    if (MAX) asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(u));
    else v += u;
  }
  if (n <= 32) return v;
  const int warp = threadIdx.x >> 5, first = (threadIdx.x / n) * (n >> 5);
  if ((threadIdx.x & 31) == 0) shared[warp] = v;
  __syncthreads();
  v = shared[first];
  for (int k = 1; k < n >> 5; ++k) {
    const float u = shared[first + k];
    if (MAX) asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(u));
    else v += u;
  }
  __syncthreads();
  return v;
}

// VEC consecutive elements as loaded: half the registers of their float32
// values where T has 16 bits.
template <typename T, int VEC>
struct Row {
  static constexpr int N = sizeof(T) * VEC > 16 ? 16 / sizeof(T) : VEC;  // at most 16 bytes at a time
  Pack<T, N> part[VEC / N];
  __device__ __forceinline__ void load(const void *base, int64_t at) {
#pragma unroll
    for (int k = 0; k < VEC / N; ++k)
      part[k] = *reinterpret_cast<const Pack<T, N> *>(static_cast<const T *>(base) + at + k * N);
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32(part[i / N].v[i % N]); }
};

template <typename T, int VEC>
__device__ __forceinline__ void load_f32(const void *base, int64_t at, float (&out)[VEC]) {
  Row<T, VEC> r;
  r.load(base, at);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = r[i];
}

template <typename T, int VEC>
__device__ __forceinline__ void store_f32(void *base, int64_t at, const float (&in)[VEC]) {
  constexpr int N = sizeof(T) * VEC > 16 ? 16 / sizeof(T) : VEC;
#pragma unroll
  for (int k = 0; k < VEC; k += N) {
    Pack<T, N> p;
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = from_f32<T>(in[k + i]);
    *reinterpret_cast<Pack<T, N> *>(static_cast<T *>(base) + at + k) = p;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const NormArgs &p, int64_t at, float (&w)[VEC]) {
  if (p.w_f32) load_f32<float, VEC>(p.w, at, w);
  else load_f32<T, VEC>(p.w, at, w);
}

// T: x and y; S: the stream.
template <typename T, typename S, int VEC, int NV, bool QUANT>
__global__ void __launch_bounds__(kMost) k_norm(NormArgs p) {
  __shared__ float shared[kMost / 32];
  const int n = p.threads, j = threadIdx.x % n;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / n) + threadIdx.x / n;
  const bool on = row < p.rows;
  float v[NV][VEC];
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * n + j) * VEC;
    if (on && c < p.D) {
      load_f32<T, VEC>(p.x, row * p.xs + c, v[k]);
      if (p.res != nullptr) {
        float r[VEC];
        load_f32<S, VEC>(p.res, row * p.rs + c, r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] = to_f32(from_f32<S>(v[k][i] + r[i]));
        store_f32<S, VEC>(p.s, row * p.D + c, v[k]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum = fmaf(v[k][i], v[k][i], sum);
    }
  }
  const float mean = over_row<false>(sum, n, shared) / (float)p.D;
  const float r = rsqrtf(mean + p.eps);
  if (on && p.r != nullptr && j == 0) p.r[row] = r;
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * n + j) * VEC;
    if (on && c < p.D) {
      float w[VEC];
      load_weight<T, VEC>(p, c, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[k][i] = v[k][i] * r * w[i];
        if (QUANT) asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(fabsf(v[k][i])));
      }
      if (!QUANT) store_f32<T, VEC>(p.y, row * p.D + c, v[k]);
    }
  }
  if (!QUANT) return;
  // Never zero: a row of zeros has codes 0, and a reader may divide by it.
  float scale = over_row<true>(top, n, shared) * (1.0f / kE4m3Max);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(scale) : "f"(scale), "f"(1.17549435e-38f));
  if (on && j == 0) p.scale[row] = scale;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * n + j) * VEC;
    if (on && c < p.D) {
      Pack<uint8_t, VEC> q;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        q.v[i] = __nv_cvt_float_to_fp8(v[k][i] / scale, __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<Pack<uint8_t, VEC> *>(p.q + row * p.D + c) = q;
    }
  }
}

// x here is the stream s as kept (x itself without a residual), of type S.
template <typename T, typename S, int VEC, int NV>
__global__ void __launch_bounds__(kMost) k_norm_backward(NormArgs p) {
  __shared__ float shared[kMost / 32];
  const int n = p.threads, j = threadIdx.x % n, group = threadIdx.x / n, groups = blockDim.x / n;
  float dw[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = 0.0f;
  for (int64_t first = (int64_t)blockIdx.x * groups; first < p.rows; first += (int64_t)gridDim.x * groups) {
    const int64_t row = first + group;
    const bool on = row < p.rows;
    const float r = on ? p.r[row] : 0.0f;
    Row<S, VEC> v[NV];
    Row<T, VEC> g[NV];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * n + j) * VEC;
      if (on && c < p.D) {
        v[k].load(p.x, row * p.xs + c);
        g[k].load(p.dy, row * p.D + c);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * n + j) * VEC;
      if (on && c < p.D) {
        float w[VEC];
        load_weight<T, VEC>(p, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float gi = g[k][i], vi = v[k][i];
          dw[k][i] = fmaf(gi, vi * r, dw[k][i]);
          sum = fmaf(gi * w[i], vi, sum);
        }
      }
    }
    const float m = over_row<false>(sum, n, shared) / (float)p.D * (r * r);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = (int64_t)(k * n + j) * VEC;
      if (on && c < p.D) {
        float w[VEC], d[VEC];
        load_weight<T, VEC>(p, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] = r * (g[k][i] * w[i] - v[k][i] * m);
        if (p.gs != nullptr) {
          float a[VEC];
          load_f32<S, VEC>(p.gs, row * p.D + c, a);
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[i] += a[i];
        }
        store_f32<T, VEC>(p.dx, row * p.D + c, d);
        if (p.dres != nullptr) store_f32<S, VEC>(p.dres, row * p.D + c, d);
      }
    }
  }
  if (p.partial == nullptr) return;
  // The block's groups hold the same columns: added one after another.
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t c = (int64_t)(k * n + j) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (c < p.D)
        p.partial[((int64_t)blockIdx.x * groups + group) * p.D + c + i] = dw[k][i];
    }
  }
}

// dw = the sum over the partial rows, 32 columns a block.
template <typename W>
__global__ void __launch_bounds__(1024) k_norm_weight(const float *partial, int64_t n, int64_t D, W *dw) {
  __shared__ float part[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float sum = 0.0f;
  if (c < D)
    for (int64_t k = threadIdx.y; k < n; k += 32) sum += partial[k * D + c];
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < D) {
    float s = 0.0f;
    for (int k = 0; k < 32; ++k) s += part[k][threadIdx.x];
    dw[c] = from_f32<W>(s);
  }
}

// A row's vectors and threads: enough threads (a power of two) that each holds
// at most `most` vectors.
struct Shape {
  int threads, block;
  int per;            // vectors a thread holds
};

Shape shape_of(int64_t D, int vec, int most) {
  const int64_t vectors = (D + vec - 1) / vec;
  Shape s;
  s.threads = 1;
  while (s.threads < kMost && (int64_t)s.threads * most < vectors) s.threads *= 2;
  s.per = (int)((vectors + s.threads - 1) / s.threads);
  s.block = s.threads < kBlock ? kBlock : s.threads;
  return s;
}

constexpr int most_of(int vec) { return vec > 1 ? 2 : 4; }

int64_t backward_rows(int64_t rows, const Shape &s) {
  const int groups = s.block / s.threads;
  const int64_t want = (rows + groups - 1) / groups;
  const int64_t cap = 148 * 2;
  return (want < cap ? want : cap) * groups;
}

template <typename T, typename S, int VEC, int NV>
cudaError_t norm_launch(const NormArgs &a, const Shape &s, bool quant, cudaStream_t stream) {
  const int groups = s.block / s.threads;
  const unsigned grid = (unsigned)((a.rows + groups - 1) / groups);
  if (quant) k_norm<T, S, VEC, NV, true><<<grid, s.block, 0, stream>>>(a);
  else k_norm<T, S, VEC, NV, false><<<grid, s.block, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename S, int VEC, int NV>
cudaError_t norm_backward_launch(const NormArgs &a, const Shape &s, cudaStream_t stream) {
  const unsigned grid = (unsigned)(backward_rows(a.rows, s) / (s.block / s.threads));
  k_norm_backward<T, S, VEC, NV><<<grid, s.block, 0, stream>>>(a);
  return cudaGetLastError();
}

// The kernel for s.per vectors a thread; kMaxWidth / kMost elements at most.
template <typename T, typename S, int VEC>
cudaError_t norm_vec(NormArgs a, bool quant, cudaStream_t stream) {
  const Shape s = shape_of(a.D, VEC, most_of(VEC));
  constexpr int kAll = (int)(kMaxWidth / kMost) / VEC;
  a.threads = s.threads;
  if (s.per <= 1) return norm_launch<T, S, VEC, 1>(a, s, quant, stream);
  if (s.per <= 2) return norm_launch<T, S, VEC, 2>(a, s, quant, stream);
  if (s.per <= 4) return norm_launch<T, S, VEC, 4>(a, s, quant, stream);
  return norm_launch<T, S, VEC, kAll>(a, s, quant, stream);
}

template <typename T, typename S, int VEC>
cudaError_t norm_backward_vec(NormArgs a, cudaStream_t stream) {
  const Shape s = shape_of(a.D, VEC, most_of(VEC));
  constexpr int kAll = (int)(kMaxWidth / kMost) / VEC;
  a.threads = s.threads;
  if (s.per <= 1) return norm_backward_launch<T, S, VEC, 1>(a, s, stream);
  if (s.per <= 2) return norm_backward_launch<T, S, VEC, 2>(a, s, stream);
  if (s.per <= 4) return norm_backward_launch<T, S, VEC, 4>(a, s, stream);
  return norm_backward_launch<T, S, VEC, kAll>(a, s, stream);
}

// Elements a 16-byte access of T moves; rows that do not allow it go one
// element at a time.
template <typename T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }

template <typename T, typename S>
cudaError_t norm_as(const NormArgs &a, bool wide, bool quant, cudaStream_t stream) {
  return wide ? norm_vec<T, S, vec_of<T>()>(a, quant, stream) : norm_vec<T, S, 1>(a, quant, stream);
}

template <typename T, typename S>
cudaError_t norm_backward_as(const NormArgs &a, bool wide, cudaStream_t stream) {
  return wide ? norm_backward_vec<T, S, vec_of<T>()>(a, stream) : norm_backward_vec<T, S, 1>(a, stream);
}

bool wide_rows(const NormArgs &a, int e, int f) {
  const int vec = 16 / e;
  return a.D % vec == 0 && aligned_to(a.x, a.xs, e, 16) && aligned_to(a.res, a.rs, f, 16) &&
         aligned_to(a.w, 0, 4, 16) && aligned_to(a.y, 0, e, 16) && aligned_to(a.s, 0, f, 16) &&
         aligned_to(a.q, 0, 1, vec) && aligned_to(a.dy, 0, e, 16) && aligned_to(a.gs, 0, f, 16) &&
         aligned_to(a.dx, 0, e, 16) && aligned_to(a.dres, 0, f, 16);
}

int check_norm(const char *fn, int dtype, int stream_dtype, int w_dtype, int64_t rows, int64_t D, float eps) {
  if (!dtype_ok(dtype) || (stream_dtype != dtype && stream_dtype != CPAB_F32) ||
      (w_dtype != dtype && w_dtype != CPAB_F32))
    return report_error(CPAB_ERR_ARG, "%s: unsupported types (x %d, stream %d, weight %d)", fn, dtype,
                        stream_dtype, w_dtype);
  if (rows < 0 || D < 1) return report_error(CPAB_ERR_ARG, "%s: bad shape", fn);
  if (D > kMaxWidth)
    return report_error(CPAB_ERR_SIZE, "%s: rows of at most %lld columns are supported, got %lld", fn,
                        (long long)kMaxWidth, (long long)D);
  if (rows >= (int64_t(1) << 31)) return report_error(CPAB_ERR_SIZE, "%s: too many rows", fn);
  if (!(eps >= 0.0f)) return report_error(CPAB_ERR_ARG, "%s: eps must not be negative", fn);
  return CPAB_OK;
}

template <typename F32, typename F16, typename BF16, typename M16, typename MBF>
cudaError_t by_type(int dtype, int stream_dtype, F32 f32, F16 f16, BF16 bf16, M16 m16, MBF mbf) {
  if (dtype == CPAB_F32) return f32();
  if (stream_dtype == CPAB_F32) return dtype == CPAB_F16 ? m16() : mbf();
  return dtype == CPAB_F16 ? f16() : bf16();
}

int forward(const char *fn, int dtype, int stream_dtype, int w_dtype, NormArgs a, bool quant,
            cudaStream_t stream) {
  const bool wide = wide_rows(a, dtype_size(dtype), dtype_size(stream_dtype));
  a.w_f32 = w_dtype == CPAB_F32;
  using H = __half;
  using B = __nv_bfloat16;
  return launch_status(by_type(dtype, stream_dtype, [&] { return norm_as<float, float>(a, wide, quant, stream); },
                               [&] { return norm_as<H, H>(a, wide, quant, stream); },
                               [&] { return norm_as<B, B>(a, wide, quant, stream); },
                               [&] { return norm_as<H, float>(a, wide, quant, stream); },
                               [&] { return norm_as<B, float>(a, wide, quant, stream); }),
                       fn);
}

}  // namespace
}  // namespace cpab

using namespace cpab;

extern "C" int cpab_b200_rms_norm(int dtype, int stream_dtype, int weight_dtype, const void *x,
                                  int64_t x_row, const void *residual, int64_t residual_row,
                                  const void *weight, int64_t rows, int64_t D, float eps, void *y,
                                  void *sum, float *rstd, cpab_stream_t stream) {
  const int st = check_norm("rms_norm", dtype, stream_dtype, weight_dtype, rows, D, eps);
  if (st != CPAB_OK) return st;
  if (rows == 0) return launch_status(cudaSuccess, "");
  if (x == nullptr || weight == nullptr || y == nullptr || (residual != nullptr && sum == nullptr))
    return report_error(CPAB_ERR_ARG, "rms_norm: null pointer");
  NormArgs a{};
  a.x = x, a.xs = x_row, a.res = residual, a.rs = residual_row, a.w = weight, a.rows = rows, a.D = D;
  a.eps = eps, a.y = y, a.s = sum, a.r = rstd;
  return forward("rms_norm", dtype, stream_dtype, weight_dtype, a, false, stream);
}

extern "C" int cpab_b200_rms_norm_quantized(int dtype, int stream_dtype, int weight_dtype,
                                            const void *x, int64_t x_row, const void *residual,
                                            int64_t residual_row, const void *weight, int64_t rows,
                                            int64_t D, float eps, uint8_t *q, float *scale,
                                            void *sum, cpab_stream_t stream) {
  const int st = check_norm("rms_norm_quantized", dtype, stream_dtype, weight_dtype, rows, D, eps);
  if (st != CPAB_OK) return st;
  if (rows == 0) return launch_status(cudaSuccess, "");
  if (x == nullptr || weight == nullptr || q == nullptr || scale == nullptr ||
      (residual != nullptr && sum == nullptr))
    return report_error(CPAB_ERR_ARG, "rms_norm_quantized: null pointer");
  NormArgs a{};
  a.x = x, a.xs = x_row, a.res = residual, a.rs = residual_row, a.w = weight, a.rows = rows, a.D = D;
  a.eps = eps, a.q = q, a.scale = scale, a.s = sum;
  return forward("rms_norm_quantized", dtype, stream_dtype, weight_dtype, a, true, stream);
}

extern "C" int64_t cpab_b200_rms_norm_workspace(int dtype, int64_t rows, int64_t D) {
  if (!dtype_ok(dtype) || rows < 1 || D < 1 || D > kMaxWidth) return 0;
  // The scalar and the vector kernel's blocks hold different numbers of rows.
  const int64_t one = backward_rows(rows, shape_of(D, 1, most_of(1)));
  const int64_t wide = backward_rows(rows, shape_of(D, 16 / dtype_size(dtype), most_of(16 / dtype_size(dtype))));
  return (one > wide ? one : wide) * D;
}

extern "C" int cpab_b200_rms_norm_backward(int dtype, int stream_dtype, int weight_dtype,
                                           const void *sum, int64_t sum_row, const void *weight,
                                           const float *rstd, int64_t rows, int64_t D,
                                           const void *grad_y, const void *grad_sum, void *grad_x,
                                           void *grad_residual, float *workspace, void *grad_weight,
                                           cpab_stream_t stream) {
  const int st = check_norm("rms_norm_backward", dtype, stream_dtype, weight_dtype, rows, D, 0.0f);
  if (st != CPAB_OK) return st;
  if (grad_weight != nullptr && rows > 0 && workspace == nullptr)
    return report_error(CPAB_ERR_ARG, "rms_norm_backward: null workspace");
  if (rows == 0) {
    if (grad_weight == nullptr) return launch_status(cudaSuccess, "");
    return launch_status(cudaMemsetAsync(grad_weight, 0, D * dtype_size(weight_dtype), stream),
                         "rms_norm_backward");
  }
  if (sum == nullptr || weight == nullptr || rstd == nullptr || grad_y == nullptr || grad_x == nullptr)
    return report_error(CPAB_ERR_ARG, "rms_norm_backward: null pointer");
  if (grad_residual != nullptr && stream_dtype == dtype)
    return report_error(CPAB_ERR_ARG, "rms_norm_backward: grad_residual is grad_x where the types are one");
  NormArgs a{};
  a.x = sum, a.xs = sum_row, a.w = weight, a.w_f32 = weight_dtype == CPAB_F32;
  a.r = const_cast<float *>(rstd), a.rows = rows, a.D = D, a.dy = grad_y, a.gs = grad_sum;
  a.dx = grad_x, a.dres = grad_residual, a.partial = grad_weight != nullptr ? workspace : nullptr;
  const int e = dtype_size(dtype), f = dtype_size(stream_dtype);
  const bool wide = wide_rows(a, e, f) && aligned_to(sum, sum_row, f, 16);
  using H = __half;
  using B = __nv_bfloat16;
  const cudaError_t err = by_type(dtype, stream_dtype, [&] { return norm_backward_as<float, float>(a, wide, stream); },
                            [&] { return norm_backward_as<H, H>(a, wide, stream); },
                            [&] { return norm_backward_as<B, B>(a, wide, stream); },
                            [&] { return norm_backward_as<H, float>(a, wide, stream); },
                            [&] { return norm_backward_as<B, float>(a, wide, stream); });
  if (err != cudaSuccess || grad_weight == nullptr) return launch_status(err, "rms_norm_backward");
  const int vec = wide ? 16 / e : 1;
  const Shape s = shape_of(D, vec, most_of(vec));
  const int64_t n = backward_rows(rows, s);
  const unsigned grid = (unsigned)((D + 31) / 32);
  const dim3 block(32, 32);
  if (weight_dtype == CPAB_F32)
    k_norm_weight<float><<<grid, block, 0, stream>>>(workspace, n, D, (float *)grad_weight);
  else if (weight_dtype == CPAB_F16)
    k_norm_weight<__half><<<grid, block, 0, stream>>>(workspace, n, D, (__half *)grad_weight);
  else
    k_norm_weight<__nv_bfloat16><<<grid, block, 0, stream>>>(workspace, n, D, (__nv_bfloat16 *)grad_weight);
  return launch_status(cudaGetLastError(), "rms_norm_backward");
}
