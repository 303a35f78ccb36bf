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
//
// Rows on vectors, of up to 8192 columns, are bound by memory: 32768x4096 bf16 with a
// residual moves 1.07 GB each way, the forward in 160 us (6.7 TB/s; a copy: 6.46), the
// gradient in 193 (5.6 TB/s: beside the row it holds its weights' sums, which leaves
// 768 threads on an SM; in float32, with half as many elements a thread, 6.5).  Other
// rows take longer for their bytes: inside vectors the masks (65536x999: 66% of the
// issue slots), of over 8192 columns 512 threads on an SM and, of float32 inside
// vectors, spills (4096x13209: 42% and 30% of the issue slots, 3.9 and 2.9 TB/s).
// Means are sums times the rounded 1 / D (at most 2^-25 of r).
#include <cuda_fp8.h>

#include <type_traits>

#include "sequence.cuh"

namespace cpab {
namespace {

constexpr int kBlock = 256;        // threads of a block whose rows take fewer
constexpr int kMost = 512;         // threads of a row at most
// Threads of an SM that the gradient's registers leave room for, by the elements a
// thread holds.  (32768x4096 bf16, 16 elements: 228 us at 512 threads, 193 at 768,
// 225 at 1024; 32768x2048 f32, 8 elements: 209, 176 and 165 us.)
__host__ __device__ constexpr int resident_of(int elements) { return elements <= 8 ? 1024 : elements <= 16 ? 768 : 512; }
constexpr int64_t kMaxWidth = 16384;
constexpr float kE4m3Max = 448.0f;
constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the smallest scale

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
  int threads_log2;        // of a row
  float inverse;           // 1 / D
};

// Sum of `sum` (and maximum of `top`) over the 2^log2 threads that share a row.
// `shared` is another half for every second row, so one barrier a row is enough.
template <bool TOP>
__device__ __forceinline__ void over_row(float &sum, float &top, int log2, float *shared) {
  for (int o = log2 < 5 ? (1 << log2) >> 1 : 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, o);
    if (TOP) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  }
  if (log2 <= 5) return;
  constexpr int kWarps = kMost / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = 1 << (log2 - 5);
  if (lane == 0) {
    shared[warp] = sum;
    if (TOP) shared[kWarps + warp] = top;
  }
  __syncthreads();
  if (warps == 2) {  // (the shuffles after cost 1536 columns 15%: 124 -> 142 us for 65537 rows)
    sum = shared[warp & ~1] + shared[warp | 1];
    if (TOP) top = fmaxf(shared[kWarps + (warp & ~1)], shared[kWarps + (warp | 1)]);
    return;
  }
  const int from = (warp & -warps) + (lane & (warps - 1));
  sum = shared[from];
  if (TOP) top = shared[kWarps + from];
  for (int o = warps >> 1; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, o);
    if (TOP) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  }
}

// VEC consecutive elements as they lie in memory: words of one float32 or two
// 16-bit elements (VEC 1: one element's bits).
template <typename T, int VEC>
struct Row {
  static constexpr int kPer = VEC == 1 ? 1 : 4 / (int)sizeof(T), kWords = VEC / kPer;
  uint32_t w[kWords];
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;

  __device__ __forceinline__ void load(const T *at) {
    if constexpr (VEC == 1) {
      w[0] = *reinterpret_cast<const Bits *>(at);
    } else {
      constexpr int N = kWords > 4 ? 4 : kWords;  // words of an access
#pragma unroll
      for (int k = 0; k < kWords; k += N) {
        const Pack<uint32_t, N> p = *reinterpret_cast<const Pack<uint32_t, N> *>(at + k * kPer);
#pragma unroll
        for (int i = 0; i < N; ++i) w[k + i] = p.v[i];
      }
    }
  }
  __device__ __forceinline__ void store(T *at) const {
    if constexpr (VEC == 1) {
      *reinterpret_cast<Bits *>(at) = (Bits)w[0];
    } else {
      constexpr int N = kWords > 4 ? 4 : kWords;
#pragma unroll
      for (int k = 0; k < kWords; k += N) {
        Pack<uint32_t, N> p;
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = w[k + i];
        *reinterpret_cast<Pack<uint32_t, N> *>(at + k * kPer) = p;
      }
    }
  }
  // Elements lo .. hi - 1 one by one, zeros around them.
  __device__ __forceinline__ void load_some(const T *at, int lo, int hi) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= lo && i < hi) w[i / kPer] |= (uint32_t)reinterpret_cast<const Bits *>(at)[i] << (16 * (i % kPer));
  }
  __device__ __forceinline__ void store_some(T *at, int lo, int hi) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= lo && i < hi) reinterpret_cast<Bits *>(at)[i] = (Bits)(w[i / kPer] >> (16 * (i % kPer)));
  }
  __device__ __forceinline__ void zero_outside(int lo, int hi) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < lo || i >= hi) w[i / kPer] &= kPer == 2 ? 0xFFFF0000u >> (16 * (i % 2)) : 0u;
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (VEC == 1) {
      return unpack_pair<T>(w[0]).x;
    } else {
      return i % 2 ? unpack_pair<T>(w[i / 2]).y : unpack_pair<T>(w[i / 2]).x;
    }
  }
  __device__ __forceinline__ void set(const float (&f)[VEC]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
      else if constexpr (VEC == 1) w[0] = pack_pair<T>(f[0], 0.0f);
      else w[i] = pack_pair<T>(f[2 * i], f[2 * i + 1]);
    }
  }
};

// The stream's new value x + residual, rounded to its type.
template <typename T, typename S, int VEC>
__device__ __forceinline__ void add_to(Row<S, VEC> &res, const Row<T, VEC> &x) {
  if constexpr (sizeof(S) == 2) {
#pragma unroll
    for (int i = 0; i < Row<S, VEC>::kWords; ++i) res.w[i] = add_pair<S>(x.w[i], res.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) res.w[i] = __float_as_uint(x[i] + res[i]);
  }
}

// A thread's vector of a row: elements lo .. hi - 1 of the vector are columns
// c + lo .. c + hi - 1 of the row (all of them, or with EDGE fewer at a row's
// ends).
struct Span {
  int c, lo, hi;
  __device__ __forceinline__ bool any() const { return hi > lo; }
};

// Where rows do not begin on a vector, all tensors' rows begin as many elements
// (`shift`) after one, and the vectors that hold a row are taken as they lie:
// those at its ends hold elements of the rows beside it too, which mask_span makes
// zeros (later: a thread's loads do not wait for one another).  Only past the last
// row there may be nothing to read (rows do not overlap: lie_of).
template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ void load_span(Row<T, VEC> &r, const T *row, const Span &s, bool last) {
  if (EDGE && last && s.hi < VEC) r.load_some(row + s.c, s.lo, s.hi);
  else r.load(row + s.c);
}

template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ void mask_span(Row<T, VEC> &r, const Span &s) {
  if (EDGE && (s.lo > 0 || s.hi < VEC)) r.zero_outside(s.lo, s.hi);
}

template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ void store_span(T *row, const Span &s, const Row<T, VEC> &r) {
  if (!EDGE || (s.lo == 0 && s.hi == VEC)) r.store(row + s.c);
  else r.store_some(row + s.c, s.lo, s.hi);
}

template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ void store_span(T *row, const Span &s, const float (&in)[VEC]) {
  Row<T, VEC> r;
  r.set(in);
  store_span<T, VEC, EDGE>(row, s, r);
}

template <typename T, int VEC, bool EDGE>
__device__ __forceinline__ void load_weight(const NormArgs &p, const Span &s, float (&w)[VEC]) {
  if constexpr (!EDGE) {
    if (p.w_f32) {
      Row<float, VEC> r;
      r.load(static_cast<const float *>(p.w) + s.c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = r[i];
    } else {
      Row<T, VEC> r;
      r.load(static_cast<const T *>(p.w) + s.c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = r[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w[i] = 0.0f;
      if (i >= s.lo && i < s.hi)
        w[i] = p.w_f32 ? static_cast<const float *>(p.w)[s.c + i] : to_f32(static_cast<const T *>(p.w)[s.c + i]);
    }
  }
}

// Vector v of a row of D columns that begins `shift` elements into one.
template <int VEC, bool EDGE>
__device__ __forceinline__ Span span_of(int v, int shift, int D) {
  Span s;
  s.c = v * VEC - (EDGE ? shift : 0);
  s.lo = EDGE ? max(0, -s.c) : 0;
  s.hi = EDGE ? max(0, min(VEC, D - s.c)) : (s.c < D ? VEC : 0);
  return s;
}

// Weights of a thread's vectors: where rows begin inside a vector (and so do the
// weights, as far into one for all of a thread's rows) kept as float32 in shared
// memory, 16 bytes of each thread side by side; else read from the caches.
template <typename T, int VEC, int NV, bool EDGE>
struct Weights {
  static_assert(!EDGE || VEC % 4 == 0, "whole 16 bytes");
  using Part = Pack<float, 4>;
  Part *mine;
  float now[VEC];
  __device__ __forceinline__ Weights(const NormArgs &p, float *shared, int log2, int j, int shift) {
    if constexpr (EDGE) {
      mine = reinterpret_cast<Part *>(shared) + threadIdx.x;
#pragma unroll(NV <= 4 ? NV : 1)
      for (int k = 0; k < NV; ++k) {
        load_weight<T, VEC, EDGE>(p, span_of<VEC, EDGE>((k << log2) + j, shift, (int)p.D), now);
#pragma unroll
        for (int q = 0; q < VEC; q += 4) mine[(k * VEC + q) / 4 * blockDim.x] = {{now[q], now[q + 1], now[q + 2], now[q + 3]}};
      }
    }
  }
  __device__ __forceinline__ const float (&of(const NormArgs &p, int k, const Span &at))[VEC] {
    if constexpr (EDGE) {
#pragma unroll
      for (int q = 0; q < VEC; q += 4) {
        const Part part = mine[(k * VEC + q) / 4 * blockDim.x];
#pragma unroll
        for (int i = 0; i < 4; ++i) now[q + i] = part.v[i];
      }
    } else {
      load_weight<T, VEC, EDGE>(p, at, now);
    }
    return now;
  }
};

// Bytes of shared memory that Weights takes.
constexpr size_t weights_bytes(int block, int elements, bool edge) {
  return edge ? (size_t)block * elements * sizeof(float) : 0;
}

// Blocks of 512 threads that k_norm's registers should leave room for, and whether
// there are enough of them to hold what a thread loads of x and the residual
// (`words` registers) at once.  Early against as they are used, bf16: 32768x4096
// (16 words) 160 and 167 us, 4096x16384 (32 words, 2 blocks) 85 and 106, 65536x999
// 105 and 125, in 8 bits 110 and 124; but 65537x1536 (24 words, 3 blocks) 132 and
// 124, in 8 bits 149 and 134; f32 4096x8192 (32 words, 3 blocks) 112 and 87.
template <typename T, typename S>
__host__ __device__ constexpr int words_of(int elements) { return elements * (int)(sizeof(T) + sizeof(S)) / 4; }
template <typename T, typename S>
__host__ __device__ constexpr int blocks_of_norm(int vec, int nv, bool quant, bool edge) {
  if (quant) return 2;
  if (!edge) return nv * vec > 24 ? 2 : 3;
  const int words = words_of<T, S>(nv * vec);
  return words > 48 ? 1 : vec == 4 && words <= 16 ? 3 : 2;
}
template <typename T, typename S>
__host__ __device__ constexpr bool loads_early(int vec, int nv, bool quant, bool edge) {
  const int words = words_of<T, S>(nv * vec);
  if (vec == 1) return false;
  if (quant) return nv * vec <= 16 && words <= (edge ? 16 : 24);
  const int blocks = blocks_of_norm<T, S>(vec, nv, quant, edge);
  return blocks == 1 || words <= (blocks == 3 ? 16 : 32);
}

// T: x and y; S: the stream.  With EDGE blocks stride over rows so that a
// thread's rows have one shift.  65537x1536 bf16: 125 us (6.5 TB/s), in 8 bits
// 136 (5.2 TB/s: it needs half as many registers again for the products with the
// weights); 65536x999, where rows begin inside a vector: 105 us (5.0 TB/s; one
// element at a time: 317).
template <typename T, typename S, int VEC, int NV, bool QUANT, bool EDGE>
__global__ void __launch_bounds__(kMost, blocks_of_norm<T, S>(VEC, NV, QUANT, EDGE)) k_norm(const __grid_constant__ NormArgs p) {
  extern __shared__ float4 memory[];  // Weights
  __shared__ float shared[2][2 * kMost / 32];
  // All of a row's loads before its first value is used, where registers allow it.
  constexpr bool kEarly = loads_early<T, S>(VEC, NV, QUANT, EDGE);
  const int log2 = p.threads_log2, j = threadIdx.x & ((1 << log2) - 1), groups = blockDim.x >> log2;
  const int D = (int)p.D;
  int64_t row = (int64_t)blockIdx.x * groups + (threadIdx.x >> log2);
  const int shift = EDGE ? (int)(row * p.D % VEC) : 0;
  Weights<T, VEC, NV, EDGE> weights(p, reinterpret_cast<float *>(memory), log2, j, shift);
  int half = 0;
  // (as many rounds for each of the block's rows: the sums wait for one another)
  for (int64_t first = (int64_t)blockIdx.x * groups; first < p.rows; first += (int64_t)gridDim.x * groups) {
    const bool on = row < p.rows, last = row == p.rows - 1;
    const T *x = static_cast<const T *>(p.x) + row * p.xs;
    const S *res = static_cast<const S *>(p.res) + row * p.rs;
    constexpr int kHold = QUANT && !kEarly ? 1 : NV;
    Row<S, VEC> v[kHold];          // the stream as it is kept
    Row<T, VEC> in[kEarly ? NV : 1];
    float t[QUANT ? NV : 1][VEC];  // or times the weights
    float sum = 0.0f, top = 0.0f;
    auto load = [&](int k, const Span &at) {
      load_span<T, VEC, EDGE>(in[kEarly ? k : 0], x, at, last);
      if (p.res != nullptr) load_span<S, VEC, EDGE>(v[k % kHold], res, at, last);
    };
    if (kEarly) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
        if (on && at.any()) load(k, at);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
      if (on && at.any()) {
        Row<S, VEC> &s = v[k % kHold];
        Row<T, VEC> &x_k = in[kEarly ? k : 0];
        if (!kEarly) load(k, at);
        mask_span<T, VEC, EDGE>(x_k, at);
        if (p.res != nullptr) {
          mask_span<S, VEC, EDGE>(s, at);
          add_to(s, x_k);
          store_span<S, VEC, EDGE>(static_cast<S *>(p.s) + row * p.D, at, s);
        } else if constexpr (sizeof(T) == sizeof(S)) {
#pragma unroll
          for (int i = 0; i < Row<S, VEC>::kWords; ++i) s.w[i] = x_k.w[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum = fmaf(s[i], s[i], sum);
        if (QUANT) {
          const float (&w)[VEC] = weights.of(p, k, at);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            t[k][i] = s[i] * w[i];
            top = fmaxf(top, fabsf(t[k][i]));
          }
        }
      }
    }
    over_row<QUANT>(sum, top, log2, shared[half]);
    half ^= 1;
    const float r = rsqrtf(fmaf(sum, p.inverse, p.eps));
    if (on && p.r != nullptr && j == 0) p.r[row] = r;
    if (!QUANT) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
        if (on && at.any()) {
          const float (&w)[VEC] = weights.of(p, k, at);
          float y[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[i] = v[k][i] * r * w[i];
          store_span<T, VEC, EDGE>(static_cast<T *>(p.y) + row * p.D, at, y);
        }
      }
    } else {
      // y = t r: its codes are those of t over the largest |t|, so r (and its
      // rounding) does not enter them.  The scale is never 0: a row of zeros
      // has codes 0, and a reader may divide by it.  A NaN in the row is in r.
      // (unit is the quotient top / 448 by Markstein's correction of the product with
      // 1 / 448, whose rounding all of a row's codes would share: of 3 10^8 elements
      // 144 instead of 184 have another code than float64 gives them, of the formula in
      // elementary float32 operations 201.  Two divisions, there and by 448 / top in
      // place of 1 / unit: 127, but rows of 15 columns take 2% longer.)
      constexpr float kPart = 1.0f / kE4m3Max;
      float unit = top * kPart;
      if (top <= 3.0e38f) unit = fmaf(fmaf(-kE4m3Max, unit, top), kPart, unit);
      const float scale = unit * r < kTiny ? kTiny : unit * r;
      const bool usual = unit >= kTiny && scale > kTiny;  // (and so 1 / unit in float32's range)
      const float factor = usual ? 1.0f / unit : r;
      if (on && j == 0) p.scale[row] = scale;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
        if (on && at.any()) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) t[k][i] *= factor;
          if (!usual) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) t[k][i] /= scale;
          }
          uint8_t *q = p.q + row * p.D + at.c;
          if (VEC > 1 && (!EDGE || (at.lo == 0 && at.hi == VEC))) {
            using Codes = Pack<uint16_t, (VEC + 1) / 2>;
            Codes c;
#pragma unroll
            for (int i = 0; i + 1 < VEC; i += 2)
              c.v[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(t[k][i], t[k][i + 1]), __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<Codes *>(q) = c;
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              if (i >= at.lo && i < at.hi) q[i] = __nv_cvt_float_to_fp8(t[k][i], __NV_SATFINITE, __NV_E4M3);
          }
        }
      }
    }
    row += (int64_t)gridDim.x * groups;
  }
}

// x here is the stream s as kept (x itself without a residual), of type S.
// With t = dy r: dw = sum t s, ds = gs + t w - s (r^2 mean(t w s)).  65537x1536
// bf16: 165 us (4.9 TB/s), 32768x2048 float32: 165 us (6.5 TB/s), 65536x999 bf16,
// where rows begin inside a vector: 121 us (4.3 TB/s).
template <typename T, typename S, int VEC, int NV, bool EDGE, int BLOCK>
__global__ void __launch_bounds__(BLOCK, resident_of(NV * VEC) / BLOCK)
    k_norm_backward(const __grid_constant__ NormArgs p) {
  // Of wide rows a thread holds too much to fetch gs early, and of them and of a
  // float32 stream beside 16 bits also to keep the products dy r w (4096x9001 f32:
  // 344 us, again from the weights 224; 32768x4096 bf16 and f32 360 and 335; but
  // bf16 alone 195 and 211).
  constexpr bool kLean = NV * VEC > 16, kAgain = kLean || sizeof(T) != sizeof(S);
  extern __shared__ float4 memory[];  // Weights, then [groups, D] where a block has several groups
  float *sums = reinterpret_cast<float *>(memory);
  __shared__ float shared[2][kMost / 32];
  const int log2 = p.threads_log2, j = threadIdx.x & ((1 << log2) - 1), groups = BLOCK >> log2;
  const int group = threadIdx.x >> log2, D = (int)p.D;
  int64_t row = (int64_t)blockIdx.x * groups + group;
  const int shift = EDGE ? (int)(row * p.D % VEC) : 0;
  Weights<T, VEC, NV, EDGE> weights(p, sums, log2, j, shift);
  float dw[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = 0.0f;
  int half = 0;
  for (int64_t first = (int64_t)blockIdx.x * groups; first < p.rows; first += (int64_t)gridDim.x * groups) {
    const bool on = row < p.rows, last = row == p.rows - 1;
    const S *x = static_cast<const S *>(p.x) + row * p.xs, *gs = static_cast<const S *>(p.gs) + row * p.D;
    const T *dy = static_cast<const T *>(p.dy) + row * p.D;
    Row<S, VEC> v[NV], a[kLean ? 1 : NV];
    Row<T, VEC> g[NV];
    const float r = on ? p.r[row] : 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
      if (on && at.any()) {
        load_span<S, VEC, EDGE>(v[k], x, at, last);
        load_span<T, VEC, EDGE>(g[k], dy, at, last);
        if (!kLean && p.gs != nullptr) load_span<S, VEC, EDGE>(a[k], gs, at, last);
      }
    }
    float tw[kAgain ? 1 : NV][VEC];
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
      if (on && at.any()) {
        mask_span<S, VEC, EDGE>(v[k], at);
        mask_span<T, VEC, EDGE>(g[k], at);
        const float (&w)[VEC] = weights.of(p, k, at);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float t = g[k][i] * r, s = v[k][i];
          dw[k][i] = fmaf(t, s, dw[k][i]);
          tw[kAgain ? 0 : k][i] = t * w[i];
          sum = fmaf(tw[kAgain ? 0 : k][i], s, sum);
        }
      }
    }
    over_row<false>(sum, none, log2, shared[half]);
    half ^= 1;
    const float m = -sum * p.inverse * (r * r);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
      if (on && at.any()) {
        if (kLean && p.gs != nullptr) load_span<S, VEC, EDGE>(a[0], gs, at, last);
        float (&d)[VEC] = tw[kAgain ? 0 : k];
        if constexpr (kAgain) {
          const float (&w)[VEC] = weights.of(p, k, at);
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[i] = g[k][i] * r * w[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] = fmaf(v[k][i], m, d[i]);
        if (p.gs != nullptr) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[i] += a[kLean ? 0 : k][i];
        }
        store_span<T, VEC, EDGE>(static_cast<T *>(p.dx) + row * p.D, at, d);
        if (p.dres != nullptr) store_span<S, VEC, EDGE>(static_cast<S *>(p.dres) + row * p.D, at, d);
      }
    }
    row += (int64_t)gridDim.x * groups;
  }
  if (p.partial == nullptr) return;
  if (EDGE && groups > 1) __syncthreads();  // (the last row's weights have been read)
  // The block's groups hold the same columns: added one after another.
  float *to = groups > 1 ? sums + group * D : p.partial + (int64_t)blockIdx.x * D;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const Span at = span_of<VEC, EDGE>((k << log2) + j, shift, D);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= at.lo && i < at.hi) to[at.c + i] = dw[k][i];
  }
  if (groups == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += BLOCK) {
    float s = 0.0f;
    for (int k = 0; k < groups; ++k) s += sums[k * D + c];
    p.partial[(int64_t)blockIdx.x * D + c] = s;
  }
}

// dw = the sum over the partial rows, 32 columns a block: 444 rows of 4096
// columns (7 MB) take 7 us beside the gradient's 188.
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
// at most `held` vectors; one more vector where rows begin inside one.  Of 1, 2, 3
// and 4 vectors the forward of 32768x4096 bf16 takes 195, 167, 167 and 185 us,
// of 65537x1536 158, 140, 124 and 124; the gradient with 1, 2 and 4 346, 192 and
// 353 us, 220, 165 and 286.
struct Shape {
  int threads_log2, block, groups;
  int per;            // vectors a thread holds
};

constexpr int kHeld = 3, kHeldBackward = 2;

Shape shape_of(int64_t D, int vec, bool edge, int held) {
  const int64_t vectors = (D + vec - 1 + (edge ? vec - 1 : 0)) / vec;
  Shape s;
  s.threads_log2 = 0;
  while (1 << s.threads_log2 < kMost && (int64_t)held << s.threads_log2 < vectors) ++s.threads_log2;
  const int threads = 1 << s.threads_log2;
  s.per = (int)((vectors + threads - 1) / threads);
  s.block = threads < kBlock ? kBlock : threads;
  s.groups = s.block / threads;
  return s;
}

// Blocks for all rows; of the gradient as many as run at once (each keeps a sum
// of the weight's gradient); with EDGE a few times as many, so that each keeps
// its weights for some rows, and so many that a thread's next row begins where
// its last one did.
int64_t blocks_of(int64_t rows, const Shape &s, int vec, bool edge, bool resident) {
  int64_t n = (rows + s.groups - 1) / s.groups;
  const int64_t cap = (int64_t)device_info().sm_count * ((resident ? resident_of(s.per * vec) : 4096) / s.block);
  if ((resident || edge) && n > cap) n = cap;
  if (edge && n * s.groups < rows) {
    const int64_t step = s.groups >= vec ? 1 : vec / s.groups;  // (divides no more than 16: n is not 0)
    n = n / step * step;
  }
  return n;
}

// Lets a kernel have that much dynamic shared memory (4 KB beside it are its own).
cudaError_t more_shared(const void *kernel, size_t bytes) {
  if (bytes <= 44 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename T, typename S, int VEC, int NV, bool EDGE>
cudaError_t norm_launch(const NormArgs &a, const Shape &s, bool quant, cudaStream_t stream) {
  const unsigned grid = (unsigned)blocks_of(a.rows, s, VEC, EDGE, false);
  const size_t smem = weights_bytes(s.block, NV * VEC, EDGE);
  const auto kernel = quant ? k_norm<T, S, VEC, NV, true, EDGE> : k_norm<T, S, VEC, NV, false, EDGE>;
  const cudaError_t e = more_shared(reinterpret_cast<const void *>(kernel), smem);
  if (e != cudaSuccess) return e;
  kernel<<<grid, s.block, smem, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename S, int VEC, int NV, bool EDGE>
cudaError_t norm_backward_launch(const NormArgs &a, const Shape &s, cudaStream_t stream) {
  const unsigned grid = (unsigned)blocks_of(a.rows, s, VEC, EDGE, true);
  const size_t sums = s.groups > 1 ? (size_t)s.groups * a.D * sizeof(float) : 0;
  const size_t weights = weights_bytes(s.block, NV * VEC, EDGE), smem = sums > weights ? sums : weights;
  const auto kernel = s.block == kBlock ? k_norm_backward<T, S, VEC, NV, EDGE, kBlock>
                                        : k_norm_backward<T, S, VEC, NV, EDGE, kMost>;
  const cudaError_t e = more_shared(reinterpret_cast<const void *>(kernel), smem);
  if (e != cudaSuccess) return e;
  kernel<<<grid, s.block, smem, stream>>>(a);
  return cudaGetLastError();
}

// The kernel for s.per vectors a thread; kMaxWidth / kMost elements at most
// (and a vector more with EDGE).
template <typename T, typename S, int VEC, bool EDGE>
cudaError_t norm_vec(NormArgs a, bool quant, cudaStream_t stream) {
  const Shape s = shape_of(a.D, VEC, EDGE, kHeld);
  constexpr int kAll = (int)(kMaxWidth / kMost) / VEC + (EDGE ? 1 : 0);
  a.threads_log2 = s.threads_log2;
  if (s.per <= 1) return norm_launch<T, S, VEC, 1, EDGE>(a, s, quant, stream);
  if (s.per <= 2) return norm_launch<T, S, VEC, 2, EDGE>(a, s, quant, stream);
  if (s.per <= 3) return norm_launch<T, S, VEC, 3, EDGE>(a, s, quant, stream);
  if (s.per <= 4) return norm_launch<T, S, VEC, 4, EDGE>(a, s, quant, stream);
  return norm_launch<T, S, VEC, kAll, EDGE>(a, s, quant, stream);
}

template <typename T, typename S, int VEC, bool EDGE>
cudaError_t norm_backward_vec(NormArgs a, cudaStream_t stream) {
  const Shape s = shape_of(a.D, VEC, EDGE, kHeldBackward);
  constexpr int kAll = (int)(kMaxWidth / kMost) / VEC + (EDGE ? 1 : 0);
  a.threads_log2 = s.threads_log2;
  if (s.per <= 1) return norm_backward_launch<T, S, VEC, 1, EDGE>(a, s, stream);
  if (s.per <= 2) return norm_backward_launch<T, S, VEC, 2, EDGE>(a, s, stream);
  if (s.per <= 4) return norm_backward_launch<T, S, VEC, 4, EDGE>(a, s, stream);
  return norm_backward_launch<T, S, VEC, kAll, EDGE>(a, s, stream);
}

// Elements a 16-byte access of T moves.
template <typename T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }

// How rows lie: all of them on vectors, all tensors' rows equally far from one,
// or otherwise (one element at a time).
enum Lie { kOnVectors, kShifted, kAnyhow };

template <typename T, typename S>
cudaError_t norm_as(const NormArgs &a, Lie lie, bool quant, cudaStream_t stream) {
  if (lie == kOnVectors) return norm_vec<T, S, vec_of<T>(), false>(a, quant, stream);
  if (lie == kShifted) return norm_vec<T, S, vec_of<T>(), true>(a, quant, stream);
  return norm_vec<T, S, 1, false>(a, quant, stream);
}

template <typename T, typename S>
cudaError_t norm_backward_as(const NormArgs &a, Lie lie, cudaStream_t stream) {
  if (lie == kOnVectors) return norm_backward_vec<T, S, vec_of<T>(), false>(a, stream);
  if (lie == kShifted) return norm_backward_vec<T, S, vec_of<T>(), true>(a, stream);
  return norm_backward_vec<T, S, 1, false>(a, stream);
}

Lie lie_of(const NormArgs &a, int e, int f, int x_size) {
  const int vec = 16 / e;
  // starts on vectors of `vec` elements, whatever a tensor's type
  auto on = [&](const void *p, int size) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)(vec * size) == 0; };
  const bool starts = on(a.x, x_size) && on(a.res, f) && on(a.y, e) && on(a.s, f) && on(a.q, 1) && on(a.dy, e) &&
                      on(a.gs, f) && on(a.dx, e) && on(a.dres, f);
  if (!starts) return kAnyhow;
  const bool strides = (a.xs - a.D) % vec == 0 && (a.res == nullptr || (a.rs - a.D) % vec == 0);
  if (!strides) return kAnyhow;
  if (a.D % vec == 0) return aligned_to(a.w, 0, 4, 16) ? kOnVectors : kAnyhow;
  // Rows that overlap (windows of one signal): the vector at a row's end could reach
  // past the last row's.
  if (a.xs < a.D || (a.res != nullptr && a.rs < a.D)) return kAnyhow;
  // One at a time what is narrower than 32 columns, where a vector's masks cost
  // more (15 columns bf16: 241 against 488 us, 31: 234 and 302, the gradient 304
  // and 322; 31 columns f32: 126 and 142, 166 and 226; but 95 columns bf16: 210
  // and 148, 433 and 237, for 64 and 32 million elements).
  return a.D < 32 ? kAnyhow : kShifted;
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
  const Lie lie = lie_of(a, dtype_size(dtype), dtype_size(stream_dtype), dtype_size(dtype));
  a.w_f32 = w_dtype == CPAB_F32;
  using H = __half;
  using B = __nv_bfloat16;
  return launch_status(by_type(dtype, stream_dtype, [&] { return norm_as<float, float>(a, lie, quant, stream); },
                               [&] { return norm_as<H, H>(a, lie, quant, stream); },
                               [&] { return norm_as<B, B>(a, lie, quant, stream); },
                               [&] { return norm_as<H, float>(a, lie, quant, stream); },
                               [&] { return norm_as<B, float>(a, lie, quant, stream); }),
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
  if (residual == nullptr && stream_dtype != dtype)
    return report_error(CPAB_ERR_ARG, "rms_norm: without a residual the stream is x, of x's type");
  NormArgs a{};
  a.x = x, a.xs = x_row, a.res = residual, a.rs = residual_row, a.w = weight, a.rows = rows, a.D = D, a.inverse = 1.0f / (float)D;
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
  if (residual == nullptr && stream_dtype != dtype)
    return report_error(CPAB_ERR_ARG, "rms_norm_quantized: without a residual the stream is x, of x's type");
  NormArgs a{};
  a.x = x, a.xs = x_row, a.res = residual, a.rs = residual_row, a.w = weight, a.rows = rows, a.D = D, a.inverse = 1.0f / (float)D;
  a.eps = eps, a.q = q, a.scale = scale, a.s = sum;
  return forward("rms_norm_quantized", dtype, stream_dtype, weight_dtype, a, true, stream);
}

extern "C" int64_t cpab_b200_rms_norm_workspace(int dtype, int64_t rows, int64_t D) {
  if (!dtype_ok(dtype) || rows < 1 || D < 1 || D > kMaxWidth) return 0;
  const int vec = 16 / dtype_size(dtype);
  int64_t most = 0;
  for (const int64_t n : {blocks_of(rows, shape_of(D, 1, false, kHeldBackward), 1, false, true),
                          blocks_of(rows, shape_of(D, vec, false, kHeldBackward), vec, false, true),
                          blocks_of(rows, shape_of(D, vec, true, kHeldBackward), vec, true, true)})
    most = n > most ? n : most;
  return most * D;
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
  a.r = const_cast<float *>(rstd), a.rows = rows, a.D = D, a.inverse = 1.0f / (float)D, a.dy = grad_y, a.gs = grad_sum;
  a.dx = grad_x, a.dres = grad_residual, a.partial = grad_weight != nullptr ? workspace : nullptr;
  const int e = dtype_size(dtype), f = dtype_size(stream_dtype);
  const Lie lie = lie_of(a, e, f, f);
  using H = __half;
  using B = __nv_bfloat16;
  const cudaError_t err = by_type(dtype, stream_dtype, [&] { return norm_backward_as<float, float>(a, lie, stream); },
                            [&] { return norm_backward_as<H, H>(a, lie, stream); },
                            [&] { return norm_backward_as<B, B>(a, lie, stream); },
                            [&] { return norm_backward_as<H, float>(a, lie, stream); },
                            [&] { return norm_backward_as<B, float>(a, lie, stream); });
  if (err != cudaSuccess || grad_weight == nullptr) return launch_status(err, "rms_norm_backward");
  const int vec = lie == kAnyhow ? 1 : 16 / e;
  const int64_t n = blocks_of(rows, shape_of(D, vec, lie == kShifted, kHeldBackward), vec, lie == kShifted, true);
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
