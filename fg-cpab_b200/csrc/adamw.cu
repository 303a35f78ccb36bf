// One AdamW step over many tensors in one launch.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// in float32 whatever the parameter's type.  States are float32 tensors, or
// 8-bit: e4m3 codes of m and of sqrt(v), each times the float32 scale of its
// block of 256 elements (the block's largest magnitude / 448).  sqrt(v) and
// not v is held because it is what divides: its range is half as many binades.
// The codes are rounded stochastically: the averages move by 0.1% (sqrt(v):
// 0.05%) of their distance per step, far less than half a code's spacing
// (3% to 6%), so rounding to nearest would leave them where they are.  The
// random bits are a hash of (seed, tensor, step, element).  A positive second
// moment never gets code 0 (its parameter's next step would divide by eps).
//
// The tensors' addresses travel in the kernel's parameters, so nothing is
// copied to the device first and a captured graph keeps them.  Blocks stride
// over chunks of 2048 elements; a chunk belongs to one tensor.
#include <cuda_fp8.h>

#include <cmath>
#include <cstring>

#include "sequence.cuh"

namespace cpab {
namespace {

constexpr int kThreads = 256;
constexpr int kChunkElems = 2048;  // 8 elements a thread, 8 scale blocks
constexpr int kScaleBlock = 256;   // elements that share a scale: one warp's
constexpr float kE4m3Max = 448.0f;
constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the smallest scale
static_assert(kChunkElems == kThreads * 8 && kScaleBlock == 32 * 8, "a warp holds a scale block");

struct Tensor {
  void *p;
  const void *g;
  void *m, *v;
  float *scales;           // [blocks, 2] or null (float32 states)
  float *step;
  const float *lr_device;  // or null: lr
  int64_t n;
  uint32_t first;          // its first chunk
  uint32_t index;          // its place in the caller's list (random bits)
  int32_t dtype;
  int32_t vec;             // its arrays allow vector accesses
  float lr, decay, wd, eps, b1, ob1, b2, ob2, log_b1, log_b2;
};

template <int N>
struct Params {
  Tensor t[N];
  int count;
  uint32_t chunks;
  uint32_t seed;
  int32_t *ticket;
};

// The 32-bit permutation PCG-RXS-M-XS (O'Neill, 2014).
__device__ __forceinline__ uint32_t hash(uint32_t x) {
  x = x * 747796405u + 2891336453u;
  x = ((x >> ((x >> 28) + 4)) ^ x) * 277803737u;
  return (x >> 22) ^ x;
}

// z in [0, 448] to e4m3 with 16 random bits u: adding u below the last kept
// mantissa bit and cutting there rounds up with the probability of z's
// distance from the code below.  Below 2^-6 codes are spaced as in the binade
// above, so 2^-6 is added first.
__device__ __forceinline__ float stochastic(float z, uint32_t u) {
  const bool low = z < 0.015625f;
  const float w = low ? z + 0.015625f : z;
  const float k = __uint_as_float((__float_as_uint(w) + (u << 4)) & ~0xFFFFFu);
  const float q = low ? k - 0.015625f : k;
  return !(z <= 448.0f) ? z : fminf(q, kE4m3Max);  // a NaN stays one
}

__device__ __forceinline__ uint32_t to_e4m3(float v) {
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float from_e4m3(uint32_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  return __half2float(__half(h));
}

// The largest of a warp's non-negative values; NaN if there is one (as
// integers such floats are ordered, NaN last).
__device__ __forceinline__ float warp_max(float v) {
  return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v)));
}

struct Rates {
  float decay, rate, root, eps, b1, ob1, b2, ob2;
};

// The separate roundings (no fused multiply-adds) are those of the formulas
// written as elementary operations, which the tests compare with bit for bit.
__device__ __forceinline__ float update(const Rates &r, float p, float g, float &m, float &v, float &root) {
  m = __fadd_rn(__fmul_rn(m, r.b1), __fmul_rn(g, r.ob1));
  v = __fadd_rn(__fmul_rn(v, r.b2), __fmul_rn(__fmul_rn(g, g), r.ob2));
  root = __fsqrt_rn(v);
  const float den = __fadd_rn(__fdiv_rn(root, r.root), r.eps);
  return __fsub_rn(__fmul_rn(p, r.decay), __fdiv_rn(__fmul_rn(r.rate, m), den));
}

template <typename T>
__device__ __forceinline__ void load4(const void *base, int64_t at, int64_t n, bool vec, float (&out)[4]) {
  const T *q = static_cast<const T *>(base);
  if (vec && at + 4 <= n) {
    const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4> *>(q + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = to_f32(p.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = at + i < n ? to_f32(q[at + i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(void *base, int64_t at, int64_t n, bool vec, const float (&in)[4]) {
  T *q = static_cast<T *>(base);
  if (vec && at + 4 <= n) {
    Pack<T, 4> p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<Pack<T, 4> *>(q + at) = p;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n) q[at + i] = from_f32<T>(in[i]);
  }
}

__device__ __forceinline__ void load4_codes(const void *base, int64_t at, int64_t n, bool vec, float (&out)[4]) {
  const uint8_t *q = static_cast<const uint8_t *>(base);
  if (vec && at + 4 <= n) {
    const uint32_t c = *reinterpret_cast<const uint32_t *>(q + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = from_e4m3(c >> (8 * i) & 255u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = at + i < n ? from_e4m3(q[at + i]) : 0.0f;
  }
}

__device__ __forceinline__ void store4_codes(void *base, int64_t at, int64_t n, bool vec, const float (&in)[4]) {
  uint8_t *q = static_cast<uint8_t *>(base);
  if (vec && at + 4 <= n) {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c |= to_e4m3(in[i]) << (8 * i);
    *reinterpret_cast<uint32_t *>(q + at) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n) q[at + i] = (uint8_t)to_e4m3(in[i]);
  }
}

// A warp's 256 elements of tensor t from element `first` on: lane i holds
// elements 4 i .. 4 i + 3 of each half.
template <typename T>
__device__ __forceinline__ void step_block(const Tensor &t, const Rates &r, int64_t first, uint32_t key) {
  const int lane = threadIdx.x & 31;
  const bool vec = t.vec != 0;
  const int64_t at0 = first + lane * 4, n = t.n;
  float p[2][4], g[2][4], m[2][4], v[2][4], root[2][4];
  const bool eight = t.scales != nullptr;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t at = at0 + k * 128;
    load4<T>(t.p, at, n, vec, p[k]);
    load4<T>(t.g, at, n, vec, g[k]);
    if (eight) {
      load4_codes(t.m, at, n, vec, m[k]);
      load4_codes(t.v, at, n, vec, v[k]);
    } else {
      load4<float>(t.m, at, n, vec, m[k]);
      load4<float>(t.v, at, n, vec, v[k]);
    }
  }
  float *sc = t.scales + first / kScaleBlock * 2;
  if (eight) {
    const float ms = sc[0], rs = sc[1];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[k][i] = __fmul_rn(m[k][i], ms);
        const float q = __fmul_rn(v[k][i], rs);
        v[k][i] = __fmul_rn(q, q);
      }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[k][i] = update(r, p[k][i], g[k][i], m[k][i], v[k][i], root[k][i]);
    store4<T>(t.p, at0 + k * 128, n, vec, p[k]);
  }
  if (!eight) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      store4<float>(t.m, at0 + k * 128, n, vec, m[k]);
      store4<float>(t.v, at0 + k * 128, n, vec, v[k]);
    }
    return;
  }
  uint32_t mt = 0, rt = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mt = max(mt, __float_as_uint(fabsf(m[k][i])));
      rt = max(rt, __float_as_uint(root[k][i]));
    }
  float ms = __fmul_rn(warp_max(__uint_as_float(mt)), 1.0f / kE4m3Max);
  float rs = __fmul_rn(warp_max(__uint_as_float(rt)), 1.0f / kE4m3Max);
  if (ms < kTiny) ms = kTiny;
  if (rs < kTiny) rs = kTiny;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t at = at0 + k * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t e = (uint64_t)(at + i);
      const uint32_t u = hash((uint32_t)e + (uint32_t)(e >> 32) * 0x9E3779B9u + key);
      m[k][i] = copysignf(stochastic(__fdiv_rn(fabsf(m[k][i]), ms), u & 0xFFFFu), m[k][i]);
      float q = stochastic(__fdiv_rn(root[k][i], rs), u >> 16);
      if (q == 0.0f && root[k][i] > 0.0f) q = 0.001953125f;
      v[k][i] = q;
    }
    store4_codes(t.m, at, n, vec, m[k]);
    store4_codes(t.v, at, n, vec, v[k]);
  }
  if (lane == 0) {
    sc[0] = ms;
    sc[1] = rs;
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads) k_adamw(const __grid_constant__ Params<N> p) {
  int at = 0;
  {  // the tensor of this block's first chunk: the last one that starts at or before it
    int lo = 0, hi = p.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (p.t[mid].first <= blockIdx.x) lo = mid;
      else hi = mid - 1;
    }
    at = lo;
  }
  int rates_of = -1;
  Rates r{};
  uint32_t key = 0;
  for (uint32_t c = blockIdx.x; c < p.chunks; c += gridDim.x) {
    while (at + 1 < p.count && p.t[at + 1].first <= c) ++at;
    const Tensor &t = p.t[at];
    if (rates_of != at) {
      const float step = *t.step + 1.0f;
      const float lr = t.lr_device != nullptr ? *t.lr_device : t.lr;
      r.decay = t.lr_device != nullptr ? __fsub_rn(1.0f, __fmul_rn(lr, t.wd)) : t.decay;
      r.rate = __fdiv_rn(lr, -expm1f(step * t.log_b1));
      r.root = __fsqrt_rn(-expm1f(step * t.log_b2));
      r.eps = t.eps;
      r.b1 = t.b1, r.ob1 = t.ob1, r.b2 = t.b2, r.ob2 = t.ob2;
      key = hash(p.seed + t.index * 0x9E3779B9u + (uint32_t)(int64_t)step * 0x85EBCA6Bu);
      rates_of = at;
    }
    const int64_t first = (int64_t)(c - t.first) * kChunkElems + (threadIdx.x >> 5) * kScaleBlock;
    if (first < t.n) {
      if (t.dtype == CPAB_F32) step_block<float>(t, r, first, key);
      else if (t.dtype == CPAB_F16) step_block<__half>(t, r, first, key);
      else step_block<__nv_bfloat16>(t, r, first, key);
    }
  }
  // The last block to come here counts the steps: every block has read them.
  __syncthreads();
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(p.ticket, 1) == (int)gridDim.x - 1;
    if (last) *p.ticket = 0;
  }
  __syncthreads();
  if (last)
    for (int k = threadIdx.x; k < p.count; k += kThreads) *p.t[k].step += 1.0f;
}

constexpr int kFew = 32, kMany = 256;  // tensors of a launch: parameters of 4 and 32 KB
static_assert(sizeof(Params<kFew>) <= 4096 && sizeof(Params<kMany>) <= 32764, "kernel parameters");

template <int N>
cudaError_t launch(const Params<kMany> &all, cudaStream_t stream) {
  Params<N> p;
  memcpy(p.t, all.t, sizeof(Tensor) * all.count);
  p.count = all.count, p.chunks = all.chunks, p.seed = all.seed, p.ticket = all.ticket;
  const uint32_t cap = (uint32_t)device_info().sm_count * 4;
  const uint32_t grid = p.chunks < 1 ? 1 : (p.chunks < cap ? p.chunks : cap);
  k_adamw<N><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace
}  // namespace cpab

using namespace cpab;

extern "C" int cpab_b200_adamw(const cpab_adamw_tensor *tensors, int count, uint32_t seed,
                               int32_t *workspace, cpab_stream_t stream) {
  if (count < 0) return report_error(CPAB_ERR_ARG, "adamw: negative tensor count");
  if (count == 0) return launch_status(cudaSuccess, "");
  if (tensors == nullptr || workspace == nullptr) return report_error(CPAB_ERR_ARG, "adamw: null pointer");
  for (int k = 0; k < count; ++k) {
    const cpab_adamw_tensor &t = tensors[k];
    if (!dtype_ok(t.dtype)) return report_error(CPAB_ERR_ARG, "adamw: tensor %d: unknown dtype %d", k, t.dtype);
    if (t.numel < 0) return report_error(CPAB_ERR_ARG, "adamw: tensor %d: negative size", k);
    if (t.numel > (int64_t(1) << 40)) return report_error(CPAB_ERR_SIZE, "adamw: tensor %d: over 2^40 elements", k);
    if (t.step == nullptr || (t.numel > 0 && (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr ||
                                              t.exp_avg_sq == nullptr)))
      return report_error(CPAB_ERR_ARG, "adamw: tensor %d: null pointer", k);
    if (t.state_bits != 32 && t.state_bits != 8)
      return report_error(CPAB_ERR_ARG, "adamw: tensor %d: states have 32 or 8 bits, got %d", k, t.state_bits);
    if (t.state_bits == 8 && t.numel > 0 && t.scales == nullptr)
      return report_error(CPAB_ERR_ARG, "adamw: tensor %d: 8-bit states need scales", k);
    if (!(t.beta1 >= 0 && t.beta1 < 1 && t.beta2 >= 0 && t.beta2 < 1))
      return report_error(CPAB_ERR_ARG, "adamw: tensor %d: betas must be in [0, 1)", k);
    if (!(t.eps >= 0)) return report_error(CPAB_ERR_ARG, "adamw: tensor %d: eps must not be negative", k);
  }
  static thread_local Params<kMany> p;
  p.seed = seed;
  p.ticket = workspace;
  for (int first = 0; first < count;) {
    uint64_t chunks = 0;
    int n = 0;
    for (; n < kMany && first + n < count; ++n) {
      const cpab_adamw_tensor &t = tensors[first + n];
      const uint64_t own = (uint64_t)(t.numel + kChunkElems - 1) / kChunkElems;
      if (chunks + own > 0x7FFFFFFFu) break;
      Tensor &q = p.t[n];
      q.p = t.param, q.g = t.grad, q.m = t.exp_avg, q.v = t.exp_avg_sq;
      q.scales = t.state_bits == 8 ? t.scales : nullptr;
      q.step = t.step, q.lr_device = t.lr_device, q.n = t.numel;
      q.first = (uint32_t)chunks, q.index = (uint32_t)(first + n), q.dtype = t.dtype;
      const int e = dtype_size(t.dtype), s = t.state_bits == 8 ? 4 : 16;
      q.vec = aligned_to(t.param, 0, e, 4 * e) && aligned_to(t.grad, 0, e, 4 * e) &&
              aligned_to(t.exp_avg, 0, e, s) && aligned_to(t.exp_avg_sq, 0, e, s);
      q.lr = (float)t.lr, q.wd = (float)t.weight_decay, q.decay = (float)(1.0 - t.lr * t.weight_decay);
      q.eps = (float)t.eps, q.b1 = (float)t.beta1, q.ob1 = (float)(1.0 - t.beta1);
      q.b2 = (float)t.beta2, q.ob2 = (float)(1.0 - t.beta2);
      q.log_b1 = (float)std::log(t.beta1), q.log_b2 = (float)std::log(t.beta2);
      chunks += own;
    }
    p.count = n;
    p.chunks = (uint32_t)chunks;
    const cudaError_t e = n <= kFew ? launch<kFew>(p, stream) : launch<kMany>(p, stream);
    if (e != cudaSuccess) return launch_status(e, "adamw");
    first += n;
  }
  return launch_status(cudaSuccess, "");
}
