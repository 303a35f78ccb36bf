// One AdamW step over many tensors in few launches: 256 tensors of one type and one
// kind of states each.
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
// copied to the device first and a captured graph keeps them.  Blocks take runs
// of chunks of 2048 elements; a chunk belongs to one tensor.
//
// With float32 states memory bounds it: 200 million float32 parameters (28 bytes
// each) take 854 us (6.6 TB/s; a copy: 6.46).  With 8-bit states 16 bytes and
// about 75 instructions, mostly the integer units' (hash, cut, the near test), are
// left of a parameter: 622 us (5.2 TB/s), 0.73 of the time for 0.57 of the
// bytes; of bfloat16 parameters 10 bytes, 588 us (3.4 TB/s, 70% of the issue slots).  A kernel for all types, branching per tensor, spilled and took 1100 us.
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
// The scale of roots where a second moment overflowed: 2^64 / 448, whose largest
// code stands for 2^64, the square of which is infinite again.
constexpr float kOverflowed = 0x1p64f / kE4m3Max;
// Blocks of an SM that the registers leave room for (8-bit states: 2, 3 and 4
// take 701, 622 and 719 us for 200 million); blocks of a launch per SM at most, if
// each has kChunksEach chunks (a block's begin is 200 instructions: one chunk a
// block takes 925 us with 8-bit states, 839 against 857 with float32 ones, and
// 700 against 689 of bfloat16 parameters).
constexpr int kResident32 = 4, kResident8 = 3, kPerSm32 = 32, kPerSm8 = 6, kChunksEach = 8;
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

// z in [0, 448] to the e4m3 value below or above it, with 16 random bits u:
// adding u below the last kept mantissa bit and cutting there rounds up with
// the probability of z's distance from the value below.  Below 2^-6 values are
// spaced as in the binade above, so 2^-6 is added first.  (Above 448 the
// conversion to 8 bits saturates.)  `sum` is what is cut.
__device__ __forceinline__ float stochastic(float z, uint32_t u, uint32_t &sum) {
  const float low = z < 0.015625f ? 0.015625f : 0.0f;
  sum = __float_as_uint(z + low) + u * 16u;
  return __uint_as_float(sum & ~0xFFFFFu) - low;
}

// The least over sums of how far they lie above 8 places before a cut: below
// kNear, another z a few last places off could have been cut elsewhere.
constexpr uint32_t kNear = 16u << 12;
__device__ __forceinline__ uint32_t from_cut(uint32_t least, uint32_t sum) { return min(least, sum * 4096u + (8u << 12)); }

__device__ __forceinline__ uint32_t to_e4m3(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 from_e4m3(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(__half2(h));
}

// The largest of a warp's non-negative values; NaN if there is one (as
// integers such floats are ordered, NaN last).
__device__ __forceinline__ float warp_max(uint32_t bits) { return __uint_as_float(__reduce_max_sync(~0u, bits)); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Rates {
  float decay, rate, root, eps, b1, ob1, b2, ob2;  // root: 1 / sqrt(1 - b2^t)
};

// The moments' separate roundings (no fused multiply-adds) are those of the
// formulas written as elementary operations, which the tests compare with bit
// for bit.  The parameter's update goes through the hardware's approximate
// reciprocal roots: 6.7e-8 of an update that is 1e-3 of the parameter off (rms; 3.1e-7
// at most), against 5.2e-8 (2.1e-7) of correctly rounded ones, which take 200 million
// parameters 703 against 622 us with 8-bit states (float32: 863 and 854).  A second moment
// below 2^-126, which they would flush to 0, counts as 2^-126 there.  One that
// overflowed has an infinite root (not inf * 0): its parameter only decays.  (8-bit
// states keep it so by kOverflowed; its block's small elements, whose roots are then
// far below the block's least code, all but stand still meanwhile.)
__device__ __forceinline__ float update(const Rates &r, float p, float g, float &m, float &v, float &root) {
  m = __fadd_rn(__fmul_rn(m, r.b1), __fmul_rn(g, r.ob1));
  v = __fadd_rn(__fmul_rn(v, r.b2), __fmul_rn(__fmul_rn(g, g), r.ob2));
  const float least = fmaxf(v, kTiny);
  float inverse;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(least));
  inverse = fmaxf(inverse, 0x1p-65f);  // (2^-64 is that of the largest number)
  const float den = fmaf(least * inverse, r.root, r.eps);
  root = v * inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(den));
  return fmaf(r.rate * m, -inverse, p * r.decay);
}

// Four consecutive elements of a tensor of n from `at` on; those past its end
// are 0 and not stored.
template <typename T, bool WHOLE>
__device__ __forceinline__ void load4(const void *base, int64_t at, int64_t n, float (&out)[4]) {
  const T *q = static_cast<const T *>(base) + at;
  if constexpr (WHOLE) {
    if constexpr (sizeof(T) == 4) {
      const float4 v = __ldcs(reinterpret_cast<const float4 *>(q));
      out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
    } else {
      const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(q));
      const float2 a = unpack_pair<T>(v.x), b = unpack_pair<T>(v.y);
      out[0] = a.x, out[1] = a.y, out[2] = b.x, out[3] = b.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = at + i < n ? to_f32(q[i]) : 0.0f;
  }
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void store4(void *base, int64_t at, int64_t n, const float (&in)[4]) {
  T *q = static_cast<T *>(base) + at;
  if constexpr (WHOLE) {
    if constexpr (sizeof(T) == 4) {
      __stcs(reinterpret_cast<float4 *>(q), make_float4(in[0], in[1], in[2], in[3]));
    } else {
      __stcs(reinterpret_cast<uint2 *>(q), make_uint2(pack_pair<T>(in[0], in[1]), pack_pair<T>(in[2], in[3])));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n) q[i] = from_f32<T>(in[i]);
  }
}

template <bool WHOLE>
__device__ __forceinline__ uint32_t load_codes(const void *base, int64_t at, int64_t n) {
  const uint8_t *q = static_cast<const uint8_t *>(base) + at;
  if constexpr (WHOLE) {
    return __ldcs(reinterpret_cast<const uint32_t *>(q));
  } else {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n) c |= (uint32_t)q[i] << (8 * i);
    return c;
  }
}

template <bool WHOLE>
__device__ __forceinline__ void store_codes(void *base, int64_t at, int64_t n, uint32_t c) {
  uint8_t *q = static_cast<uint8_t *>(base) + at;
  if constexpr (WHOLE) {
    __stcs(reinterpret_cast<uint32_t *>(q), c);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < n) q[i] = (uint8_t)(c >> (8 * i));
  }
}

// What a block keeps of the tensor it is in.
struct Here {
  void *p, *m, *v;
  const void *g;
  float *scales;
  int64_t n;
  uint32_t first, next;    // its first chunk, and that of the tensor after it
  uint32_t key;
  bool vec;
  Rates r;
};

// A warp's 256 elements from element `first` on: lane i holds elements 4 i ..
// 4 i + 3 of each half.
template <typename T, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void step_block(const Here &t, int64_t first) {
  const int lane = threadIdx.x & 31;
  const int64_t at0 = first + lane * 4, n = t.n;
  float p[2][4], g[2][4], m[2][4], v[2][4], root[2][4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    load4<T, WHOLE>(t.g, at0 + k * 128, n, g[k]);
    load4<T, WHOLE>(t.p, at0 + k * 128, n, p[k]);
  }
  if constexpr (EIGHT) {
    const float2 sc = *reinterpret_cast<const float2 *>(t.scales + first / kScaleBlock * 2);
    uint32_t mc[2], vc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mc[k] = load_codes<WHOLE>(t.m, at0 + k * 128, n);
      vc[k] = load_codes<WHOLE>(t.v, at0 + k * 128, n);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float2 a = from_e4m3(mc[k] >> (8 * i) & 0xFFFFu), b = from_e4m3(vc[k] >> (8 * i) & 0xFFFFu);
        m[k][i] = __fmul_rn(a.x, sc.x), m[k][i + 1] = __fmul_rn(a.y, sc.x);
        const float x = __fmul_rn(b.x, sc.y), y = __fmul_rn(b.y, sc.y);
        v[k][i] = __fmul_rn(x, x), v[k][i + 1] = __fmul_rn(y, y);
      }
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      load4<float, WHOLE>(t.m, at0 + k * 128, n, m[k]);
      load4<float, WHOLE>(t.v, at0 + k * 128, n, v[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[k][i] = update(t.r, p[k][i], g[k][i], m[k][i], v[k][i], root[k][i]);
    store4<T, WHOLE>(t.p, at0 + k * 128, n, p[k]);
    if (!EIGHT) {
      store4<float, WHOLE>(t.m, at0 + k * 128, n, m[k]);
      store4<float, WHOLE>(t.v, at0 + k * 128, n, v[k]);
    }
  }
  if constexpr (EIGHT) {
    float mt = 0.0f;
    uint32_t vt = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mt = fmaxf(mt, fabsf(m[k][i]));
        vt = max(vt, __float_as_uint(v[k][i]));  // (a NaN, which m has where v has, is the largest)
      }
    float ms = __fmul_rn(warp_max(__float_as_uint(mt)), 1.0f / kE4m3Max);
    float rs = __fmul_rn(__fsqrt_rn(warp_max(vt)), 1.0f / kE4m3Max);
    if (rs != rs) ms = rs;
    rs = rs > kOverflowed ? kOverflowed : rs;  // (a NaN stays)
    if (ms < kTiny) ms = kTiny;
    if (rs < kTiny) rs = kTiny;
    if (lane == 0) *reinterpret_cast<float2 *>(t.scales + first / kScaleBlock * 2) = make_float2(ms, rs);
    // Where the approximations below would not do: values that are not finite,
    // and moments near 2^-126 (else a smaller one has a code below the least).
    const bool odd = !(ms <= 3.0e38f && rs <= 3.0e38f) || (rs < 1.0e-16f && rs > kTiny);
    const float mi = __fdiv_rn(1.0f, ms), ri = __fdiv_rn(1.0f, rs);
    const uint32_t start = (uint32_t)at0 + (uint32_t)((uint64_t)at0 >> 32) * 0x9E3779B9u + t.key;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float mq[4], rq[4];
      uint32_t least = odd ? 0u : ~0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = hash(start + k * 128 + i);
        uint32_t a, b;
        mq[i] = stochastic(fabsf(m[k][i]) * mi, u & 0xFFFFu, a);
        rq[i] = stochastic(root[k][i] * ri, u >> 16, b);
        least = from_cut(from_cut(least, a), b);
      }
      // The products stand for the quotients |m| / ms and sqrt(v) / rs, from which
      // they are a few last places off: where that could matter (once in 30,000
      // elements), the quotients themselves.
      if (least < kNear) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = hash(start + k * 128 + i);
          uint32_t a;
          const float mv = i == 0 ? m[k][0] : i == 1 ? m[k][1] : i == 2 ? m[k][2] : m[k][3];
          const float vv = i == 0 ? v[k][0] : i == 1 ? v[k][1] : i == 2 ? v[k][2] : v[k][3];
          float z = __fdiv_rn(fabsf(mv), ms), y = __fdiv_rn(__fsqrt_rn(vv), rs);
          if (z <= kE4m3Max + 1.0f) z = stochastic(z, u & 0xFFFFu, a);
          if (y <= kE4m3Max + 1.0f) y = stochastic(y, u >> 16, a);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q == i) mq[q] = z, rq[q] = y;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mq[i] = copysignf(mq[i], m[k][i]);
        // (2^-9 where v is positive, else 0: 2^200 v is far above it or 0)
        rq[i] = max_nan(rq[i], fminf(v[k][i] * 0x1p100f * 0x1p100f, 0.001953125f));
      }
      store_codes<WHOLE>(t.m, at0 + k * 128, n, to_e4m3(mq[0], mq[1]) | to_e4m3(mq[2], mq[3]) << 16);
      store_codes<WHOLE>(t.v, at0 + k * 128, n, to_e4m3(rq[0], rq[1]) | to_e4m3(rq[2], rq[3]) << 16);
    }
  }
}

template <int N>
__device__ __forceinline__ Here enter(const Params<N> &p, int at) {
  const Tensor &t = p.t[at];
  Here h;
  h.p = t.p, h.g = t.g, h.m = t.m, h.v = t.v, h.scales = t.scales, h.n = t.n, h.vec = t.vec != 0;
  h.first = t.first, h.next = at + 1 < p.count ? p.t[at + 1].first : p.chunks;
  const float step = *t.step + 1.0f;
  const float lr = t.lr_device != nullptr ? *t.lr_device : t.lr;
  h.r.decay = t.lr_device != nullptr ? __fsub_rn(1.0f, __fmul_rn(lr, t.wd)) : t.decay;
  h.r.rate = __fdiv_rn(lr, -expm1f(step * t.log_b1));
  h.r.root = __fdiv_rn(1.0f, __fsqrt_rn(-expm1f(step * t.log_b2)));
  h.r.eps = t.eps, h.r.b1 = t.b1, h.r.ob1 = t.ob1, h.r.b2 = t.b2, h.r.ob2 = t.ob2;
  h.key = hash(p.seed + t.index * 0x9E3779B9u + (uint32_t)(int64_t)step * 0x85EBCA6Bu);
  return h;
}

template <typename T, bool EIGHT, int N>
__global__ void __launch_bounds__(kThreads, EIGHT ? kResident8 : kResident32) k_adamw(const __grid_constant__ Params<N> p) {
  // The block's chunks lie in a row: it rarely comes to another tensor.
  const uint32_t each = p.chunks / gridDim.x, more = p.chunks % gridDim.x;
  uint32_t c = blockIdx.x * each + min(blockIdx.x, more);
  const uint32_t end = c + each + (blockIdx.x < more ? 1 : 0);
  if (c < end) {
    int at = 0;  // the first chunk's tensor: the last one that starts at or before it
    for (int hi = p.count - 1; at < hi;) {
      const int mid = (at + hi + 1) / 2;
      if (p.t[mid].first <= c) at = mid;
      else hi = mid - 1;
    }
    Here h = enter(p, at);
    for (; c < end; ++c) {
      if (c >= h.next) {
        while (at + 1 < p.count && p.t[at + 1].first <= c) ++at;
        h = enter(p, at);
      }
      const int64_t first = (int64_t)(c - h.first) * kChunkElems + (threadIdx.x >> 5) * kScaleBlock;
      if (h.vec && first + kScaleBlock <= h.n) step_block<T, EIGHT, true>(h, first);
      else if (first < h.n) step_block<T, EIGHT, false>(h, first);
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

template <typename T, bool EIGHT, int N>
cudaError_t launch_as(const Params<kMany> &all, cudaStream_t stream) {
  Params<N> p;
  memcpy(p.t, all.t, sizeof(Tensor) * all.count);
  p.count = all.count, p.chunks = all.chunks, p.seed = all.seed, p.ticket = all.ticket;
  const uint32_t sms = (uint32_t)device_info().sm_count;
  const uint32_t least = sms * (EIGHT ? kResident8 : kResident32), most = sms * (EIGHT ? kPerSm8 : kPerSm32);
  uint32_t grid = p.chunks / kChunksEach;
  grid = grid < least ? least : grid > most ? most : grid;
  if (grid > p.chunks) grid = p.chunks > 0 ? p.chunks : 1;
  k_adamw<T, EIGHT, N><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T, bool EIGHT>
cudaError_t launch(const Params<kMany> &p, cudaStream_t stream) {
  return p.count <= kFew ? launch_as<T, EIGHT, kFew>(p, stream) : launch_as<T, EIGHT, kMany>(p, stream);
}

cudaError_t launch_kind(const Params<kMany> &p, int dtype, bool eight, cudaStream_t stream) {
  if (dtype == CPAB_F32) return eight ? launch<float, true>(p, stream) : launch<float, false>(p, stream);
  if (dtype == CPAB_F16) return eight ? launch<__half, true>(p, stream) : launch<__half, false>(p, stream);
  return eight ? launch<__nv_bfloat16, true>(p, stream) : launch<__nv_bfloat16, false>(p, stream);
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
    if (t.state_bits == 8 && t.numel > 0 && (t.scales == nullptr || !aligned_to(t.scales, 0, 4, 8)))
      return report_error(CPAB_ERR_ARG, "adamw: tensor %d: 8-bit states need scales (8-byte aligned)", k);
    if (!(t.beta1 >= 0 && t.beta1 < 1 && t.beta2 >= 0 && t.beta2 < 1))
      return report_error(CPAB_ERR_ARG, "adamw: tensor %d: betas must be in [0, 1)", k);
    if (!(t.eps >= 0)) return report_error(CPAB_ERR_ARG, "adamw: tensor %d: eps must not be negative", k);
  }
  static thread_local Params<kMany> p;
  p.seed = seed;
  p.ticket = workspace;
  // A launch takes tensors of one type with states of one kind.
  for (const int dtype : {CPAB_F32, CPAB_F16, CPAB_BF16}) {
    for (const int bits : {32, 8}) {
      uint64_t chunks = 0;
      p.count = 0;
      for (int k = 0; k <= count; ++k) {
        const bool end = k == count;
        if (!end && (tensors[k].dtype != dtype || tensors[k].state_bits != bits)) continue;
        const uint64_t own = end ? 0 : (uint64_t)(tensors[k].numel + kChunkElems - 1) / kChunkElems;
        if (p.count > 0 && (end || p.count == kMany || chunks + own > 0x7FFFFFFFu)) {
          p.chunks = (uint32_t)chunks;
          const cudaError_t e = launch_kind(p, dtype, bits == 8, stream);
          if (e != cudaSuccess) return launch_status(e, "adamw");
          chunks = 0;
          p.count = 0;
        }
        if (end) break;
        const cpab_adamw_tensor &t = tensors[k];
        Tensor &q = p.t[p.count++];
        q.p = t.param, q.g = t.grad, q.m = t.exp_avg, q.v = t.exp_avg_sq, q.scales = t.scales;
        q.step = t.step, q.lr_device = t.lr_device, q.n = t.numel;
        q.first = (uint32_t)chunks, q.index = (uint32_t)k;
        const int e = dtype_size(t.dtype), s = bits == 8 ? 4 : 16;
        q.vec = aligned_to(t.param, 0, e, 4 * e) && aligned_to(t.grad, 0, e, 4 * e) &&
                aligned_to(t.exp_avg, 0, e, s) && aligned_to(t.exp_avg_sq, 0, e, s);
        q.lr = (float)t.lr, q.wd = (float)t.weight_decay, q.decay = (float)(1.0 - t.lr * t.weight_decay);
        q.eps = (float)t.eps, q.b1 = (float)t.beta1, q.ob1 = (float)(1.0 - t.beta1);
        q.b2 = (float)t.beta2, q.ob2 = (float)(1.0 - t.beta2);
        q.log_b1 = (float)std::log(t.beta1), q.log_b2 = (float)std::log(t.beta2);
        chunks += own;
      }
    }
  }
  return launch_status(cudaSuccess, "");
}
