// The gated linear recurrence over time and its gradient.
//
//   a_t = sigmoid(z_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t
//
// per channel, for gate logits z and inputs x [B, T, D] in f32, f16 or bf16
// and a float32 state.  Both a and 1 - a come from one exponential in float32
// (1 - a = sigmoid(-z) keeps its relative precision as a -> 1).
//
// A step (a, b): h -> a h + b; two steps compose to (a2 a1, a2 b1 + b2), which
// is associative.  A block owns a tile of channels of one series and walks it
// stage by stage; within a stage each thread reads a segment of kSteps samples
// of its channels, composes them, and the segments' compositions are scanned
// over the warp (shuffles) and the block (shared memory) to give each segment
// the state it starts from; a second pass over the registers writes the
// segment's states.  Every input is read once and every output written once.
//
// The gradient runs the same way from the last sample back:
//   delta_t = dh_t + c_{t+1},  c_t = a_t delta_t
//   dx_t = (1 - a_t) delta_t,  dz_t = c_t (h_{t-1} - x_t) (1 - a_t)
// with h_{t-1} recomputed in float32 from the states that the forward keeps at
// the start of every kChunk samples (reading the rounded output instead would
// cost more bytes and lose the difference h_{t-1} - x_t where it is small).
#include "sequence.cuh"

namespace cpab {
namespace {

constexpr int kChunk = 64;    // samples between two kept states
constexpr int kWarps = 8;     // warps of a full block
constexpr int kFwdSteps = 16; // samples of a thread's segment (divide kChunk)
constexpr int kBwdSteps = 8;
static_assert(kChunk % kFwdSteps == 0 && kChunk % kBwdSteps == 0, "states start segments");
static_assert((kWarps * kBwdSteps) % kChunk == 0, "a full block's stage starts on a kept state");

struct ScanArgs {
  const void *x, *gate;
  int64_t xb, xt, gb, gt;   // strides of series and samples, in elements
  int64_t T, D;
  const int32_t *lengths;   // [B] or null
  const float *h0;          // [B, D] or null (zeros)
  void *h;                  // [B, T, D]
  float *last;              // [B, D] or null
  float *states;            // [B, ceil(T / kChunk), D]
  const void *grad_h;       // [B, T, D] or null (zeros)
  const float *grad_last;   // [B, D] or null (zeros)
  void *grad_x, *grad_gate;
  int64_t dxb, dxt, dgb, dgt;
  float *grad_h0;           // [B, D] or null
  int lanes;                // lanes of a warp that lie along the channels (a power of two)
  int64_t tiles;            // channel tiles of a series
};

// a = sigmoid(z) and f = 1 - a = sigmoid(-z) from e = exp(-z), by the hardware's
// approximate exponential and reciprocal (2 and 1 units in the last place).
// f = e / (1 + e) keeps its relative precision as a -> 1; where e > 1, 1 - a
// loses none and is right for e = inf too.
__device__ __forceinline__ void gate_of(float z, float &a, float &f) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(1.0f + e));
  f = e > 1.0f ? 1.0f - a : e * a;
}

// Inclusive scan of (A, H) over a warp's segments: lanes `lanes` apart hold
// consecutive segments.
template <int VEC>
__device__ __forceinline__ void warp_compose(float (&A)[VEC], float (&H)[VEC], int lanes, int lane) {
  for (int o = lanes; o < 32; o <<= 1) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float pa = __shfl_up_sync(~0u, A[v], o), ph = __shfl_up_sync(~0u, H[v], o);
      if (lane >= o) {
        H[v] = fmaf(A[v], ph, H[v]);
        A[v] *= pa;
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kWarps * 32) k_scan(ScanArgs p) {
  constexpr int L = kFwdSteps;
  __shared__ float2 total[2][kWarps][32][VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int sub = lane / p.lanes, cl = lane % p.lanes, subs = 32 / p.lanes;
  const int64_t b = blockIdx.x / p.tiles;
  const int64_t d = ((blockIdx.x % p.tiles) * p.lanes + cl) * VEC;
  const bool on = d < p.D;
  int64_t len = p.T;
  if (p.lengths != nullptr) len = min(max((int64_t)p.lengths[b], (int64_t)0), p.T);
  const T *x = static_cast<const T *>(p.x) + b * p.xb + d;
  const T *g = static_cast<const T *>(p.gate) + b * p.gb + d;
  T *h = static_cast<T *>(p.h) + b * p.T * p.D + d;
  const int64_t chunks = (p.T + kChunk - 1) / kChunk;

  float carry[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    carry[v] = on && p.h0 != nullptr ? p.h0[b * p.D + d + v] : 0.0f;

  const int64_t stage = (int64_t)warps * subs * L;
  int buf = 0;
  for (int64_t s0 = 0; s0 < p.T; s0 += stage, buf ^= 1) {
    const int64_t t0 = s0 + (int64_t)(warp * subs + sub) * L;
    float a[L][VEC], in[L][VEC];
    float A[VEC], H[VEC];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool live = on && t0 + i < len;
      Pack<T, VEC> xv{}, gv{};
      if (live) {
        xv = *reinterpret_cast<const Pack<T, VEC> *>(x + (t0 + i) * p.xt);
        gv = *reinterpret_cast<const Pack<T, VEC> *>(g + (t0 + i) * p.gt);
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float f;
        gate_of(to_f32(gv.v[v]), a[i][v], f);
        in[i][v] = live ? f * to_f32(xv.v[v]) : 0.0f;
        if (!live) a[i][v] = 1.0f;
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = 1.0f;
      H[v] = 0.0f;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        H[v] = fmaf(a[i][v], H[v], in[i][v]);
        A[v] *= a[i][v];
      }
    }
    warp_compose(A, H, p.lanes, lane);
    if (sub == subs - 1) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) total[buf][warp][cl][v] = make_float2(A[v], H[v]);
    }
    __syncthreads();
    float state[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float ea = __shfl_up_sync(~0u, A[v], p.lanes), eh = __shfl_up_sync(~0u, H[v], p.lanes);
      float c = carry[v], start = 0.0f;
      for (int w = 0; w < warps; ++w) {
        if (w == warp) start = c;
        const float2 q = total[buf][w][cl][v];
        c = fmaf(q.x, c, q.y);
      }
      carry[v] = c;
      state[v] = sub > 0 ? fmaf(ea, start, eh) : start;
    }
    if (on && p.states != nullptr && t0 < p.T && t0 % kChunk == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        p.states[(b * chunks + t0 / kChunk) * p.D + d + v] = state[v];
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
      Pack<T, VEC> hv;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        state[v] = fmaf(a[i][v], state[v], in[i][v]);
        hv.v[v] = from_f32<T>(t0 + i < len ? state[v] : 0.0f);
      }
      if (on && t0 + i < p.T) *reinterpret_cast<Pack<T, VEC> *>(h + (t0 + i) * p.D) = hv;
    }
  }
  if (on && p.last != nullptr && warp == 0 && sub == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.last[b * p.D + d + v] = carry[v];
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kWarps * 32) k_scan_backward(ScanArgs p) {
  constexpr int L = kBwdSteps;
  __shared__ float4 total[2][kWarps][32][VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int sub = lane / p.lanes, cl = lane % p.lanes, subs = 32 / p.lanes;
  const int64_t b = blockIdx.x / p.tiles;
  const int64_t d = ((blockIdx.x % p.tiles) * p.lanes + cl) * VEC;
  const bool on = d < p.D;
  int64_t len = p.T;
  if (p.lengths != nullptr) len = min(max((int64_t)p.lengths[b], (int64_t)0), p.T);
  const T *x = static_cast<const T *>(p.x) + b * p.xb + d;
  const T *g = static_cast<const T *>(p.gate) + b * p.gb + d;
  const T *dh = static_cast<const T *>(p.grad_h) + b * p.T * p.D + d;
  T *dx = static_cast<T *>(p.grad_x) + b * p.dxb + d;
  T *dg = static_cast<T *>(p.grad_gate) + b * p.dgb + d;
  const int64_t chunks = (p.T + kChunk - 1) / kChunk;

  float carry[VEC];  // c of the first sample after the stage
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    carry[v] = on && p.grad_last != nullptr ? p.grad_last[b * p.D + d + v] : 0.0f;

  const int64_t stage = (int64_t)warps * subs * L;
  int buf = 0;
  for (int64_t s0 = (p.T - 1) / stage * stage; s0 >= 0; s0 -= stage, buf ^= 1) {
    const int64_t t0 = s0 + (int64_t)(warp * subs + sub) * L;
    float a[L][VEC], f[L][VEC], xs[L][VEC], gr[L][VEC];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool live = on && t0 + i < len;
      Pack<T, VEC> xv{}, gv{}, dv{};
      if (live) {
        xv = *reinterpret_cast<const Pack<T, VEC> *>(x + (t0 + i) * p.xt);
        gv = *reinterpret_cast<const Pack<T, VEC> *>(g + (t0 + i) * p.gt);
        if (p.grad_h != nullptr)
          dv = *reinterpret_cast<const Pack<T, VEC> *>(dh + (t0 + i) * p.D);
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        gate_of(to_f32(gv.v[v]), a[i][v], f[i][v]);
        xs[i][v] = to_f32(xv.v[v]);
        gr[i][v] = to_f32(dv.v[v]);
        if (!live) {
          a[i][v] = 1.0f;
          f[i][v] = 0.0f;
        }
      }
    }
    // (A, H): the segment's samples forward; (A, R): c at its first sample is
    // A c_next + R.
    float A[VEC], H[VEC], R[VEC], base[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = 1.0f;
      H[v] = R[v] = 0.0f;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        H[v] = fmaf(a[i][v], H[v], f[i][v] * xs[i][v]);
        A[v] *= a[i][v];
        R[v] = a[L - 1 - i][v] * (R[v] + gr[L - 1 - i][v]);
      }
      base[v] = on ? p.states[(b * chunks + s0 / kChunk) * p.D + d + v] : 0.0f;
    }
    // Scans over the warp's segments: forward ones up, backward ones down.
    float Af[VEC], Ab[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) Af[v] = Ab[v] = A[v];
    for (int o = p.lanes; o < 32; o <<= 1) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float pa = __shfl_up_sync(~0u, Af[v], o), ph = __shfl_up_sync(~0u, H[v], o);
        const float na = __shfl_down_sync(~0u, Ab[v], o), nr = __shfl_down_sync(~0u, R[v], o);
        if (lane >= o) {
          H[v] = fmaf(Af[v], ph, H[v]);
          Af[v] *= pa;
        }
        if (lane + o < 32) {
          R[v] = fmaf(Ab[v], nr, R[v]);
          Ab[v] *= na;
        }
      }
    }
    // The warp's totals: A and H from its last segment, R from its first.
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float r0 = __shfl_sync(~0u, R[v], cl);
      if (sub == subs - 1) total[buf][warp][cl][v] = make_float4(Af[v], H[v], r0, 0.0f);
    }
    __syncthreads();
    float state[VEC], c[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float ea = __shfl_up_sync(~0u, Af[v], p.lanes), eh = __shfl_up_sync(~0u, H[v], p.lanes);
      const float na = __shfl_down_sync(~0u, Ab[v], p.lanes), nr = __shfl_down_sync(~0u, R[v], p.lanes);
      float s = base[v];
      for (int w = 0; w < warp; ++w) {
        const float4 q = total[buf][w][cl][v];
        s = fmaf(q.x, s, q.y);
      }
      float r = carry[v], after = 0.0f;
      for (int w = warps - 1; w >= 0; --w) {
        if (w == warp) after = r;
        const float4 q = total[buf][w][cl][v];
        r = fmaf(q.x, r, q.z);
      }
      carry[v] = r;
      state[v] = sub > 0 ? fmaf(ea, s, eh) : s;
      c[v] = sub < subs - 1 ? fmaf(na, after, nr) : after;
    }
    // Forward once more for h_{t-1} - x_t, then back.
#pragma unroll
    for (int i = 0; i < L; ++i) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float before = state[v];
        state[v] = fmaf(a[i][v], before, f[i][v] * xs[i][v]);
        xs[i][v] = before - xs[i][v];
      }
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      Pack<T, VEC> dxv, dgv;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float delta = gr[i][v] + c[v];
        c[v] = a[i][v] * delta;
        const bool live = t0 + i < len;
        dxv.v[v] = from_f32<T>(live ? f[i][v] * delta : 0.0f);
        dgv.v[v] = from_f32<T>(live ? c[v] * xs[i][v] * f[i][v] : 0.0f);
      }
      if (on && t0 + i < p.T) {
        *reinterpret_cast<Pack<T, VEC> *>(dx + (t0 + i) * p.dxt) = dxv;
        *reinterpret_cast<Pack<T, VEC> *>(dg + (t0 + i) * p.dgt) = dgv;
      }
    }
  }
  if (on && p.grad_h0 != nullptr && warp == 0 && sub == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.grad_h0[b * p.D + d + v] = carry[v];
  }
}

// One sample of B streams whose states are rows of a table.
template <typename T, int VEC>
__global__ void k_scan_step(const T *x, int64_t xs, const T *gate, int64_t gs, int64_t n, int64_t D,
                            const int32_t *slots, int64_t rows, float *state, T *h) {
  const int64_t per = D / VEC;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n * per) return;
  const int64_t b = i / per, d = i % per * VEC;
  const int64_t row = slots != nullptr ? slots[b] : b;
  Pack<T, VEC> out{};
  if (row >= 0 && row < rows) {
    const Pack<T, VEC> xv = *reinterpret_cast<const Pack<T, VEC> *>(x + b * xs + d);
    const Pack<T, VEC> gv = *reinterpret_cast<const Pack<T, VEC> *>(gate + b * gs + d);
    float *st = state + row * D + d;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float a, f;
      gate_of(to_f32(gv.v[v]), a, f);
      const float s = fmaf(a, st[v], f * to_f32(xv.v[v]));
      st[v] = s;
      out.v[v] = from_f32<T>(s);
    }
  }
  *reinterpret_cast<Pack<T, VEC> *>(h + b * D + d) = out;
}

// How a launch covers the series: as few lanes along the channels as hold
// them, and no more warps than the samples fill.
struct Shape {
  int lanes, threads;
  int64_t tiles;
};

Shape shape_of(int64_t T, int64_t D, int vec, int steps) {
  Shape s;
  s.lanes = 1;
  while (s.lanes < 32 && (int64_t)s.lanes * vec < D) s.lanes *= 2;
  s.tiles = (D + (int64_t)s.lanes * vec - 1) / ((int64_t)s.lanes * vec);
  int warps = 1;
  while (warps < kWarps && (int64_t)warps * (32 / s.lanes) * steps < T) warps *= 2;
  s.threads = warps * 32;
  return s;
}

template <typename T>
cudaError_t scan_as(ScanArgs a, int64_t B, bool pairs, cudaStream_t stream) {
  const Shape s = shape_of(a.T, a.D, pairs ? 2 : 1, kFwdSteps);
  a.lanes = s.lanes;
  a.tiles = s.tiles;
  const unsigned grid = (unsigned)(B * s.tiles);
  if (pairs) k_scan<T, 2><<<grid, s.threads, 0, stream>>>(a);
  else k_scan<T, 1><<<grid, s.threads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t scan_backward_as(ScanArgs a, int64_t B, bool pairs, cudaStream_t stream) {
  const Shape s = shape_of(a.T, a.D, pairs ? 2 : 1, kBwdSteps);
  a.lanes = s.lanes;
  a.tiles = s.tiles;
  const unsigned grid = (unsigned)(B * s.tiles);
  if (pairs) k_scan_backward<T, 2><<<grid, s.threads, 0, stream>>>(a);
  else k_scan_backward<T, 1><<<grid, s.threads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t step_as(const void *x, int64_t xs, const void *gate, int64_t gs, int64_t B, int64_t D,
                    const int32_t *slots, int64_t rows, float *state, void *h, bool pairs,
                    cudaStream_t stream) {
  const int64_t work = B * (pairs ? D / 2 : D);
  const unsigned grid = (unsigned)((work + 255) / 256);
  const T *xp = static_cast<const T *>(x), *gp = static_cast<const T *>(gate);
  if (pairs)
    k_scan_step<T, 2><<<grid, 256, 0, stream>>>(xp, xs, gp, gs, B, D, slots, rows, state, (T *)h);
  else
    k_scan_step<T, 1><<<grid, 256, 0, stream>>>(xp, xs, gp, gs, B, D, slots, rows, state, (T *)h);
  return cudaGetLastError();
}

// Checks shared by the scan's two directions.
int check_scan(const char *fn, int dtype, const void *x, const void *gate, int64_t B, int64_t T,
               int64_t D) {
  if (!dtype_ok(dtype)) return report_error(CPAB_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
  if (B < 0 || T < 0 || D < 0) return report_error(CPAB_ERR_ARG, "%s: negative size", fn);
  if (T >= (int64_t(1) << 31)) return report_error(CPAB_ERR_SIZE, "%s: T must be below 2^31", fn);
  if (D > 0 && B > (int64_t(1) << 30) / D)
    return report_error(CPAB_ERR_SIZE, "%s: B * D must not exceed 2^30", fn);
  if (B > 0 && T > 0 && D > 0 && (x == nullptr || gate == nullptr))
    return report_error(CPAB_ERR_ARG, "%s: null input pointer", fn);
  return CPAB_OK;
}

}  // namespace
}  // namespace cpab

using namespace cpab;

extern "C" int cpab_b200_gated_scan_chunk(void) { return kChunk; }

extern "C" int cpab_b200_gated_scan(int dtype, const void *x, int64_t x_series, int64_t x_sample,
                                    const void *gate, int64_t gate_series, int64_t gate_sample,
                                    int64_t B, int64_t T, int64_t D, const int32_t *lengths,
                                    const float *h0, void *h, float *h_last, float *states,
                                    cpab_stream_t stream) {
  const int st = check_scan("gated_scan", dtype, x, gate, B, T, D);
  if (st != CPAB_OK) return st;
  if (B == 0 || D == 0) return launch_status(cudaSuccess, "");
  if (T == 0) {  // no samples: the state is what it was
    if (h_last == nullptr) return launch_status(cudaSuccess, "");
    const size_t bytes = (size_t)B * D * sizeof(float);
    return launch_status(h0 != nullptr ? cudaMemcpyAsync(h_last, h0, bytes, cudaMemcpyDeviceToDevice, stream)
                                       : cudaMemsetAsync(h_last, 0, bytes, stream), "gated_scan");
  }
  if (h == nullptr) return report_error(CPAB_ERR_ARG, "gated_scan: null output pointer");
  ScanArgs a{};
  a.x = x, a.gate = gate, a.xb = x_series, a.xt = x_sample, a.gb = gate_series, a.gt = gate_sample;
  a.T = T, a.D = D, a.lengths = lengths, a.h0 = h0, a.h = h, a.last = h_last, a.states = states;
  const int e = dtype_size(dtype);
  const bool pairs = D % 2 == 0 && aligned_to(x, x_series, e, 2 * e) && aligned_to(x, x_sample, e, 2 * e) &&
                     aligned_to(gate, gate_series, e, 2 * e) && aligned_to(gate, gate_sample, e, 2 * e) &&
                     aligned_to(h, 0, e, 2 * e);
  const cudaError_t err = dtype == CPAB_F32   ? scan_as<float>(a, B, pairs, stream)
                          : dtype == CPAB_F16 ? scan_as<__half>(a, B, pairs, stream)
                                              : scan_as<__nv_bfloat16>(a, B, pairs, stream);
  return launch_status(err, "gated_scan");
}

extern "C" int cpab_b200_gated_scan_backward(
    int dtype, const void *x, int64_t x_series, int64_t x_sample, const void *gate,
    int64_t gate_series, int64_t gate_sample, int64_t B, int64_t T, int64_t D,
    const int32_t *lengths, const float *states, const void *grad_h, const float *grad_last,
    void *grad_x, int64_t grad_x_series, int64_t grad_x_sample, void *grad_gate,
    int64_t grad_gate_series, int64_t grad_gate_sample, float *grad_h0, cpab_stream_t stream) {
  const int st = check_scan("gated_scan_backward", dtype, x, gate, B, T, D);
  if (st != CPAB_OK) return st;
  if (B == 0 || D == 0) return launch_status(cudaSuccess, "");
  if (T == 0) {
    if (grad_h0 == nullptr) return launch_status(cudaSuccess, "");
    const size_t bytes = (size_t)B * D * sizeof(float);
    return launch_status(grad_last != nullptr
                             ? cudaMemcpyAsync(grad_h0, grad_last, bytes, cudaMemcpyDeviceToDevice, stream)
                             : cudaMemsetAsync(grad_h0, 0, bytes, stream), "gated_scan_backward");
  }
  if (states == nullptr || grad_x == nullptr || grad_gate == nullptr)
    return report_error(CPAB_ERR_ARG, "gated_scan_backward: null states or gradient pointer");
  ScanArgs a{};
  a.x = x, a.gate = gate, a.xb = x_series, a.xt = x_sample, a.gb = gate_series, a.gt = gate_sample;
  a.T = T, a.D = D, a.lengths = lengths, a.states = const_cast<float *>(states);
  a.grad_h = grad_h, a.grad_last = grad_last, a.grad_x = grad_x, a.grad_gate = grad_gate;
  a.dxb = grad_x_series, a.dxt = grad_x_sample, a.dgb = grad_gate_series, a.dgt = grad_gate_sample;
  a.grad_h0 = grad_h0;
  const int e = dtype_size(dtype);
  const bool pairs = D % 2 == 0 && aligned_to(x, x_series, e, 2 * e) && aligned_to(x, x_sample, e, 2 * e) &&
                     aligned_to(gate, gate_series, e, 2 * e) && aligned_to(gate, gate_sample, e, 2 * e) &&
                     aligned_to(grad_h, 0, e, 2 * e) &&
                     aligned_to(grad_x, grad_x_series, e, 2 * e) && aligned_to(grad_x, grad_x_sample, e, 2 * e) &&
                     aligned_to(grad_gate, grad_gate_series, e, 2 * e) &&
                     aligned_to(grad_gate, grad_gate_sample, e, 2 * e);
  const cudaError_t err = dtype == CPAB_F32   ? scan_backward_as<float>(a, B, pairs, stream)
                          : dtype == CPAB_F16 ? scan_backward_as<__half>(a, B, pairs, stream)
                                              : scan_backward_as<__nv_bfloat16>(a, B, pairs, stream);
  return launch_status(err, "gated_scan_backward");
}

extern "C" int cpab_b200_gated_scan_step(int dtype, const void *x, int64_t x_row, const void *gate,
                                         int64_t gate_row, int64_t B, int64_t D,
                                         const int32_t *slots, int64_t rows, float *state, void *h,
                                         cpab_stream_t stream) {
  const int st = check_scan("gated_scan_step", dtype, x, gate, B, 1, D);
  if (st != CPAB_OK) return st;
  if (rows < 0 || (slots == nullptr && rows < B))
    return report_error(CPAB_ERR_ARG, "gated_scan_step: %lld state rows for %lld streams",
                        (long long)rows, (long long)B);
  if (B == 0 || D == 0) return launch_status(cudaSuccess, "");
  if (h == nullptr || (state == nullptr && rows > 0))
    return report_error(CPAB_ERR_ARG, "gated_scan_step: null state or output pointer");
  const int e = dtype_size(dtype);
  const bool pairs = D % 2 == 0 && aligned_to(x, x_row, e, 2 * e) && aligned_to(gate, gate_row, e, 2 * e) &&
                     aligned_to(h, 0, e, 2 * e);
  const cudaError_t err =
      dtype == CPAB_F32   ? step_as<float>(x, x_row, gate, gate_row, B, D, slots, rows, state, h, pairs, stream)
      : dtype == CPAB_F16 ? step_as<__half>(x, x_row, gate, gate_row, B, D, slots, rows, state, h, pairs, stream)
                          : step_as<__nv_bfloat16>(x, x_row, gate, gate_row, B, D, slots, rows, state, h,
                                                   pairs, stream);
  return launch_status(err, "gated_scan_step");
}
