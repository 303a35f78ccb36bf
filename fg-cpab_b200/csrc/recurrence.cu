// The gated linear recurrence over time and its gradient.
//
//   a_t = sigmoid(z_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t
//
// per channel, for gate logits z and inputs x [B, T, D] in f32, f16 or bf16
// and a float32 state.  Both a and 1 - a come from one exponential in float32
// (1 - a = sigmoid(-z) keeps its relative precision as a -> 1: gate_of).
//
// A step (a, b): h -> a h + b; two steps compose to (a2 a1, a2 b1 + b2), which
// is associative.  (Where the a's are so near 1 that a product's second-order term
// falls below half its last place, that term is lost each time: 8192 samples of
// logits N(12, 1.5), a memory of 50,000, are 8e-6 off, sample by sample 3e-6.)
//
// A block owns a tile of channels of one piece of a series and walks it stage by
// stage: cp.async brings the next stages into shared memory, each thread reads a
// segment of kFwdSteps or kBwdSteps samples of its channels from there and composes
// them, and the segments' compositions are scanned over the warp (shuffles) and the
// block (shared memory) to give each segment the state it starts from; a second
// pass over the registers writes the segment's states.
//
// A series is one piece where there are tiles enough to fill the GPU.  Else a
// kernel before composes every kSpan samples, and a block begins at the state
// that the spans before its own piece lead to.
//
// The gradient runs the same way from the last sample back:
//   delta_t = dh_t + c_{t+1},  c_t = a_t delta_t
//   dx_t = (1 - a_t) delta_t,  dz_t = c_t (h_{t-1} - x_t) (1 - a_t)
// with h_{t-1} recomputed in float32 from the states that the forward keeps at
// the start of every kChunk samples (reading the rounded output instead would
// cost more bytes and lose the difference h_{t-1} - x_t where it is small).
//
// What bounds it.  In 16 bits the forward moves 6 and the gradient 10 bytes per
// sample and channel, against 24 and 47 instructions (two of them the special
// functions'): with tiles enough the blocks issue 72% and 75% of the time and
// move 5.9 and 5.4 TB/s (64x512x2048 bf16: 69 and 123 us; a copy: 6.46 TB/s).
// Tiles of 64-byte rows and blocks of 4 warps are the fastest of 32, 64 and 128
// bytes (64x512x2048: forward 85, 69, 81 us, gradient 141, 123 of 32 and 64).
// With few tiles the spread over the SMs costs most (16x2048x1024: 512 tiles on
// 148 SMs, 41 and 71 us, 5.0 and 4.8 TB/s); clusters of blocks that exchange their
// compositions stage by stage were slower than composing the spans first
// (1x65536x512: 76 and 143 us with the best cluster sizes, 67 and 97 with spans).
#include <type_traits>

#include "sequence.cuh"

namespace cpab {
namespace {

constexpr int kChunk = 64;     // samples between two kept states
constexpr int kFwdSteps = 16;  // samples of a thread's segment (divide kChunk)
constexpr int kBwdSteps = 8;
// Samples composed together where a series is cut into pieces, of which these are
// multiples (128, 256, 512 samples: 1x65536x512 bf16 70, 67, 70 us, gradient 102, 97,
// 103; 3x9000x333 42, 48, 56; 1x65536x256 f32 72, 66, 64, gradient 112, 96, 91).
constexpr int kSpan = 256;
static_assert(kChunk % kFwdSteps == 0 && kChunk % kBwdSteps == 0, "states start segments");
// Warps of a full block with 2^log2 lanes along the channels: a stage has 8
// segments (16 in blocks of 8 warps, for tiles that are too few to keep 4 blocks on
// an SM).  16 warps fit on an SM.
__host__ __device__ constexpr int warps_of(int log2) { return log2 == 4 ? 4 : 2; }
constexpr int kWide = 8, kResidentWarps = 16;
static_assert((8 * kBwdSteps) % kChunk == 0, "a full block's stage starts on a kept state");

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
  int aligned;              // every row of a tile starts on 16 bytes
  int words;                // inputs' and outputs' rows start on words
  int64_t x_end, gate_end, grad_h_end;  // bytes from a tensor's start to its end
  int ring;                 // stages in shared memory
  int64_t tiles;            // channel tiles of a series
  int64_t piece;            // samples of a piece of a series (of kSpan, if more than one)
  int pieces;
  float2 *totals;           // [B, ceil(T / kSpan), D]: compositions of spans (pieces > 1)
};

// The channels a lane holds: a 32-bit word's worth.
template <int V>
struct Lane {
  float v[V];
  __device__ __forceinline__ float operator[](int i) const { return v[i]; }
  __device__ __forceinline__ void set(int i, float f) { v[i] = f; }
};
template <int V>
__device__ __forceinline__ Lane<V> fma(Lane<V> a, Lane<V> b, Lane<V> c) {
  Lane<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = fmaf(a.v[i], b.v[i], c.v[i]);
  return r;
}
template <int V>
__device__ __forceinline__ Lane<V> operator*(Lane<V> a, Lane<V> b) {
  Lane<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = a.v[i] * b.v[i];
  return r;
}
template <int V>
__device__ __forceinline__ Lane<V> operator+(Lane<V> a, Lane<V> b) {
  Lane<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = a.v[i] + b.v[i];
  return r;
}
template <int V>
__device__ __forceinline__ Lane<V> all(float f) {
  Lane<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, f);
  return r;
}

// Words of shared or global memory as float32 channels and back.
__device__ __forceinline__ Lane<1> unpack(uint32_t w, float) { return {{__uint_as_float(w)}}; }
template <typename T>
__device__ __forceinline__ Lane<2> unpack(uint32_t w, T) {
  const float2 f = unpack_pair<T>(w);
  return {{f.x, f.y}};
}
__device__ __forceinline__ uint32_t pack(Lane<1> a, float) { return __float_as_uint(a[0]); }
template <typename T>
__device__ __forceinline__ uint32_t pack(Lane<2> a, T) {
  return pack_pair<T>(a[0], a[1]);
}
// +inf in every element: the gate of a sample that is none (a = 1, 1 - a = 0).
__device__ __forceinline__ uint32_t closed_gate(float) { return 0x7F800000u; }
__device__ __forceinline__ uint32_t closed_gate(__nv_bfloat16) { return 0x7F807F80u; }
__device__ __forceinline__ uint32_t closed_gate(__half) { return 0x7C007C00u; }

// The hardware's approximate exponential (2^t) and reciprocal: 2 and 1 units in the
// last place.
__device__ __forceinline__ float exp2_near(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ float reciprocal_near(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

// a = sigmoid(z) and f = 1 - a = sigmoid(-z) from one exponential; f = e / (1 + e)
// with e = exp(-z) keeps its size's precision as a -> 1.
//
// In float32 (PRECISE) both are as good as the two instructions.  The exponential's
// argument t is rounded, which is off by up to 2^-24 |t| ln 2 of e (3e-7 at |z| = 7,
// 2e-6 at 40): what is left of z beside t ln 2 is put back.  And the larger of a
// and f is 1 less the smaller, rounded once: the reciprocal itself is off by 1.3e-8
// on average near a logit of 7, which a memory of 1 / (1 - a) samples adds up
// (states of 8192 samples of logits N(7, 1.5): 3.0e-6 off against 3.6e-7, the same
// recursion sample by sample 7.5e-7).
//
// 16-bit inputs are rounded to 2^-12 of their size at best, and so are the outputs (the
// last state, in float32, holds no more than they gave).
// There that precision is not worth its five instructions a sample and channel, of
// 24 that bound the kernel (the last two cost 8x16384x1024 bf16 160 -> 167 us and its
// gradient 293 -> 309; float32, with twice the bytes and 52% of the issue slots taken,
// hardly shows them: 8x8192x512 78 and 119 us with and without, 8x8192x499 190 -> 192,
// 256x4x4096 18 -> 20 and 23 -> 27).
template <bool PRECISE, int V>
__device__ __forceinline__ void gate_of(Lane<V> z, Lane<V> &a, Lane<V> &f) {
  constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  if constexpr (PRECISE) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float t = fabsf(z[i]) * -kLog2E;
      float e = exp2_near(t);  // of -|z|
      if (t > -126.0f) e = fmaf(e, fmaf(t, -kLn2, -fabsf(z[i])), e);
      const float r = reciprocal_near(e + 1.0f), less = e * r, more = fmaf(-e, r, 1.0f);
      a.set(i, z[i] > 0.0f ? more : less);
      f.set(i, z[i] > 0.0f ? less : more);
    }
  } else {
    // (step by step over the lane's channels: together they cost the gradient 4%)
    const Lane<V> t = z * all<V>(-kLog2E);
    Lane<V> e;
#pragma unroll
    for (int i = 0; i < V; ++i) e.set(i, exp2_near(t[i]));
    const Lane<V> d = e + all<V>(1.0f);
#pragma unroll
    for (int i = 0; i < V; ++i) a.set(i, reciprocal_near(d[i]));
    f = e * a;
    // (where e > 1, 1 - a loses nothing and is right for e = inf too)
    const Lane<V> g = fma(a, all<V>(-1.0f), all<V>(1.0f));
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e[i] > 1.0f) f.set(i, g[i]);
  }
}

__device__ __forceinline__ uint32_t shared_address(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// One input: a tile's samples of a series.
template <typename T>
struct Rows {
  const T *first;           // sample 0, the tile's first channel
  int64_t stride;           // of samples, in elements
  const char *begin, *end;  // of the whole tensor
  uint32_t fill;            // the value of a sample that is none
};

// A stage in shared memory: a row per sample, `kPitch` words of it, and a gap of
// a row after each segment of L, which keeps a warp's segments on different
// banks.  Rows that start on 16 bytes lie there from word 0 on.  Of others the
// 16-byte pieces of memory that hold them are copied as they are, so a row
// starts at byte (address & 15).
template <int L, int LOG2, bool ALIGNED>
struct Stage {
  static constexpr int kPitch = (1 << LOG2) + (ALIGNED ? 0 : 4);
  static constexpr int kCopies = kPitch / 4;  // of 16 bytes, per row
  __host__ __device__ static constexpr int words(int samples) { return (samples + samples / L) * kPitch; }
  __device__ static __forceinline__ int row(int r) { return (r + r / L) * kPitch; }
};

// Copies samples s0 .. s0 + rows - 1 of a tile to `to`.  Nothing is read of
// samples from `len` on nor outside the tensor.
template <typename T, int L, int LOG2, bool ALIGNED>
__device__ __forceinline__ void copy_stage(uint32_t *to, const Rows<T> &in, int s0, int rows, int len, int channels) {
  using S = Stage<L, LOG2, ALIGNED>;
  constexpr int V = 4 / sizeof(T);
  const uint4 fill = make_uint4(in.fill, in.fill, in.fill, in.fill);
  if constexpr (ALIGNED) {
    const int step = blockDim.x / S::kCopies, word = (threadIdx.x % S::kCopies) * 4;
    int r = threadIdx.x / S::kCopies;
    const T *src = in.first + (int64_t)(s0 + r) * in.stride + word * V;
    if (s0 + rows <= len && channels >= V << LOG2) {
#pragma unroll
      for (int k = 0; k < L / 4; ++k, r += step, src += step * in.stride)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(to + S::row(r) + word)),
                     "l"(src));
      return;
    }
#pragma unroll
    for (int k = 0; k < L / 4; ++k, r += step, src += step * in.stride) {
      uint32_t *dst = to + S::row(r) + word;
      if (s0 + r < len && word * V < channels) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(dst)), "l"(src));
      } else {
        *reinterpret_cast<uint4 *>(dst) = fill;
      }
    }
  } else {
    for (int q = threadIdx.x; q < rows * S::kCopies; q += blockDim.x) {
      const int r = q / S::kCopies, piece = q % S::kCopies;
      uint32_t *dst = to + S::row(r) + piece * 4;
      if (s0 + r >= len) {
        *reinterpret_cast<uint4 *>(dst) = fill;
        continue;
      }
      const char *row = reinterpret_cast<const char *>(in.first + (int64_t)(s0 + r) * in.stride);
      const char *src = reinterpret_cast<const char *>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15) + piece * 16;
      const char *row_end = row + channels * (int)sizeof(T);
      if (src >= row_end) continue;
      if (src >= in.begin && src + 16 <= in.end) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(dst)), "l"(src));
      } else {  // the tensor's first or last bytes: its elements one by one
        for (int i = 0; i < 16; i += (int)sizeof(T))
          if (src + i >= row && src + i < row_end)
            reinterpret_cast<T *>(dst)[i / sizeof(T)] = *reinterpret_cast<const T *>(src + i);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ Rows<T> rows_of(const void *tensor, int64_t at, int64_t stride, int64_t bytes, uint32_t fill) {
  const char *begin = static_cast<const char *>(tensor);
  return {static_cast<const T *>(tensor) + at, stride, begin, begin + bytes, fill};
}

// copy_stage for the stages of a full block whose rows start on 16 bytes and
// are all there, with what a thread's addresses have in common kept.
template <typename T, int L, int LOG2, int WARPS>
struct Feed {
  using S = Stage<L, LOG2, true>;
  static constexpr int kThreads = WARPS * 32, kRows = kThreads / S::kCopies;  // rows copied at a time
  static_assert(kRows % L == 0, "a thread's rows lie equally far apart in shared memory");
  const char *src;          // the thread's first copy of the next stage
  int64_t row_step, stage_step;
  __device__ __forceinline__ Feed(const Rows<T> &in, int s0, int stage, int direction) {
    constexpr int V = 4 / sizeof(T);
    src = reinterpret_cast<const char *>(in.first + (int64_t)(s0 + (int)threadIdx.x / S::kCopies) * in.stride +
                                         (threadIdx.x % S::kCopies) * 4 * V);
    row_step = kRows * in.stride * (int64_t)sizeof(T);
    stage_step = direction * (int64_t)stage * in.stride * (int64_t)sizeof(T);
  }
  // Bytes of the thread's first copy from the start of a stage in shared memory.
  static __device__ __forceinline__ uint32_t place() {
    return (S::row((int)threadIdx.x / S::kCopies) + (threadIdx.x % S::kCopies) * 4) * 4;
  }
  __device__ __forceinline__ void copy(uint32_t to) const {
#pragma unroll
    for (int k = 0; k < L / 4; ++k)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * (kRows + kRows / L) * S::kPitch * 4),
                   "l"(src + k * row_step));
  }
  __device__ __forceinline__ void next() { src += stage_step; }
};

// A lane's word of each of L consecutive samples, from sample t0 of a tile and
// row r of its stage on.
template <typename T, int L, int LOG2, bool ALIGNED>
struct Words {
  using S = Stage<L, LOG2, ALIGNED>;
  const uint32_t *row;
  int at, step;             // of the row's start, as bytes beyond a multiple of 16
  __device__ __forceinline__ Words(const uint32_t *stage, int r, int cl, const Rows<T> &in, int t0) {
    row = stage + S::row(r) + cl;
    at = ALIGNED ? 0 : (int)(reinterpret_cast<uintptr_t>(in.first + t0 * in.stride) & 15);
    step = ALIGNED ? 0 : (int)(in.stride * (int64_t)sizeof(T)) & 15;
  }
  __device__ __forceinline__ uint32_t operator[](int i) const {
    const uint32_t *w = row + i * S::kPitch;
    if constexpr (ALIGNED) {
      return *w;
    } else {
      const char *q = reinterpret_cast<const char *>(w) + ((at + i * step) & 15);
      if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t *>(q);
      // (two halves: a word and a funnel shift over two cost 5% more)
      const unsigned short *h = reinterpret_cast<const unsigned short *>(q);
      return h[0] | (uint32_t)h[1] << 16;
    }
  }
};

// Stores a lane's channels of one sample: as a word, or of 16-bit elements
// whose pairs do not lie on words the first `n`.
template <bool WORDS, typename T, int V>
__device__ __forceinline__ void store_lane(T *row, Lane<V> v, int n) {
  const uint32_t w = pack(v, T{});
  if (WORDS || V == 1) {
    *reinterpret_cast<uint32_t *>(row) = w;
  } else {
    unsigned short *q = reinterpret_cast<unsigned short *>(row);
    q[0] = (unsigned short)w;
    if (n > 1) q[1] = (unsigned short)(w >> 16);
  }
}

template <int V>
__device__ __forceinline__ Lane<V> load_state(const float *row, int64_t d, int64_t D) {
  Lane<V> r = all<V>(0.0f);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (d + i < D) r.set(i, row[d + i]);
  return r;
}
template <int V>
__device__ __forceinline__ void store_state(float *row, int64_t d, int64_t D, Lane<V> v) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (d + i < D) row[d + i] = v[i];
}

template <int V>
__device__ __forceinline__ Lane<V> shuffle_up(Lane<V> v, int o) {
  Lane<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, __shfl_up_sync(~0u, v[i], o));
  return r;
}
template <int V>
__device__ __forceinline__ Lane<V> shuffle_down(Lane<V> v, int o) {
  Lane<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, __shfl_down_sync(~0u, v[i], o));
  return r;
}

// A composition of steps: state -> A state + H.
template <int V>
struct Step {
  Lane<V> A, H;
};
template <int V>
__device__ __forceinline__ void put(float2 *at, Lane<V> A, Lane<V> H) {
#pragma unroll
  for (int i = 0; i < V; ++i) at[i] = make_float2(A[i], H[i]);
}
template <int V>
__device__ __forceinline__ Step<V> get(const float2 *at) {
  Step<V> s;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s.A.set(i, at[i].x);
    s.H.set(i, at[i].y);
  }
  return s;
}

// Where a thread stands.
template <int L, int LOG2, int V>
struct Place {
  static constexpr int kLanes = 1 << LOG2, kSubs = 32 >> LOG2;
  int lane, warp, sub, cl, seg;
  int64_t b, d;          // series; first channel of the lane
  int channels;          // of the tile
  int len, stage;
  int piece, first, end; // the block's samples; from len on there are none
  int live;              // stages that have some
  __device__ __forceinline__ Place(const ScanArgs &p) {
    lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    sub = lane >> LOG2, cl = lane & (kLanes - 1), seg = warp * kSubs + sub;
    // neighbouring blocks: neighbouring channels
    const int64_t c = blockIdx.x / p.tiles, d0 = (blockIdx.x % p.tiles) * (kLanes * V);
    b = c / p.pieces;
    piece = (int)(c % p.pieces);
    d = d0 + cl * V;
    channels = (int)min((int64_t)(kLanes * V), p.D - d0);
    len = (int)p.T;
    if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), len);
    stage = (int)(blockDim.x >> 5) * kSubs * L;
    first = (int)(piece * p.piece);
    end = (int)min((piece + 1) * p.piece, p.T);
    live = len > first ? (min(len, end) - first + stage - 1) / stage : 0;
  }
};

// `ring` is 1, 2 or 3 (shape_of).
__device__ __forceinline__ void wait_for_stage(int ring) {
  if (ring == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (ring == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
  __syncthreads();
}

// The compositions of spans of kSpan samples: forward (A, H) with the state
// after one A state + H, for the gradient (A, R) with c at its first sample
// A c + R.  A block takes a span of 32 lanes' channels, a warp a part of it:
// 1x65536x512 bf16 in 30 us (134 MB, 4.5 TB/s, 65% of the issue slots), read once
// more by the main kernel.  The spans that no piece needs (those of
// the last piece, for the gradient of the first) are left out.
constexpr int kTotalWarps = 8, kTotalSteps = kSpan / kTotalWarps;

template <typename T>
__device__ __forceinline__ uint32_t load_word(const T *row, int n, bool words) {
  if (sizeof(T) == 4 || words) return *reinterpret_cast<const uint32_t *>(row);
  const unsigned short *q = reinterpret_cast<const unsigned short *>(row);
  return q[0] | (n > 1 ? (uint32_t)q[1] << 16 : 0u);
}

// How many of a series' spans are composed: those before its last piece, for the
// gradient those after its first.
template <bool BACK>
__host__ __device__ __forceinline__ int64_t spans_needed(const ScanArgs &p) {
  return BACK ? (p.T + kSpan - 1) / kSpan - p.piece / kSpan : (p.pieces - 1) * (p.piece / kSpan);
}

template <typename T, bool BACK>
__global__ void __launch_bounds__(kTotalWarps * 32) k_scan_totals(const __grid_constant__ ScanArgs p) {
  constexpr int L = 16, V = 4 / sizeof(T);
  static_assert(kTotalSteps % L == 0, "a warp's part of a span is read L samples at a time");
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ float2 total[kTotalWarps][32][V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t tiles = (p.D + 32 * V - 1) / (32 * V), spans = (p.T + kSpan - 1) / kSpan;
  const int64_t c = blockIdx.x / tiles, d = (blockIdx.x % tiles) * (32 * V) + lane * V;
  const int64_t needed = spans_needed<BACK>(p), b = c / needed, span = c % needed + (BACK ? spans - needed : 0);
  const int n = (int)min(p.D - d, (int64_t)V);
  int len = (int)p.T;
  if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), len);
  // u: what is added per sample, f x or dh
  const T *u = BACK ? static_cast<const T *>(p.grad_h) + b * p.T * p.D + d
                    : static_cast<const T *>(p.x) + b * p.xb + d;
  const int64_t ut = BACK ? p.D : p.xt;
  const T *g = static_cast<const T *>(p.gate) + b * p.gb + d;
  const int first = (int)(span * kSpan) + warp * kTotalSteps;
  const bool any = n > 0 && (!BACK || p.grad_h != nullptr);
  Lane<V> A = all<V>(1.0f), H = all<V>(0.0f);
#pragma unroll 1
  for (int k = 0; k < kTotalSteps; k += L) {
    const int t0 = first + (BACK ? kTotalSteps - L - k : k);
    if (t0 >= len) continue;
    uint32_t gw[L], uw[L];
    const T *gr = g + t0 * p.gt, *ur = u + t0 * ut;
    if (any && p.words && t0 + L <= len) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        gw[i] = *reinterpret_cast<const uint32_t *>(gr + i * p.gt);
        uw[i] = *reinterpret_cast<const uint32_t *>(ur + i * ut);
      }
    } else if (sizeof(T) == 2 && any && n == V && t0 + L <= len) {
      // a lane's second element by itself where pairs do not lie on words
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const unsigned short *gh = reinterpret_cast<const unsigned short *>(gr + i * p.gt);
        const unsigned short *uh = reinterpret_cast<const unsigned short *>(ur + i * ut);
        gw[i] = gh[0] | (uint32_t)gh[V - 1] << 16;
        uw[i] = uh[0] | (uint32_t)uh[V - 1] << 16;
      }
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i, gr += p.gt, ur += ut) {
        gw[i] = closed_gate(T{});
        uw[i] = 0u;
        if (n > 0 && t0 + i < len) gw[i] = load_word(gr, n, p.words);
        if (any && t0 + i < len) uw[i] = load_word(ur, n, p.words);
      }
    }
#pragma unroll
    for (int k = 0; k < L; ++k) {
      const int i = BACK ? L - 1 - k : k;
      Lane<V> a, f;
      gate_of<sizeof(T) == 4>(unpack(gw[i], T{}), a, f);
      H = BACK ? a * (H + unpack(uw[i], T{})) : fma(a, H, f * unpack(uw[i], T{}));
      A = A * a;
    }
  }
  put(total[warp][lane], A, H);
  __syncthreads();
  if (warp != 0 || n <= 0) return;
  A = all<V>(1.0f), H = all<V>(0.0f);
#pragma unroll
  for (int k = 0; k < kTotalWarps; ++k) {
    const Step<V> q = get<V>(total[BACK ? kTotalWarps - 1 - k : k][lane]);
    H = fma(q.A, H, q.H);
    A = A * q.A;
  }
  float2 *to = p.totals + (b * spans + span) * p.D + d;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) to[i] = make_float2(A[i], H[i]);
}

// A lane's state at the start of its piece from the spans before it (forward),
// or its c after the piece from those after it (gradient).  The block's
// segments compose a part each; `total` is shared memory of kWarps * kSubs.
template <int V, bool BACK, typename At>
__device__ __forceinline__ Lane<V> through_spans(const ScanArgs &p, const At &at, float2 (*total)[V], int mine,
                                                 Lane<V> c) {
  if (p.pieces == 1) return c;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int all_spans = (int)((p.T + kSpan - 1) / kSpan), each = (int)(p.piece / kSpan);
  const int from = BACK ? min((at.piece + 1) * each, all_spans) : 0;
  const int count = BACK ? all_spans - from : at.piece * each;
  const int segments = (int)(blockDim.x >> 5) * At::kSubs, share = (count + segments - 1) / segments;
  const int lo = min(at.seg * share, count), hi = min(lo + share, count);
  Lane<V> A = all<V>(1.0f), H = all<V>(0.0f);
  const float2 *q = p.totals + (at.b * all_spans + from) * p.D + at.d;
#pragma unroll 4
  for (int k = 0; k < hi - lo; ++k) {
    const float2 *row = q + (int64_t)(BACK ? hi - 1 - k : lo + k) * p.D;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < mine) {
        const float2 t = row[i];
        H.set(i, fmaf(t.x, H[i], t.y));
        A.set(i, A[i] * t.x);
      }
  }
  put(total[at.seg * At::kLanes + at.cl], A, H);
  __syncthreads();
  for (int k = 0; k < segments; ++k) {
    const Step<V> t = get<V>(total[(BACK ? segments - 1 - k : k) * At::kLanes + at.cl]);
    c = fma(t.A, c, t.H);
  }
  __syncthreads();
  return c;
}

// The forward.  Segments of 16 samples: their composition over the warp and the
// block costs 6 shuffles and 4 reads of shared memory per segment, which 8
// samples do not pay for.  Two stages in flight: a third costs a block of an SM.
template <typename T, int LOG2, int WARPS, bool ALIGNED>
__global__ void __launch_bounds__(WARPS * 32, kResidentWarps / WARPS) k_scan(const __grid_constant__ ScanArgs p) {
  constexpr int L = kFwdSteps, V = 4 / sizeof(T), kWarps = WARPS;
  using At = Place<L, LOG2, V>;
  extern __shared__ uint4 ring_memory[];
  __shared__ float2 warp_total[kWarps][At::kLanes][V], span_total[kWarps * 32][V];
  const At at(p);
  const int mine = at.channels - at.cl * V;  // channels of this lane, if positive
  const bool on = mine > 0;
  const int64_t d0 = at.d - at.cl * V;
  const Rows<T> x = rows_of<T>(p.x, at.b * p.xb + d0, p.xt, p.x_end, 0u);
  const Rows<T> g = rows_of<T>(p.gate, at.b * p.gb + d0, p.gt, p.gate_end, closed_gate(T{}));
  T *h = static_cast<T *>(p.h) + at.b * p.T * p.D + at.d;
  const int64_t chunks = (p.T + kChunk - 1) / kChunk;
  const int words = Stage<L, LOG2, ALIGNED>::words(at.stage);  // of one tensor's stage
  uint32_t *ring = reinterpret_cast<uint32_t *>(ring_memory);

  const bool whole = ALIGNED && blockDim.x == kWarps * 32 && at.channels == At::kLanes * V;
  Feed<T, L, LOG2, WARPS> x_feed(x, at.first, at.stage, 1), g_feed(g, at.first, at.stage, 1);
  const uint32_t place = shared_address(ring) + Feed<T, L, LOG2, WARPS>::place();
  auto fetch = [&](int k, int slot) {
    if (k < at.live) {
      const int s0 = at.first + k * at.stage;
      if (whole && s0 + at.stage <= at.len) {
        x_feed.copy(place + slot * 2 * words * 4);
        g_feed.copy(place + (slot * 2 + 1) * words * 4);
      } else {
        uint32_t *to = ring + slot * 2 * words;
        copy_stage<T, L, LOG2, ALIGNED>(to, x, s0, at.stage, at.len, at.channels);
        copy_stage<T, L, LOG2, ALIGNED>(to + words, g, s0, at.stage, at.len, at.channels);
      }
      x_feed.next();
      g_feed.next();
    }
    asm volatile("cp.async.commit_group;");
  };
  for (int k = 0; k < p.ring; ++k) fetch(k, k);

  for (int k = threadIdx.x; k < kWarps * At::kLanes; k += blockDim.x)  // warps that are not there
    put(warp_total[k >> LOG2][k & (At::kLanes - 1)], all<V>(1.0f), all<V>(0.0f));
  Lane<V> carry = all<V>(0.0f);
  if (p.h0 != nullptr) carry = load_state<V>(p.h0 + at.b * p.D, at.d, p.D);
  carry = through_spans<V, false>(p, at, span_total, mine, carry);

  T *h_row = h + (int64_t)(at.first + at.seg * L) * p.D;
  const int64_t h_stage = at.stage * p.D;
  int slot = 0;
  for (int k = 0; k < at.live; ++k) {
    const int t0 = at.first + k * at.stage + at.seg * L;
    wait_for_stage(p.ring);
    const uint32_t *here = ring + slot * 2 * words;
    const Words<T, L, LOG2, ALIGNED> xs(here, at.seg * L, at.cl, x, t0), gs(here + words, at.seg * L, at.cl, g, t0);
    Lane<V> a[L], in[L], A = all<V>(1.0f), H = all<V>(0.0f);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      Lane<V> f;
      gate_of<sizeof(T) == 4>(unpack(gs[i], T{}), a[i], f);
      in[i] = f * unpack(xs[i], T{});
      H = fma(a[i], H, in[i]);
      A = A * a[i];
    }
#pragma unroll
    for (int o = At::kLanes; o < 32; o <<= 1) {
      const Lane<V> pa = shuffle_up(A, o), ph = shuffle_up(H, o);
      if (at.lane >= o) {
        H = fma(A, ph, H);
        A = A * pa;
      }
    }
    if (at.sub == At::kSubs - 1) put(warp_total[at.warp][at.cl], A, H);
    __syncthreads();
    fetch(k + p.ring, slot);
    slot = slot + 1 == p.ring ? 0 : slot + 1;
    Lane<V> start = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == at.warp) start = carry;
      const Step<V> q = get<V>(warp_total[w][at.cl]);
      carry = fma(q.A, carry, q.H);
    }
    Lane<V> state = start;
    const Lane<V> ea = shuffle_up(A, At::kLanes), eh = shuffle_up(H, At::kLanes);
    if (at.sub > 0) state = fma(ea, start, eh);
    if (p.states != nullptr && t0 % kChunk == 0 && t0 < at.len)
      store_state(p.states + (at.b * chunks + t0 / kChunk) * p.D, at.d, p.D, state);
    auto write = [&](auto words) {
      T *row = h_row;
      if (t0 + L <= at.len) {
#pragma unroll
        for (int i = 0; i < L; ++i, row += p.D) {
          state = fma(a[i], state, in[i]);
          store_lane<words.value>(row, state, mine);
        }
      } else {
#pragma unroll
        for (int i = 0; i < L; ++i, row += p.D) {
          state = fma(a[i], state, in[i]);
          if (t0 + i < p.T) store_lane<words.value>(row, t0 + i < at.len ? state : all<V>(0.0f), mine);
        }
      }
    };
    if (on) {
      if (p.words) write(std::true_type{});
      else write(std::false_type{});
    }
    h_row += h_stage;
  }
  // Stages past the series' end: zeros.
  for (int s0 = at.first + at.live * at.stage; s0 < at.end; s0 += at.stage) {
    const int t0 = s0 + at.seg * L;
    for (int i = 0; i < L; ++i)
      if (on && t0 + i < at.end) store_lane<false>(h + (t0 + i) * p.D, all<V>(0.0f), mine);
  }
  if (p.last != nullptr && at.piece == p.pieces - 1 && at.warp == 0 && at.sub == 0)
    store_state(p.last + at.b * p.D, at.d, p.D, carry);
}

// The gradient.  Both directions are composed in one pass over a stage: from the
// kept state forward for h_{t-1}, and from the last sample back for c.  a, f, x
// and dh of a segment stay in registers between, which 8 samples of leave room
// for (128 registers a thread, no spills).
template <typename T, int LOG2, int WARPS, bool ALIGNED>
__global__ void __launch_bounds__(WARPS * 32, kResidentWarps / WARPS) k_scan_backward(const __grid_constant__ ScanArgs p) {
  constexpr int L = kBwdSteps, V = 4 / sizeof(T), kWarps = WARPS;
  using At = Place<L, LOG2, V>;
  extern __shared__ uint4 ring_memory[];
  __shared__ float2 up_total[kWarps][At::kLanes][V], down_total[kWarps][At::kLanes][V];
  __shared__ float2 span_total[kWarps * 32][V];
  const At at(p);
  const int mine = at.channels - at.cl * V;  // channels of this lane, if positive
  const bool on = mine > 0;
  const int64_t d0 = at.d - at.cl * V;
  const Rows<T> x = rows_of<T>(p.x, at.b * p.xb + d0, p.xt, p.x_end, 0u);
  const Rows<T> g = rows_of<T>(p.gate, at.b * p.gb + d0, p.gt, p.gate_end, closed_gate(T{}));
  const Rows<T> dh = rows_of<T>(p.grad_h, at.b * p.T * p.D + d0, p.D, p.grad_h_end, 0u);
  T *dx = static_cast<T *>(p.grad_x) + at.b * p.dxb + at.d;
  T *dg = static_cast<T *>(p.grad_gate) + at.b * p.dgb + at.d;
  const int64_t chunks = (p.T + kChunk - 1) / kChunk;
  const int words = Stage<L, LOG2, ALIGNED>::words(at.stage);
  uint32_t *ring = reinterpret_cast<uint32_t *>(ring_memory);

  // Stage k counts from the last one with samples back.
  const int s_last = at.first + (at.live - 1) * at.stage;
  const bool whole = ALIGNED && blockDim.x == kWarps * 32 && at.channels == At::kLanes * V && p.grad_h != nullptr;
  Feed<T, L, LOG2, WARPS> x_feed(x, s_last, at.stage, -1), g_feed(g, s_last, at.stage, -1), d_feed(dh, s_last, at.stage, -1);
  const uint32_t place = shared_address(ring) + Feed<T, L, LOG2, WARPS>::place();
  auto fetch = [&](int k, int slot) {
    if (k < at.live) {
      const int s0 = s_last - k * at.stage;
      if (whole && s0 + at.stage <= at.len) {
        x_feed.copy(place + slot * 3 * words * 4);
        g_feed.copy(place + (slot * 3 + 1) * words * 4);
        d_feed.copy(place + (slot * 3 + 2) * words * 4);
      } else {
        uint32_t *to = ring + slot * 3 * words;
        copy_stage<T, L, LOG2, ALIGNED>(to, x, s0, at.stage, at.len, at.channels);
        copy_stage<T, L, LOG2, ALIGNED>(to + words, g, s0, at.stage, at.len, at.channels);
        copy_stage<T, L, LOG2, ALIGNED>(to + 2 * words, dh, s0, at.stage, p.grad_h != nullptr ? at.len : 0,
                                        at.channels);
      }
      x_feed.next();
      g_feed.next();
      d_feed.next();
    }
    asm volatile("cp.async.commit_group;");
  };
  for (int k = 0; k < p.ring; ++k) fetch(k, k);

  for (int k = threadIdx.x; k < kWarps * At::kLanes; k += blockDim.x) {
    put(up_total[k >> LOG2][k & (At::kLanes - 1)], all<V>(1.0f), all<V>(0.0f));
    put(down_total[k >> LOG2][k & (At::kLanes - 1)], all<V>(1.0f), all<V>(0.0f));
  }
  Lane<V> carry = all<V>(0.0f);  // c of the first sample after the stage
  if (p.grad_last != nullptr) carry = load_state<V>(p.grad_last + at.b * p.D, at.d, p.D);
  carry = through_spans<V, true>(p, at, span_total, mine, carry);

  const float *base_row = p.states + (at.b * chunks + s_last / kChunk) * p.D;
  T *dx_row = dx + (int64_t)(s_last + at.seg * L + L - 1) * p.dxt, *dg_row = dg + (int64_t)(s_last + at.seg * L + L - 1) * p.dgt;
  const int64_t dx_stage = at.stage * p.dxt, dg_stage = at.stage * p.dgt;
  int slot = 0;
  for (int k = 0; k < at.live; ++k) {
    const int t0 = s_last - k * at.stage + at.seg * L;
    Lane<V> base = load_state<V>(base_row, at.d, p.D);
    base_row -= at.stage / kChunk * p.D;
    wait_for_stage(p.ring);
    const uint32_t *here = ring + slot * 3 * words;
    const Words<T, L, LOG2, ALIGNED> xs(here, at.seg * L, at.cl, x, t0), gs(here + words, at.seg * L, at.cl, g, t0);
    const Words<T, L, LOG2, ALIGNED> ds(here + 2 * words, at.seg * L, at.cl, dh, t0);
    Lane<V> a[L], f[L], xv[L], gr[L];
    Lane<V> A = all<V>(1.0f), H = all<V>(0.0f), R = all<V>(0.0f);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      gate_of<sizeof(T) == 4>(unpack(gs[i], T{}), a[i], f[i]);
      xv[i] = unpack(xs[i], T{});
      gr[i] = unpack(ds[i], T{});
      H = fma(a[i], H, f[i] * xv[i]);
      A = A * a[i];
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) R = a[i] * (R + gr[i]);
    // Over the warp's segments: (Af, H) from the first on, (Ab, R) from the last back.
    Lane<V> Af = A, Ab = A;
#pragma unroll
    for (int o = At::kLanes; o < 32; o <<= 1) {
      const Lane<V> pa = shuffle_up(Af, o), ph = shuffle_up(H, o);
      const Lane<V> na = shuffle_down(Ab, o), nr = shuffle_down(R, o);
      if (at.lane >= o) {
        H = fma(Af, ph, H);
        Af = Af * pa;
      }
      if (at.lane + o < 32) {
        R = fma(Ab, nr, R);
        Ab = Ab * na;
      }
    }
    if (at.sub == At::kSubs - 1) put(up_total[at.warp][at.cl], Af, H);
    if (at.sub == 0) put(down_total[at.warp][at.cl], Ab, R);
    __syncthreads();
    fetch(k + p.ring, slot);
    slot = slot + 1 == p.ring ? 0 : slot + 1;
    Lane<V> after = carry;
#pragma unroll
    for (int w = kWarps - 1; w >= 0; --w) {
      if (w == at.warp) after = carry;
      const Step<V> q = get<V>(down_total[w][at.cl]);
      carry = fma(q.A, carry, q.H);
    }
    {
      Lane<V> c = base;
#pragma unroll
      for (int w = 0; w < kWarps - 1; ++w) {
        const Step<V> q = get<V>(up_total[w][at.cl]);
        c = fma(q.A, c, q.H);
        if (w + 1 == at.warp) base = c;
      }
    }
    Lane<V> state = base, c = after;
    const Lane<V> ea = shuffle_up(Af, At::kLanes), eh = shuffle_up(H, At::kLanes);
    const Lane<V> na = shuffle_down(Ab, At::kLanes), nr = shuffle_down(R, At::kLanes);
    if (at.sub > 0) state = fma(ea, base, eh);
    if (at.sub < At::kSubs - 1) c = fma(na, after, nr);
    // Forward once more for h_{t-1} - x_t, then back.
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const Lane<V> before = state;
      state = fma(a[i], before, f[i] * xv[i]);
      xv[i] = fma(xv[i], all<V>(-1.0f), before);
    }
    auto write = [&](auto words) {
      T *rx = dx_row, *rg = dg_row;
      if (t0 + L <= at.len) {
#pragma unroll
        for (int i = L - 1; i >= 0; --i, rx -= p.dxt, rg -= p.dgt) {
          const Lane<V> delta = gr[i] + c;
          c = a[i] * delta;
          store_lane<words.value>(rx, f[i] * delta, mine);
          store_lane<words.value>(rg, c * xv[i] * f[i], mine);
        }
      } else {
#pragma unroll
        for (int i = L - 1; i >= 0; --i, rx -= p.dxt, rg -= p.dgt) {
          const Lane<V> delta = gr[i] + c;
          c = a[i] * delta;
          if (t0 + i < p.T) {
            const bool live = t0 + i < at.len;
            store_lane<words.value>(rx, live ? f[i] * delta : all<V>(0.0f), mine);
            store_lane<words.value>(rg, live ? c * xv[i] * f[i] : all<V>(0.0f), mine);
          }
        }
      }
    };
    if (on) {
      if (p.words) write(std::true_type{});
      else write(std::false_type{});
    }
    dx_row -= dx_stage;
    dg_row -= dg_stage;
  }
  for (int s0 = at.first + at.live * at.stage; s0 < at.end; s0 += at.stage) {
    const int t0 = s0 + at.seg * L;
    for (int i = 0; i < L; ++i)
      if (on && t0 + i < at.end) {
        store_lane<false>(dx + (t0 + i) * p.dxt, all<V>(0.0f), mine);
        store_lane<false>(dg + (t0 + i) * p.dgt, all<V>(0.0f), mine);
      }
  }
  if (p.grad_h0 != nullptr && at.piece == 0 && at.warp == 0 && at.sub == 0)
    store_state(p.grad_h0 + at.b * p.D, at.d, p.D, carry);
}

// Series of a few samples (the forward: of up to kChunk where there are channels
// enough): a thread walks a lane's channels of one series sample by
// sample, with the loads of M samples in flight.  A tile's blocks would
// have nothing to split, and spend their time beginning.  256 series of 4096
// channels bf16 in place of tiles: 4 samples 58 -> 21 us (gradient 56 -> 20; the
// host's call alone is 20), 8: 56 -> 21 (60 -> 25), 16: 58 -> 30, 32: 52 -> 49,
// 64: 98 -> 87 us (4.7 TB/s); the gradient of 16 samples 55 -> 66, so it stops at 8.
constexpr int kShort = 16;

template <typename T, bool WORDS>
__device__ __forceinline__ uint32_t load_lane(const T *row, int n) {
  if constexpr (WORDS || sizeof(T) == 4) {
    return *reinterpret_cast<const uint32_t *>(row);
  } else {
    const unsigned short *q = reinterpret_cast<const unsigned short *>(row);
    return q[0] | (n > 1 ? (uint32_t)q[1] << 16 : 0u);
  }
}

template <typename T, int M, bool WORDS>
__global__ void __launch_bounds__(256) k_scan_short(const __grid_constant__ ScanArgs p, uint32_t lanes) {
  constexpr int V = 4 / sizeof(T);
  const uint32_t per = (uint32_t)((p.D + V - 1) / V), i = blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;
  const int64_t b = i / per, d = (int64_t)(i % per) * V;
  const int n = (int)min(p.D - d, (int64_t)V), samples = (int)p.T;
  int len = samples;
  if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), len);
  const T *x = static_cast<const T *>(p.x) + b * p.xb + d, *g = static_cast<const T *>(p.gate) + b * p.gb + d;
  T *h = static_cast<T *>(p.h) + b * p.T * p.D + d;
  Lane<V> state = all<V>(0.0f);
  if (p.h0 != nullptr) state = load_state<V>(p.h0 + b * p.D, d, p.D);
  if (p.states != nullptr) store_state(p.states + b * p.D, d, p.D, state);  // (T <= kChunk)
  for (int t0 = 0; t0 < samples; t0 += M) {
    uint32_t xw[M], gw[M];
#pragma unroll
    for (int k = 0; k < M; ++k) {
      xw[k] = 0u, gw[k] = closed_gate(T{});
      if (t0 + k < len) {
        xw[k] = load_lane<T, WORDS>(x + (t0 + k) * p.xt, n);
        gw[k] = load_lane<T, WORDS>(g + (t0 + k) * p.gt, n);
      }
    }
#pragma unroll
    for (int k = 0; k < M; ++k) {
      Lane<V> a, f;
      gate_of<sizeof(T) == 4>(unpack(gw[k], T{}), a, f);
      state = fma(a, state, f * unpack(xw[k], T{}));
      if (t0 + k < samples)
        store_lane<WORDS>(h + (t0 + k) * p.D, t0 + k < len ? state : all<V>(0.0f), n);
    }
  }
  if (p.last != nullptr) store_state(p.last + b * p.D, d, p.D, state);
}

template <typename T, int M, bool WORDS>
__global__ void __launch_bounds__(256) k_scan_short_backward(const __grid_constant__ ScanArgs p, uint32_t lanes) {
  constexpr int V = 4 / sizeof(T);
  const uint32_t per = (uint32_t)((p.D + V - 1) / V), i = blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;
  const int64_t b = i / per, d = (int64_t)(i % per) * V;
  const int n = (int)min(p.D - d, (int64_t)V), samples = (int)p.T;
  int len = samples;
  if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), len);
  const T *x = static_cast<const T *>(p.x) + b * p.xb + d, *g = static_cast<const T *>(p.gate) + b * p.gb + d;
  const T *dh = static_cast<const T *>(p.grad_h) + b * p.T * p.D + d;
  T *dx = static_cast<T *>(p.grad_x) + b * p.dxb + d, *dg = static_cast<T *>(p.grad_gate) + b * p.dgb + d;
  uint32_t gw[M], dw[M];
  Lane<V> u[M];  // x, then h_{t-1} - x_t
#pragma unroll
  for (int k = 0; k < M; ++k) {
    uint32_t xw = 0u;
    gw[k] = closed_gate(T{}), dw[k] = 0u;
    if (k < len) {
      xw = load_lane<T, WORDS>(x + k * p.xt, n);
      gw[k] = load_lane<T, WORDS>(g + k * p.gt, n);
      if (p.grad_h != nullptr) dw[k] = load_lane<T, WORDS>(dh + k * p.D, n);
    }
    u[k] = unpack(xw, T{});
  }
  Lane<V> state = load_state<V>(p.states + b * p.D, d, p.D), c = all<V>(0.0f);
  if (p.grad_last != nullptr) c = load_state<V>(p.grad_last + b * p.D, d, p.D);
#pragma unroll
  for (int k = 0; k < M; ++k) {
    Lane<V> a, f;
    gate_of<sizeof(T) == 4>(unpack(gw[k], T{}), a, f);
    const Lane<V> before = state;
    state = fma(a, before, f * u[k]);
    u[k] = fma(u[k], all<V>(-1.0f), before);
  }
#pragma unroll
  for (int k = M - 1; k >= 0; --k) {
    if (k < samples) {
      Lane<V> a, f;
      gate_of<sizeof(T) == 4>(unpack(gw[k], T{}), a, f);
      const Lane<V> delta = unpack(dw[k], T{}) + c;
      c = a * delta;
      const bool live = k < len;
      store_lane<WORDS>(dx + k * p.dxt, live ? f * delta : all<V>(0.0f), n);
      store_lane<WORDS>(dg + k * p.dgt, live ? c * u[k] * f : all<V>(0.0f), n);
    }
  }
  if (p.grad_h0 != nullptr) store_state(p.grad_h0 + b * p.D, d, p.D, c);
}

template <typename T, int M, bool BACK>
cudaError_t scan_short(const ScanArgs &a, int64_t B, cudaStream_t stream) {
  constexpr int V = 4 / sizeof(T);
  const uint32_t lanes = (uint32_t)(B * ((a.D + V - 1) / V)), grid = (lanes + 255) / 256;
  if (BACK && a.words) k_scan_short_backward<T, M, true><<<grid, 256, 0, stream>>>(a, lanes);
  else if (BACK) k_scan_short_backward<T, M, false><<<grid, 256, 0, stream>>>(a, lanes);
  else if (a.words) k_scan_short<T, M, true><<<grid, 256, 0, stream>>>(a, lanes);
  else k_scan_short<T, M, false><<<grid, 256, 0, stream>>>(a, lanes);
  return cudaGetLastError();
}

// One sample of B streams whose states are rows of a table.  64x512 bf16 moves
// 0.5 MB: a launch (2 us on the device) and the host's call (7 us) bound it, so a
// thread does an element or two and the whole GPU is not needed.
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
      Lane<1> a, f;
      gate_of<sizeof(T) == 4>(all<1>(to_f32(gv.v[v])), a, f);
      const float s = fmaf(a[0], st[v], f[0] * to_f32(xv.v[v]));
      st[v] = s;
      out.v[v] = from_f32<T>(s);
    }
  }
  *reinterpret_cast<Pack<T, VEC> *>(h + b * D + d) = out;
}

// How a launch covers the series.
struct Shape {
  int lanes_log2, full_warps, threads, ring, smem;
  int64_t tiles, piece, pieces;
};

Shape shape_of(int64_t B, int64_t T, int64_t D, int vec, bool back, bool aligned) {
  const int steps = back ? kBwdSteps : kFwdSteps, tensors = back ? 3 : 2;
  Shape s;
  // Rows of 64 bytes, of 32 for 8 lanes' channels.
  s.lanes_log2 = D <= 8 * vec ? 3 : 4;
  s.tiles = (D + ((int64_t)vec << s.lanes_log2) - 1) / ((int64_t)vec << s.lanes_log2);
  auto stage_at = [&](int warps) { return (int64_t)warps * (32 >> s.lanes_log2) * steps; };
  s.full_warps = warps_of(s.lanes_log2);
  int warps = 1;
  while (warps < s.full_warps && stage_at(warps) < T) warps *= 2;
  // One piece, or as many as give four blocks (what its registers hold) to
  // each SM.  A block takes a unit of time per stage and some to begin, longer
  // on an SM that waits for it alone; composing the spans reads as much again
  // as two thirds (the gradient: two fifths) of what the main kernel moves.
  // In one piece and cut, bf16: 1x65536x512 453 and 67 us (gradient 821 and 97),
  // 2x32768x1024 232 and 130 (425 and 187), 1x4096x512 32 and 23 (54 and 22),
  // 6x8192x1024 84 and 92 (150 and 129); but 8x4096x1024 48 and 72 (85 and 105),
  // 4x8192x2048 91 and 132 (161 and 195), which stay in one.
  // Blocks of 4 and of 8 warps where an SM has two tiles at most, in one piece:
  // 8x16384x1024 177 and 157 us (gradient 316 and 304), 4x8192x2048 92 and 85 (162 and
  // 153), 8x8192x999 215 and 165 (352 and 286); but 16x2048x1024 41 and 46 (71 and 81).
  const int64_t stages = (T + stage_at(warps) - 1) / stage_at(warps), sms = device_info().sm_count;
  const int64_t tiles = B * s.tiles, spans = (T + kSpan - 1) / kSpan;
  const int64_t full = kResidentWarps / s.full_warps * sms;
  int64_t each = (spans * tiles + full - 1) / full;  // spans of a piece
  const double share = (double)(tiles * stages) / (double)sms;
  const int64_t fullest = (tiles + sms - 1) / sms;
  const bool wide = s.lanes_log2 == 4 && fullest <= 2 && T >= 2 * stage_at(kWide);
  const double whole = (double)fullest * (double)(stages + 1) * (fullest == 1 ? 1.4 : 1.0) *
                       (wide && !back ? 0.88 : 1.0);
  s.pieces = 1;
  if (spans > 1 && tiles < full && share * (back ? 1.4 : 1.67) + 8.0 < whole && each < spans) {
    s.piece = each * kSpan;
    s.pieces = (T + s.piece - 1) / s.piece;
  } else if (wide) {
    s.full_warps = warps = kWide;
  }
  s.threads = warps * 32;
  const int64_t stage = stage_at(warps);
  if (s.pieces == 1) s.piece = (T + stage - 1) / stage * stage;
  const int64_t rounds = s.piece / stage;
  const int ring = back ? 3 : 2;
  s.ring = (int)(rounds < ring ? rounds : ring);
  s.smem = (int)(s.ring * tensors * (stage + stage / steps) * ((1 << s.lanes_log2) + (aligned ? 0 : 4)) * 4);
  return s;
}

template <typename T, int LOG2, int WARPS, bool BACK, bool ALIGNED>
cudaError_t scan_launch(const ScanArgs &a, const Shape &s, int64_t B, cudaStream_t stream) {
  const auto kernel = BACK ? k_scan_backward<T, LOG2, WARPS, ALIGNED> : k_scan<T, LOG2, WARPS, ALIGNED>;
  cudaError_t e = cudaSuccess;
  if (s.smem > 40 * 1024) {  // (8 KB beside it are the kernel's own)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, s.smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t c{};
  cudaLaunchAttribute attr{};
  if (s.pieces > 1) {  // begins, and fetches its first stages, while the pieces are composed
    const int64_t vec = 4 / sizeof(T), tiles = (a.D + 32 * vec - 1) / (32 * vec);
    k_scan_totals<T, BACK><<<(unsigned)(B * spans_needed<BACK>(a) * tiles), kTotalWarps * 32, 0, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr, c.numAttrs = 1;
  }
  c.gridDim = dim3((unsigned)(B * s.pieces * s.tiles)), c.blockDim = dim3(s.threads);
  c.dynamicSmemBytes = s.smem, c.stream = stream;
  return cudaLaunchKernelEx(&c, kernel, a);
}

template <typename T, bool BACK, bool ALIGNED>
cudaError_t scan_shape(const ScanArgs &a, const Shape &s, int64_t B, cudaStream_t stream) {
  if (s.lanes_log2 == 3) return scan_launch<T, 3, warps_of(3), BACK, ALIGNED>(a, s, B, stream);
  if (s.full_warps == kWide) return scan_launch<T, 4, kWide, BACK, ALIGNED>(a, s, B, stream);
  return scan_launch<T, 4, warps_of(4), BACK, ALIGNED>(a, s, B, stream);
}

template <typename T, bool BACK>
cudaError_t scan_as(ScanArgs a, int64_t B, cudaStream_t stream) {
  constexpr int V = 4 / sizeof(T);
  if (a.T <= 4) return scan_short<T, 4, BACK>(a, B, stream);
  if (a.T <= 8) return scan_short<T, 8, BACK>(a, B, stream);
  // 1024 lanes on each SM keep the forward's loads coming.
  if (!BACK && (a.T <= kShort || (a.T <= kChunk && B * a.D / V >= 1024 * (int64_t)device_info().sm_count)))
    return scan_short<T, kShort, false>(a, B, stream);
  const Shape s = shape_of(B, a.T, a.D, V, BACK, a.aligned);
  a.tiles = s.tiles, a.piece = s.piece, a.pieces = (int)s.pieces, a.ring = s.ring;
  return a.aligned ? scan_shape<T, BACK, true>(a, s, B, stream) : scan_shape<T, BACK, false>(a, s, B, stream);
}

// Fills in what the kernels need to know of the inputs' and outputs' places.
void set_places(ScanArgs &a, int64_t B, int e) {
  auto rows_on = [&](int w) {
    return a.D * e % w == 0 && aligned_to(a.x, a.xb, e, w) && aligned_to(a.x, a.xt, e, w) &&
           aligned_to(a.gate, a.gb, e, w) && aligned_to(a.gate, a.gt, e, w) && aligned_to(a.grad_h, 0, e, w);
  };
  a.aligned = rows_on(16);
  a.words = rows_on(4) && aligned_to(a.h, 0, e, 4) && aligned_to(a.grad_x, a.dxb, e, 4) &&
            aligned_to(a.grad_x, a.dxt, e, 4) && aligned_to(a.grad_gate, a.dgb, e, 4) &&
            aligned_to(a.grad_gate, a.dgt, e, 4);
  a.x_end = ((B - 1) * a.xb + (a.T - 1) * a.xt + a.D) * e;
  a.gate_end = ((B - 1) * a.gb + (a.T - 1) * a.gt + a.D) * e;
  a.grad_h_end = B * a.T * a.D * e;
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
int check_scan(const char *fn, int dtype, const void *x, int64_t x_series, int64_t x_sample,
               const void *gate, int64_t gate_series, int64_t gate_sample, int64_t B, int64_t T, int64_t D) {
  if (!dtype_ok(dtype)) return report_error(CPAB_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
  if (B < 0 || T < 0 || D < 0) return report_error(CPAB_ERR_ARG, "%s: negative size", fn);
  if (x_series < 0 || x_sample < 0 || gate_series < 0 || gate_sample < 0)
    return report_error(CPAB_ERR_ARG, "%s: negative stride", fn);
  if (T > (int64_t(1) << 31) - 4096) return report_error(CPAB_ERR_SIZE, "%s: T must not exceed 2^31 - 4096", fn);
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

extern "C" int64_t cpab_b200_gated_scan_workspace(int dtype, int64_t B, int64_t T, int64_t D) {
  if (!dtype_ok(dtype) || B < 1 || T < 1 || D < 1 || T > (int64_t(1) << 31) - 4096 || B > (int64_t(1) << 30) / D)
    return 0;
  const int vec = 4 / dtype_size(dtype);
  const bool cut = shape_of(B, T, D, vec, false, true).pieces > 1 || shape_of(B, T, D, vec, true, true).pieces > 1;
  return cut ? 2 * B * D * ((T + kSpan - 1) / kSpan) : 2;
}

extern "C" int cpab_b200_gated_scan(int dtype, const void *x, int64_t x_series, int64_t x_sample,
                                    const void *gate, int64_t gate_series, int64_t gate_sample,
                                    int64_t B, int64_t T, int64_t D, const int32_t *lengths,
                                    const float *h0, void *h, float *h_last, float *states,
                                    float *workspace, cpab_stream_t stream) {
  const int st = check_scan("gated_scan", dtype, x, x_series, x_sample, gate, gate_series, gate_sample, B, T, D);
  if (st != CPAB_OK) return st;
  if (B == 0 || D == 0) return launch_status(cudaSuccess, "");
  if (T == 0) {  // no samples: the state is what it was
    if (h_last == nullptr) return launch_status(cudaSuccess, "");
    const size_t bytes = (size_t)B * D * sizeof(float);
    return launch_status(h0 != nullptr ? cudaMemcpyAsync(h_last, h0, bytes, cudaMemcpyDeviceToDevice, stream)
                                       : cudaMemsetAsync(h_last, 0, bytes, stream), "gated_scan");
  }
  if (h == nullptr) return report_error(CPAB_ERR_ARG, "gated_scan: null output pointer");
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
    return report_error(CPAB_ERR_ARG, "gated_scan: null or misaligned workspace");
  ScanArgs a{};
  a.x = x, a.gate = gate, a.xb = x_series, a.xt = x_sample, a.gb = gate_series, a.gt = gate_sample;
  a.T = T, a.D = D, a.lengths = lengths, a.h0 = h0, a.h = h, a.last = h_last, a.states = states;
  a.totals = reinterpret_cast<float2 *>(workspace);
  set_places(a, B, dtype_size(dtype));
  const cudaError_t err = dtype == CPAB_F32   ? scan_as<float, false>(a, B, stream)
                          : dtype == CPAB_F16 ? scan_as<__half, false>(a, B, stream)
                                              : scan_as<__nv_bfloat16, false>(a, B, stream);
  return launch_status(err, "gated_scan");
}

extern "C" int cpab_b200_gated_scan_backward(
    int dtype, const void *x, int64_t x_series, int64_t x_sample, const void *gate,
    int64_t gate_series, int64_t gate_sample, int64_t B, int64_t T, int64_t D,
    const int32_t *lengths, const float *states, const void *grad_h, const float *grad_last,
    void *grad_x, int64_t grad_x_series, int64_t grad_x_sample, void *grad_gate,
    int64_t grad_gate_series, int64_t grad_gate_sample, float *grad_h0, float *workspace,
    cpab_stream_t stream) {
  const int st = check_scan("gated_scan_backward", dtype, x, x_series, x_sample, gate, gate_series, gate_sample, B, T,
                            D);
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
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 8 != 0)
    return report_error(CPAB_ERR_ARG, "gated_scan_backward: null or misaligned workspace");
  ScanArgs a{};
  a.x = x, a.gate = gate, a.xb = x_series, a.xt = x_sample, a.gb = gate_series, a.gt = gate_sample;
  a.T = T, a.D = D, a.lengths = lengths, a.states = const_cast<float *>(states);
  a.grad_h = grad_h, a.grad_last = grad_last, a.grad_x = grad_x, a.grad_gate = grad_gate;
  a.dxb = grad_x_series, a.dxt = grad_x_sample, a.dgb = grad_gate_series, a.dgt = grad_gate_sample;
  a.grad_h0 = grad_h0, a.totals = reinterpret_cast<float2 *>(workspace);
  set_places(a, B, dtype_size(dtype));
  const cudaError_t err = dtype == CPAB_F32   ? scan_as<float, true>(a, B, stream)
                          : dtype == CPAB_F16 ? scan_as<__half, true>(a, B, stream)
                                              : scan_as<__nv_bfloat16, true>(a, B, stream);
  return launch_status(err, "gated_scan_backward");
}

extern "C" int cpab_b200_gated_scan_step(int dtype, const void *x, int64_t x_row, const void *gate,
                                         int64_t gate_row, int64_t B, int64_t D,
                                         const int32_t *slots, int64_t rows, float *state, void *h,
                                         cpab_stream_t stream) {
  const int st = check_scan("gated_scan_step", dtype, x, x_row, 0, gate, gate_row, 0, B, 1, D);
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
