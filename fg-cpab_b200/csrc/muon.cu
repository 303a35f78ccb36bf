// Orthogonalised directions: Newton-Schulz products of whole lists of matrices,
// and the optimizer step made of them.
//
//   X = G / (|G|_F + eps)                      (m x n, transposed so that m <= n)
//   steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// which moves every singular value of X towards 1 and leaves the singular vectors.
// The products run on the tensor cores in halves with float32 sums; A and B are
// symmetric, so only tiles on and above the diagonal are computed and each is
// stored twice.  A matrix is kept as 2^10 times its values in two halves, a value
// rounded to a half and its remainder (22 bits together):
//
//   - parameters and matrices of 16 bits, of more than 256 rows, are multiplied by
//     their first halves (11 bits, 2^-12 off); the remainder enters the terms a X and b A, which would
//     otherwise drown small singular values beside large ones.  The result is
//     1.5e-3 to 2.7e-3 off (relative 2-norm, normal matrices of up to 1500 rows),
//     about a rounding to bfloat16 (1.7e-3).
//   - float32 ones and small ones take three products, first x first + first x remainder +
//     remainder x first (4e-7 to 3e-6 off): a float32 parameter keeps that many
//     bits of its update.
//
// 2^10 keeps values from 6e-8 in a half's normal range and leaves room to 64.  Where
// eps is not small beside |G|_F, X is: it is kept as theta Y with theta a power of two
// and |Y|_F in (1/2, 1], and the steps are taken in Y with
//   Y <- r (a + theta^2 b Y Y^T + theta^4 c (Y Y^T)^2) Y,   r = theta / theta',
// theta' = min(1, 2^ceil(log2 a) theta), until theta is 1.
#include <algorithm>
#include <cmath>
#include <vector>

#include "product_core.cuh"
#include "sequence.cuh"

namespace cpab {
namespace {

constexpr float kUnit = 1024.f;       // stored = value * kUnit
constexpr int kPartials = 256;        // partial sums of squares of a matrix
constexpr int kGroups = 8;            // shapes in a launch
constexpr int kPrepared = 64;         // matrices in a launch that reads them
// Matrices of so few rows take pairs of halves whatever their type: their launches are
// bound by latency, and a few singular values do not average the errors of halves (a
// single one was 5e-3 off).
constexpr int kFewRows = 256;
constexpr int kMatrices = 128;        // parameters in a sequence of launches

__device__ __forceinline__ float read_as(const void *p, int dtype, int64_t i) {
  if (dtype == CPAB_F32) return static_cast<const float *>(p)[i];
  if (dtype == CPAB_F16) return to_f32(static_cast<const __half *>(p)[i]);
  return to_f32(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void write_as(void *p, int dtype, int64_t i, float v) {
  if (dtype == CPAB_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == CPAB_F16) static_cast<__half *>(p)[i] = from_f32<__half>(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = from_f32<__nv_bfloat16>(v);
}

// ---- what goes in ----------------------------------------------------------------

struct Prepared {
  const void *grad;   // [rows, cols] of dtype, contiguous
  float *momentum;    // float32, updated; null: the matrix itself is taken
  __half *hi, *lo;    // [m, pitch]
  double *partials;   // [kPartials]
  float *terms;       // [kTerms]
  int64_t pitch;
  int rows, cols;
  int dtype;
  int turned;         // hi and lo are [cols, rows]
};
struct PrepareArgs {
  Prepared m[kPrepared];
  float momentum;
  int nesterov, steps;
  double eps, a, b, c;
};

// Each step's coefficients for Y, three floats, and the last theta behind them.
constexpr int kMostSteps = 64;
constexpr int kTerms = 3 * kMostSteps + 1;

__device__ __forceinline__ double first_theta(double norm, double eps) {
  const double x = norm / (norm + eps);
  if (!(x > 0.0) || x >= 0.5) return 1.0;  // (of zeros, and of NaN, 1)
  return exp2(ceil(log2(x)));
}
__device__ __forceinline__ void write_terms(float *to, double theta, double a, double b, double c, int steps) {
  const double growth = exp2(ceil(log2(fmax(1.0, fabs(a)))));
  for (int k = 0; k < steps; ++k) {
    const double next = fmin(1.0, growth * theta), r = theta / next, q = theta * theta;
    to[3 * k] = (float)(a * r), to[3 * k + 1] = (float)(b * q * r), to[3 * k + 2] = (float)(c * q * q * r);
    theta = next;
  }
  to[3 * kMostSteps] = (float)theta;
}

// The direction: m = momentum m + (1 - momentum) g, and with nesterov
// (1 - momentum) g + momentum m of the new m.
__device__ __forceinline__ float direction(const Prepared &p, const PrepareArgs &a, int64_t i, float m) {
  return a.nesterov ? (1.f - a.momentum) * read_as(p.grad, p.dtype, i) + a.momentum * m : m;
}

// Momenta, and partial sums of the directions' squares (in float64: a square may
// leave float32's range where its element does not).
__global__ void __launch_bounds__(256) k_direction(const __grid_constant__ PrepareArgs a) {
  const Prepared &p = a.m[blockIdx.y];
  tc::dep_launch();
  tc::dep_wait();
  const int64_t n = (int64_t)p.rows * p.cols;
  double sum = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float u;
    if (p.momentum != nullptr) {
      const float m = a.momentum * p.momentum[i] + (1.f - a.momentum) * read_as(p.grad, p.dtype, i);
      p.momentum[i] = m;
      u = direction(p, a, i, m);
    } else {
      u = read_as(p.grad, p.dtype, i);
    }
    sum += (double)u * (double)u;
  }
  __shared__ double part[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int i = 0; i < 8; ++i) sum += part[i];
    p.partials[blockIdx.x] = sum;
  }
}

__device__ __forceinline__ void store_halves(__half *hi, __half *lo, int64_t i, float v) {
  const __half h = __float2half_rn(v);
  hi[i] = h;
  lo[i] = __float2half_rn(v - __half2float(h));
}

// Directions over their norms, as halves; tiles of 64 x 64.
__global__ void __launch_bounds__(256) k_normalise(const __grid_constant__ PrepareArgs a, int partials) {
  const Prepared &p = a.m[blockIdx.y];
  const int tiles_x = (p.cols + 63) / 64, tiles = tiles_x * ((p.rows + 63) / 64);
  tc::dep_launch();
  tc::dep_wait();
  if ((int)blockIdx.x >= tiles) return;
  __shared__ double part[8];
  __shared__ float tile[64][65];
  double sum = 0;
  for (int i = threadIdx.x; i < partials; i += 256) sum += p.partials[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < 8; ++i) sum += part[i];
  const double norm = sqrt(sum), theta = first_theta(norm, a.eps), scale = (double)kUnit / ((norm + a.eps) * theta);
  if (blockIdx.x == 0 && threadIdx.x == 0) write_terms(p.terms, theta, a.a, a.b, a.c, a.steps);
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int r0 = t / tiles_x * 64, c0 = t % tiles_x * 64, x = threadIdx.x & 63;
    for (int y = threadIdx.x >> 6; y < 64; y += 4) {
      if (r0 + y >= p.rows || c0 + x >= p.cols) continue;
      const int64_t i = (int64_t)(r0 + y) * p.cols + c0 + x;
      const float u = p.momentum != nullptr ? direction(p, a, i, p.momentum[i]) : read_as(p.grad, p.dtype, i);
      const float v = (float)((double)u * scale);
      if (p.turned) tile[y][x] = v;
      else store_halves(p.hi, p.lo, (int64_t)(r0 + y) * p.pitch + c0 + x, v);
    }
    if (!p.turned) continue;
    __syncthreads();
    for (int y = threadIdx.x >> 6; y < 64; y += 4)
      if (c0 + y < p.cols && r0 + x < p.rows)
        store_halves(p.hi, p.lo, (int64_t)(c0 + y) * p.pitch + r0 + x, tile[x][y]);
    __syncthreads();
  }
}

// ---- the products ------------------------------------------------------------------

enum Phase { kGram, kSquare, kUpdate, kFinal };

struct PhaseGroup {
  CUtensorMap a[2], b[2];          // first halves and remainders of the operands
  const __half *read[2];           // A (kSquare) or X (kUpdate, kFinal)
  __half *write[2];                // A, B or the next X
  int64_t read_pitch, read_plane, write_pitch, write_plane;
  int m, n;                        // of the result
  int steps;                       // stages of 64 summed
  int tiles_m, tiles_n, end;       // tiles of one matrix; end of the group's in the launch
  int write_lo;
  const float *terms;              // of the set's first matrix, kTerms apart
};
struct FinalGroup {
  void *out;                       // of matrix z: out + z * stride elements, or table[first + z]
  int64_t stride;
  int first;                       // -1: out and stride
  int dtype, turned, update;       // turned: stored transposed; update: a parameter's step
  int wide;                        // all rows begin on 32 bytes
  float decay, rate;               // p (1 - lr decay) - lr rate O
  const float *lr_device;
  float lr;
};
template <bool FINAL>
struct PhaseArgs {
  PhaseGroup g[kGroups];
  int groups, step;
};
template <>
struct PhaseArgs<true> {
  PhaseGroup g[kGroups];
  FinalGroup f[kGroups];
  void *table[kMatrices];
  int groups, step;
};

template <int PHASE, int PARTS, int CTAS, int BN>
struct Schulz {
  static constexpr int kCtas = CTAS, kBN = BN, kAcc = 2, kParts = PARTS, kChunk = 16;
  // (16-bit results: up to 1.5e-5 of the sum at 4096 summed, against 2^-12 of its operands)
  static constexpr int kSegment = PARTS == 2 ? 4 : 0;
  static constexpr bool kScaled = false, kBMn = PHASE >= kUpdate, kSymmetric = PHASE <= kSquare;
  static constexpr int kBM = 128 * CTAS;
  static_assert(kBM == BN, "symmetric results are computed by square tiles");
  struct alignas(16) Shared {
    int unused;
  };
  struct Tile {
    int m0, n0, steps, z, g;
    bool mirror;
  };
  const PhaseArgs<PHASE == kFinal> &p;

  __device__ int tiles() const { return p.g[p.groups - 1].end; }
  __device__ Tile tile(int i) const {
    int g = 0, begin = 0;
    while (i >= p.g[g].end) begin = p.g[g++].end;
    const PhaseGroup &q = p.g[g];
    i -= begin;
    Tile t;
    t.g = g, t.steps = q.steps;
    if (kSymmetric) {
      const int per = q.tiles_m * (q.tiles_m + 1) / 2;
      t.z = i / per, i %= per;
      int column = (int)((sqrtf(8.f * (float)i + 1.f) - 1.f) * 0.5f);
      while (column * (column + 1) / 2 > i) --column;
      while ((column + 1) * (column + 2) / 2 <= i) ++column;
      const int row = i - column * (column + 1) / 2;
      t.m0 = row * kBM, t.n0 = column * BN, t.mirror = row != column;
    } else {
      const int per = q.tiles_m * q.tiles_n;
      t.z = i / per, i %= per;
      t.m0 = i % q.tiles_m * kBM, t.n0 = i / q.tiles_m * BN, t.mirror = false;
    }
    return t;
  }
  __device__ void load(const Tile &t, int k, uint32_t sa, uint32_t sb, uint32_t bar, uint32_t rank) const {
    const PhaseGroup &q = p.g[t.g];
    const int at = k * 64, n = t.n0 + rank * (BN / CTAS);
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      tc::tile_load<CTAS>(sa + h * tc::kAHalf, &q.a[h], bar, at, t.m0 + rank * 128, t.z);
      const uint32_t to = sb + h * (BN / CTAS * 128);
      if constexpr (kBMn) {  // 64 summed rows of 64 columns, twice
        tc::tile_load<CTAS>(to, &q.b[h], bar, n, at, t.z);
        tc::tile_load<CTAS>(to + 8192, &q.b[h], bar, n + 64, at, t.z);
      } else {
        tc::tile_load<CTAS>(to, &q.b[h], bar, at, n, t.z);
      }
    }
  }
  __device__ void begin(const Tile &, Shared &, int) const {}

  __device__ void store(const Tile &t, const Shared &, int row, int c, const float *acc) const {
    const PhaseGroup &q = p.g[t.g];
    const int col = t.n0 + c;
    if (row >= q.m || col >= q.n) return;
    const bool whole = col + 16 <= q.n;
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = acc[j] * (1.f / kUnit);
    if constexpr (PHASE != kGram) {
      const float *terms = q.terms + t.z * kTerms + 3 * p.step;
      const float mine = terms[PHASE == kSquare ? 1 : 0], product = PHASE == kSquare ? terms[2] : 1.f;
      const int64_t at = t.z * q.read_plane + row * q.read_pitch + col;
      const __half *hi = q.read[0] + at, *lo = q.read[1] + at;
      if (whole) {
        uint32_t h[8], l[8];
        tc::load_sector(hi, h);
        tc::load_sector(lo, l);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 x = unpack_pair<__half>(h[j]), y = unpack_pair<__half>(l[j]);
          v[2 * j] = mine * (x.x + y.x) + product * v[2 * j];
          v[2 * j + 1] = mine * (x.y + y.y) + product * v[2 * j + 1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (col + j < q.n) v[j] = mine * (__half2float(hi[j]) + __half2float(lo[j])) + product * v[j];
      }
    }
    if constexpr (PHASE == kFinal) {
      finish(t, q, row, col, v);
      return;
    }
    __half *hi = q.write[0] + t.z * q.write_plane, *lo = q.write[1] + t.z * q.write_plane;
    const int64_t at = row * q.write_pitch + col;
    uint32_t h[8], l[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[j] = pack_pair<__half>(v[2 * j], v[2 * j + 1]);
      const float2 x = unpack_pair<__half>(h[j]);
      l[j] = pack_pair<__half>(v[2 * j] - x.x, v[2 * j + 1] - x.y);
    }
    if (whole) {
      tc::store_sector(hi + at, h);
      if (q.write_lo) tc::store_sector(lo + at, l);
    }
    if (!whole || t.mirror) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (col + j < q.n) {
          const uint16_t x = (uint16_t)(h[j >> 1] >> (16 * (j & 1))), y = (uint16_t)(l[j >> 1] >> (16 * (j & 1)));
          const __half xh = __ushort_as_half(x), yh = __ushort_as_half(y);
          if (!whole) {
            hi[at + j] = xh;
            if (q.write_lo) lo[at + j] = yh;
          }
          if (t.mirror) {
            const int64_t to = (int64_t)(col + j) * q.write_pitch + row;
            hi[to] = xh;
            if (q.write_lo) lo[to] = yh;
          }
        }
    }
  }

  // The last step's values: the result, or a parameter's step.
  __device__ void finish(const Tile &t, const PhaseGroup &q, int row, int col, float (&v)[16]) const {
    if constexpr (PHASE == kFinal) {
      const FinalGroup &f = p.f[t.g];
      const int e = f.dtype == CPAB_F32 ? 4 : 2;
      void *out = f.first >= 0 ? p.table[f.first + t.z] : static_cast<char *>(f.out) + t.z * f.stride * e;
      const float lr = f.lr_device != nullptr ? *f.lr_device : f.lr;
      const float last = q.terms[t.z * kTerms + 3 * kMostSteps] * (1.f / kUnit);
      const float keep = f.update ? 1.f - lr * f.decay : 0.f, move = (f.update ? -lr * f.rate : 1.f) * last;
      if (f.wide && col + 16 <= q.n) {
        const int64_t i = (int64_t)row * q.n + col;
        if (f.dtype == CPAB_F32) whole<float>(static_cast<float *>(out) + i, f.update, keep, move, v);
        else if (f.dtype == CPAB_F16) whole<__half>(static_cast<__half *>(out) + i, f.update, keep, move, v);
        else whole<__nv_bfloat16>(static_cast<__nv_bfloat16 *>(out) + i, f.update, keep, move, v);
        return;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (col + j >= q.n) break;
        const int64_t i = f.turned ? (int64_t)(col + j) * q.m + row : (int64_t)row * q.n + col + j;
        const float o = move * v[j];
        write_as(out, f.dtype, i, f.update ? fmaf(keep, read_as(out, f.dtype, i), o) : o);
      }
    }
  }
  // 16 values of a row that begins on 32 bytes.
  template <typename T>
  static __device__ void whole(T *out, int update, float keep, float move, const float (&v)[16]) {
    uint32_t w[8];
    if constexpr (sizeof(T) == 2) {
      if (update) tc::load_sector(out, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 x = update ? unpack_pair<T>(w[j]) : make_float2(0.f, 0.f);
        const float a = move * v[2 * j], b = move * v[2 * j + 1];
        w[j] = update ? pack_pair<T>(fmaf(keep, x.x, a), fmaf(keep, x.y, b)) : pack_pair<T>(a, b);
      }
      tc::store_sector(out, w);
    } else {
#pragma unroll
      for (int h = 0; h < 16; h += 8) {
        if (update) tc::load_sector(out + h, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float o = move * v[h + j];
          w[j] = __float_as_uint(update ? fmaf(keep, __uint_as_float(w[j]), o) : o);
        }
        tc::store_sector(out + h, w);
      }
    }
  }
};

template <int PHASE, int PARTS, int CTAS, int BN>
__global__ void __launch_bounds__(tc::kCoreThreads, 1)
    k_schulz(const __grid_constant__ PhaseArgs<PHASE == kFinal> a) {
  tc::core(Schulz<PHASE, PARTS, CTAS, BN>{a});
}

template <int PHASE, int PARTS, int CTAS, int BN>
cudaError_t launch_phase_as(PhaseArgs<PHASE == kFinal> &a, const int *batch, cudaStream_t s) {
  using S = tc::CoreShape<Schulz<PHASE, PARTS, CTAS, BN>>;
  auto *kernel = k_schulz<PHASE, PARTS, CTAS, BN>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (e != cudaSuccess) return e;
  int64_t tiles = 0;
  for (int g = 0; g < a.groups; ++g) {
    PhaseGroup &q = a.g[g];
    q.tiles_m = (q.m + BN - 1) / BN, q.tiles_n = (q.n + BN - 1) / BN;
    const int64_t per = PHASE <= kSquare ? (int64_t)q.tiles_m * (q.tiles_m + 1) / 2 : (int64_t)q.tiles_m * q.tiles_n;
    tiles += per * batch[g];
    if (tiles >= int64_t(1) << 30) return cudaErrorInvalidValue;
    q.end = (int)tiles;
  }
  return tc::launch(kernel, (unsigned)(CTAS * std::min<int64_t>(tiles, device_info().sm_count / CTAS)), tc::kCoreThreads,
                    S::kBytes, CTAS, s, a);
}

// ---- a sequence of launches ---------------------------------------------------------

// A set of `batch` matrices of one shape and type.
struct Set {
  int rows, cols, dtype, batch;
  int m() const { return std::min(rows, cols); }
  int n() const { return std::max(rows, cols); }
  bool turned() const { return rows > cols; }
  int parts() const { return dtype == CPAB_F32 || m() <= kFewRows ? 2 : 1; }
  // (rows begin on 32 bytes: whole sectors are moved)
  int64_t x_pitch() const { return (n() + 15) / 16 * 16; }
  int64_t a_pitch() const { return (m() + 15) / 16 * 16; }
  int64_t x_halves() const { return (int64_t)batch * m() * x_pitch(); }
  int64_t a_halves() const { return (int64_t)batch * m() * a_pitch(); }
};
int64_t round_up(int64_t n) { return (n + 255) / 256 * 256; }

struct Places {
  __half *x[2][2], *a[2], *b[2];  // [buffer][half]
  float *terms;
};
// Bytes of the sets' workspace; with `base`, the places too.
int64_t place(const std::vector<Set> &sets, int64_t matrices, char *base, std::vector<Places> *places, double **partials) {
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char *p = base + at;
    at += round_up(bytes);
    return p;
  };
  if (places != nullptr) places->resize(sets.size());
  char *d = take(matrices * kPartials * (int64_t)sizeof(double));
  if (partials != nullptr) *partials = reinterpret_cast<double *>(d);
  for (size_t i = 0; i < sets.size(); ++i) {
    const Set &s = sets[i];
    float *terms = reinterpret_cast<float *>(take((int64_t)s.batch * kTerms * (int64_t)sizeof(float)));
    if (places != nullptr) (*places)[i].terms = terms;
    for (int k = 0; k < 8; ++k) {
      __half *p = reinterpret_cast<__half *>(take(2 * (k < 4 ? s.x_halves() : s.a_halves())));
      if (places == nullptr) continue;
      Places &q = (*places)[i];
      if (k < 4) q.x[k >> 1][k & 1] = p;
      else if (k < 6) q.a[k & 1] = p;
      else q.b[k & 1] = p;
    }
  }
  return at;
}

bool map_of(CUtensorMap *map, const __half *p, int columns, int rows, int batch, int64_t pitch, int box_rows) {
  return make_tile_map(map, true, p, columns, rows, batch, pitch * 2, pitch * 2 * rows, box_rows);
}

template <int PHASE, int PARTS>
cudaError_t launch_phase(PhaseArgs<PHASE == kFinal> &a, const int *batch, cudaStream_t s) {
  int64_t tiles = 0;
  for (int g = 0; g < a.groups; ++g) {
    const int64_t tm = (a.g[g].m + 255) / 256, tn = (a.g[g].n + 255) / 256;
    tiles += (PHASE <= kSquare ? tm * (tm + 1) / 2 : tm * tn) * batch[g];
  }
  return tiles * 2 >= device_info().sm_count / 2 ? launch_phase_as<PHASE, PARTS, 2, 256>(a, batch, s)
                                                 : launch_phase_as<PHASE, PARTS, 1, 128>(a, batch, s);
}

// The products of at most kGroups sets, all of one kind.
template <int PARTS>
cudaError_t schulz_as(const std::vector<Set> &sets, const std::vector<Places> &places, const FinalGroup *finals,
                      void *const *table, int table_size, int steps, cudaStream_t s) {
  int batch[kGroups];
  PhaseArgs<false> a;
  PhaseArgs<true> last;
  const int groups = (int)sets.size();
  a.groups = last.groups = groups;
  for (int i = 0; i < table_size; ++i) last.table[i] = table[i];
  for (int g = 0; g < groups; ++g) last.f[g] = finals[g], batch[g] = sets[g].batch;
  for (int step = 0; step < steps; ++step) {
    const int now = step & 1;
    a.step = last.step = step;
    bool ok = true;
    cudaError_t e;
    for (int g = 0; g < groups; ++g) {
      const Set &t = sets[g];
      const Places &w = places[g];
      PhaseGroup &q = a.g[g];
      for (int h = 0; h < 2; ++h) {
        ok = ok && map_of(&q.a[h], w.x[now][h], t.n(), t.m(), t.batch, t.x_pitch(), 128);
        q.b[h] = q.a[h];
        q.read[h] = nullptr, q.write[h] = w.a[h];
      }
      q.terms = w.terms;
      q.write_pitch = t.a_pitch(), q.write_plane = t.m() * t.a_pitch();
      q.m = q.n = t.m(), q.steps = (t.n() + 63) / 64, q.write_lo = 1;
    }
    if (!ok) return cudaErrorInvalidValue;
    if ((e = launch_phase<kGram, PARTS>(a, batch, s)) != cudaSuccess) return e;
    for (int g = 0; g < groups; ++g) {
      const Set &t = sets[g];
      const Places &w = places[g];
      PhaseGroup &q = a.g[g];
      for (int h = 0; h < 2; ++h) {
        ok = ok && map_of(&q.a[h], w.a[h], t.m(), t.m(), t.batch, t.a_pitch(), 128);
        q.b[h] = q.a[h];
        q.read[h] = w.a[h], q.write[h] = w.b[h];
      }
      q.read_pitch = t.a_pitch(), q.read_plane = t.m() * t.a_pitch();
      q.steps = (t.m() + 63) / 64, q.write_lo = PARTS == 2;
    }
    if (!ok) return cudaErrorInvalidValue;
    if ((e = launch_phase<kSquare, PARTS>(a, batch, s)) != cudaSuccess) return e;
    for (int g = 0; g < groups; ++g) {
      const Set &t = sets[g];
      const Places &w = places[g];
      PhaseGroup &q = a.g[g];
      for (int h = 0; h < 2; ++h) {
        ok = ok && map_of(&q.a[h], w.b[h], t.m(), t.m(), t.batch, t.a_pitch(), 128);
        ok = ok && map_of(&q.b[h], w.x[now][h], t.n(), t.m(), t.batch, t.x_pitch(), 64);
        q.read[h] = w.x[now][h], q.write[h] = w.x[now ^ 1][h];
      }
      q.read_pitch = q.write_pitch = t.x_pitch(), q.read_plane = q.write_plane = t.m() * t.x_pitch();
      q.n = t.n(), q.write_lo = 1;
    }
    if (!ok) return cudaErrorInvalidValue;
    if (step + 1 < steps) {
      e = launch_phase<kUpdate, PARTS>(a, batch, s);
    } else {
      for (int g = 0; g < groups; ++g) last.g[g] = a.g[g];
      e = launch_phase<kFinal, PARTS>(last, batch, s);
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t schulz(const std::vector<Set> &sets, const std::vector<Places> &places, const FinalGroup *finals,
                   void *const *table, int table_size, int steps, cudaStream_t s) {
  return sets[0].parts() == 2 ? schulz_as<2>(sets, places, finals, table, table_size, steps, s)
                              : schulz_as<1>(sets, places, finals, table, table_size, steps, s);
}

// Launches what reads the matrices in.
cudaError_t prepare(const std::vector<Prepared> &list, float momentum, int nesterov, int steps, const double *c,
                    double eps, cudaStream_t s) {
  for (size_t first = 0; first < list.size(); first += kPrepared) {
    const int n = (int)std::min<size_t>(kPrepared, list.size() - first);
    PrepareArgs a;
    int64_t most = 0, tiles = 0;
    for (int i = 0; i < n; ++i) {
      a.m[i] = list[first + i];
      most = std::max(most, (int64_t)a.m[i].rows * a.m[i].cols);
      tiles = std::max(tiles, (int64_t)((a.m[i].rows + 63) / 64) * ((a.m[i].cols + 63) / 64));
    }
    a.momentum = momentum, a.nesterov = nesterov, a.steps = steps, a.eps = eps, a.a = c[0], a.b = c[1], a.c = c[2];
    const int partials = (int)std::min<int64_t>(kPartials, (most + 2047) / 2048);
    cudaError_t e = tc::launch(k_direction, dim3(partials, n), 256, 0, 1, s, a);
    if (e == cudaSuccess)
      e = tc::launch(k_normalise, dim3((unsigned)std::min<int64_t>(tiles, 65535), n), 256, 0, 1, s, a, partials);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

constexpr int64_t kMostRows = 1 << 20;

const char *check_steps(int steps, const double *c, double eps) {
  if (steps < 1 || steps > kMostSteps) return "steps must be 1 to 64";
  if (!(eps >= 0)) return "eps must not be negative";
  // Where the singular values of X can be after each step, and the magnitudes of what is stored.
  double most = 1;
  for (int k = 0; k < steps; ++k) {
    double next = 0;
    for (int i = 0; i <= 1000; ++i) {
      const double x = most * i / 1000, q = x * x, b = c[1] * q + c[2] * q * q;
      const double value = std::fabs(c[0] * x + b * x);
      if (!(std::fabs(c[0]) < 60) || !(std::fabs(b) < 60) || !(q < 60) || !(value < 60))
        return "coefficients let values outgrow their range of 60";
      next = std::max(next, value);
    }
    most = next;
  }
  return nullptr;
}

}  // namespace
}  // namespace cpab

using namespace cpab;

extern "C" int64_t cpab_b200_orthogonalize_workspace(int dtype, int64_t batch, int64_t rows, int64_t columns) {
  if (!dtype_ok(dtype) || batch < 1 || rows < 1 || columns < 1 || batch > 65536 || rows > kMostRows || columns > kMostRows)
    return 0;
  return place({{(int)rows, (int)columns, dtype, (int)batch}}, batch, nullptr, nullptr, nullptr);
}

extern "C" int cpab_b200_orthogonalize(int dtype, const void *x, int64_t batch, int64_t rows, int64_t columns,
                                       int steps, const double *coefficients, double eps, void *out, void *workspace,
                                       cpab_stream_t stream) {
  if (!dtype_ok(dtype)) return report_error(CPAB_ERR_ARG, "%s", "orthogonalize: unknown element type");
  if (batch < 0 || rows < 0 || columns < 0 || coefficients == nullptr)
    return report_error(CPAB_ERR_ARG, "%s", "orthogonalize: negative size or null coefficients");
  const char *why = check_steps(steps, coefficients, eps);
  if (why != nullptr) return report_error(CPAB_ERR_ARG, "orthogonalize: %s", why);
  if (batch == 0 || rows == 0 || columns == 0) return report_error(CPAB_OK, "%s", "");
  if (batch > 65536 || rows > kMostRows || columns > kMostRows)
    return report_error(CPAB_ERR_SIZE, "%s", "orthogonalize: at most 65536 matrices of 2^20 rows and columns");
  if (x == nullptr || out == nullptr || workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256)
    return report_error(CPAB_ERR_ARG, "%s", "orthogonalize: null pointer, or a workspace off 256 bytes");
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const std::vector<Set> sets = {{(int)rows, (int)columns, dtype, (int)batch}};
  std::vector<Places> places;
  double *partials;
  place(sets, batch, static_cast<char *>(workspace), &places, &partials);
  std::vector<Prepared> list((size_t)batch);
  const Set &t = sets[0];
  for (int64_t z = 0; z < batch; ++z) {
    const int64_t at = z * t.m() * t.x_pitch();
    list[z] = {static_cast<const char *>(x) + z * rows * columns * dtype_size(dtype), nullptr, places[0].x[0][0] + at,
               places[0].x[0][1] + at, partials + z * kPartials, places[0].terms + z * kTerms, t.x_pitch(), (int)rows, (int)columns, dtype, t.turned()};
  }
  cudaError_t e = prepare(list, 0.f, 0, steps, coefficients, eps, s);
  FinalGroup f = {};
  f.out = out, f.stride = rows * columns, f.first = -1, f.dtype = dtype, f.turned = t.turned();
  f.wide = !t.turned() && aligned_to(out, columns, dtype_size(dtype), 32);
  if (e == cudaSuccess) e = schulz(sets, places, &f, nullptr, 0, steps, s);
  return launch_status(e, "orthogonalize");
}

namespace cpab {
namespace {

// The tensors of one sequence of launches: sets of one shape and type, and the
// tensors of each in turn.
struct Sequence {
  std::vector<Set> sets;
  std::vector<int> tensors;
};

std::vector<Sequence> sequences(const cpab_muon_tensor *tensors, int count) {
  std::vector<Set> shapes;
  std::vector<std::vector<int>> members;
  for (int i = 0; i < count; ++i) {
    const cpab_muon_tensor &t = tensors[i];
    if (t.rows == 0 || t.columns == 0) continue;
    size_t k = 0;
    while (k < shapes.size() && !(shapes[k].rows == t.rows && shapes[k].cols == t.columns && shapes[k].dtype == t.dtype &&
                                  shapes[k].batch < kMatrices))
      ++k;
    if (k == shapes.size()) {
      shapes.push_back({(int)t.rows, (int)t.columns, t.dtype, 0});
      members.emplace_back();
    }
    ++shapes[k].batch;
    members[k].push_back(i);
  }
  std::vector<Sequence> list;
  for (size_t k = 0; k < shapes.size(); ++k) {
    if (list.empty() || list.back().sets.size() == kGroups ||
        list.back().sets[0].parts() != shapes[k].parts() ||
        list.back().tensors.size() + members[k].size() > (size_t)kMatrices)
      list.emplace_back();
    list.back().sets.push_back(shapes[k]);
    list.back().tensors.insert(list.back().tensors.end(), members[k].begin(), members[k].end());
  }
  return list;
}

// What the list lacks, or null.
const char *check_tensors(const cpab_muon_tensor *tensors, int count) {
  if (count < 0 || (count > 0 && tensors == nullptr)) return "null tensors or a negative count";
  for (int i = 0; i < count; ++i) {
    const cpab_muon_tensor &t = tensors[i];
    if (!dtype_ok(t.dtype)) return "unknown element type";
    if (t.rows < 0 || t.columns < 0 || t.rows > kMostRows || t.columns > kMostRows)
      return "a matrix of a negative size or over 2^20 rows or columns";
    if (t.rows > 0 && t.columns > 0 && (t.param == nullptr || t.grad == nullptr || t.momentum == nullptr))
      return "null parameter, gradient or momentum";
  }
  return nullptr;
}

}  // namespace
}  // namespace cpab

extern "C" int64_t cpab_b200_muon_workspace(const cpab_muon_tensor *tensors, int count) {
  int64_t most = 0;
  if (check_tensors(tensors, count) != nullptr) return 0;
  for (const Sequence &q : sequences(tensors, count))
    most = std::max(most, place(q.sets, (int64_t)q.tensors.size(), nullptr, nullptr, nullptr));
  return most;
}

extern "C" int cpab_b200_muon(const cpab_muon_tensor *tensors, int count, double lr, const float *lr_device,
                              double momentum, int nesterov, double weight_decay, int steps,
                              const double *coefficients, double eps, int adjust, void *workspace,
                              cpab_stream_t stream) {
  if (coefficients == nullptr) return report_error(CPAB_ERR_ARG, "%s", "muon: null coefficients");
  const char *why = check_tensors(tensors, count);
  if (why == nullptr) why = check_steps(steps, coefficients, eps);
  if (why == nullptr && adjust != 0 && adjust != 1) why = "adjust must be 0 or 1";
  if (why != nullptr) return report_error(CPAB_ERR_ARG, "muon: %s", why);
  const std::vector<Sequence> list = sequences(tensors, count);
  if (!list.empty() && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256))
    return report_error(CPAB_ERR_ARG, "%s", "muon: null workspace, or one off 256 bytes");
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  for (const Sequence &q : list) {
    std::vector<Places> places;
    double *partials;
    place(q.sets, (int64_t)q.tensors.size(), static_cast<char *>(workspace), &places, &partials);
    std::vector<Prepared> in;
    std::vector<FinalGroup> finals(q.sets.size());
    void *table[kMatrices];
    for (size_t g = 0; g < q.sets.size(); ++g) {
      const Set &t = q.sets[g];
      FinalGroup &f = finals[g];
      f = {};
      f.first = (int)in.size(), f.dtype = t.dtype, f.turned = t.turned(), f.update = 1;
      f.decay = (float)weight_decay, f.lr = (float)lr, f.lr_device = lr_device;
      f.rate = (float)(adjust ? 0.2 * std::sqrt((double)t.n()) : std::sqrt(std::max(1.0, (double)t.rows / t.cols)));
      for (int z = 0; z < t.batch; ++z) {
        const int k = (int)in.size();
        const cpab_muon_tensor &m = tensors[q.tensors[k]];
        const int64_t at = z * t.m() * t.x_pitch();
        table[k] = m.param;
        if (z == 0) f.wide = !t.turned();
        f.wide = f.wide && aligned_to(m.param, t.cols, dtype_size(t.dtype), 32);
        in.push_back({m.grad, m.momentum, places[g].x[0][0] + at, places[g].x[0][1] + at, partials + k * kPartials,
                      places[g].terms + z * kTerms, t.x_pitch(), t.rows, t.cols, t.dtype, t.turned()});
      }
    }
    if ((e = prepare(in, (float)momentum, nesterov, steps, coefficients, eps, s)) != cudaSuccess) break;
    if ((e = schulz(q.sets, places, finals.data(), table, (int)in.size(), steps, s)) != cudaSuccess) break;
  }
  return launch_status(e, "muon");
}
