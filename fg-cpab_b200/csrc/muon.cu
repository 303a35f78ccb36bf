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
//     their first halves (11 bits, 2^-12 off); the remainder enters the terms a X and
//     b A, which would otherwise drown small singular values beside large ones.  The
//     result is 1.5e-3 to 2.7e-3 off (relative 2-norm, normal matrices of up to 1500
//     rows), about a rounding to bfloat16 (1.7e-3); three products would take 2.2 times
//     as long.
//   - float32 ones and small ones take three products, first x first + first x
//     remainder + remainder x first (up to 5e-6 off): a float32 parameter keeps that
//     many bits of its update.
//
// 2^10 keeps values from 6e-8 in a half's normal range and leaves room to 64.  Where
// eps is not small beside |G|_F, X is: it is kept as theta Y with theta a power of two
// and |Y|_F in (1/2, 1], and the steps are taken in Y with
//   Y <- r (a + theta^2 b Y Y^T + theta^4 c (Y Y^T)^2) Y,   r = theta / theta',
// theta' the least power of two that keeps |Y| at 1 (by the coefficients' magnitudes), until
// theta is 1.
#include <algorithm>
#include <cmath>
#include <exception>
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
  int vectors;        // grad and momentum begin on 16 bytes
};
struct PrepareArgs {
  Prepared m[kPrepared];
  float momentum, rest;  // rest: 1 - momentum, of which the rounded momentum has fewer bits
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
  double most = 1.0;  // |Y| is no more
  for (int k = 0; k < steps; ++k) {
    const double q = theta * theta;
    double next = 1.0, r = 1.0;
    if (theta < 1.0) {
      const double x = q * most * most;
      most *= fabs(a) + x * (fabs(b) + x * fabs(c));
      int e;
      if (frexp(fmax(1.0, most), &e) == 0.5) --e;  // (powers of two themselves)
      next = fmin(1.0, ldexp(theta, e)), r = theta / next;
      most *= r;
    }
    to[3 * k] = (float)(a * r), to[3 * k + 1] = (float)(b * q * r), to[3 * k + 2] = (float)(c * q * q * r);
    theta = next;
  }
  to[3 * kMostSteps] = (float)theta;
}

// Eight elements from i on as float32 (wide: whole vectors).
__device__ __forceinline__ void read_eight(const void *p, int dtype, int64_t i, float (&v)[8]) {
  if (dtype == CPAB_F32) {
    const float4 x = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    const float4 y = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + 4);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    return;
  }
  const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = dtype == CPAB_F16 ? unpack_pair<__half>(q[k]) : unpack_pair<__nv_bfloat16>(q[k]);
    v[2 * k] = x.x, v[2 * k + 1] = x.y;
  }
}
__device__ __forceinline__ void write_eight(float *p, const float (&v)[8]) {
  *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// Momenta, and partial sums of the directions' squares (in float64: a square may
// leave float32's range where its element does not).
__global__ void __launch_bounds__(256) k_direction(const __grid_constant__ PrepareArgs a) {
  const Prepared &p = a.m[blockIdx.y];
  tc::dep_launch();
  tc::dep_wait();
  const int64_t n = (int64_t)p.rows * p.cols;
  const bool moving = p.momentum != nullptr;
  const float k = a.momentum;
  double sum = 0;
  auto one = [&](float g, float m, float *next) {
    float u = g;
    if (moving) {
      m = k * m + a.rest * g;
      u = a.nesterov ? a.rest * g + k * m : m;
    }
    *next = m;
    sum += (double)u * (double)u;
  };
  // (eights of whole vectors, then what is left)
  const int64_t eights = p.vectors ? n / 8 : 0;
#pragma unroll 2
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < eights; e += (int64_t)gridDim.x * 256) {
    float g[8], m[8] = {};
    read_eight(p.grad, p.dtype, 8 * e, g);
    if (moving) read_eight(p.momentum, CPAB_F32, 8 * e, m);
#pragma unroll
    for (int j = 0; j < 8; ++j) one(g[j], m[j], &m[j]);
    if (moving) write_eight(p.momentum + 8 * e, m);
  }
  for (int64_t i = 8 * eights + (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float m = moving ? p.momentum[i] : 0.f;
    one(read_as(p.grad, p.dtype, i), m, &m);
    if (moving) p.momentum[i] = m;
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

// Eight neighbours as halves and their remainders (rows are padded to 16).
__device__ __forceinline__ void store_eight(__half *hi, __half *lo, int64_t i, const float (&v)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[k] = pack_pair<__half>(v[2 * k], v[2 * k + 1]);
    const float2 x = unpack_pair<__half>(h[k]);
    l[k] = pack_pair<__half>(v[2 * k] - x.x, v[2 * k + 1] - x.y);
  }
  *reinterpret_cast<uint4 *>(hi + i) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4 *>(lo + i) = make_uint4(l[0], l[1], l[2], l[3]);
}

// Directions over their norms, as halves; tiles of 64 x 64, a thread eight columns
// of two rows (turned ones: eight rows of two columns on the way out).
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
  const bool moving = p.momentum != nullptr, whole = p.vectors && p.cols % 8 == 0;
  const int x = (threadIdx.x & 7) * 8, y0 = threadIdx.x >> 3;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int r0 = t / tiles_x * 64, c0 = t % tiles_x * 64;
#pragma unroll
    for (int y = y0; y < 64; y += 32) {
      const int64_t i = (int64_t)(r0 + y) * p.cols + c0 + x;
      if (r0 + y >= p.rows || c0 + x >= p.cols) continue;
      float g[8], m[8] = {};
      if (whole) {
        read_eight(p.grad, p.dtype, i, g);
        if (moving) read_eight(p.momentum, CPAB_F32, i, m);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = c0 + x + j < p.cols;
          g[j] = in ? read_as(p.grad, p.dtype, i + j) : 0.f;
          if (moving) m[j] = in ? p.momentum[i + j] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = !moving ? g[j] : a.nesterov ? a.rest * g[j] + a.momentum * m[j] : m[j];
        g[j] = (float)((double)u * scale);
        if (p.turned) tile[y][x + j] = g[j];
      }
      if (!p.turned) store_eight(p.hi, p.lo, (int64_t)(r0 + y) * p.pitch + c0 + x, g);
    }
    if (!p.turned) continue;
    __syncthreads();
#pragma unroll
    for (int y = y0; y < 64; y += 32) {
      if (c0 + y < p.cols && r0 + x < p.rows) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = r0 + x + j < p.rows ? tile[x + j][y] : 0.f;
        store_eight(p.hi, p.lo, (int64_t)(c0 + y) * p.pitch + r0 + x, v);
      }
    }
    __syncthreads();
  }
}

// ---- what comes out ------------------------------------------------------------

struct Finished {
  const __half *hi, *lo;  // [m, pitch]
  const float *terms;
  void *out;              // [rows, cols] of dtype, contiguous
  int64_t pitch;
  float rate;             // update: p (1 - lr decay) - lr rate O
  int rows, cols, dtype, turned, update;
  int vectors;            // out's rows begin on 16 bytes
};
struct FinishArgs {
  Finished m[kPrepared];
  float lr, decay;
  const float *lr_device;
};

// Results, or parameters' steps; tiles as those of k_normalise.  (In the last
// product's epilogue, where a thread has a row's columns, transposed parameters cost
// 430 us more for 42 million of them than this pass's 80.)
__global__ void __launch_bounds__(256) k_finish(const __grid_constant__ FinishArgs a) {
  const Finished &p = a.m[blockIdx.y];
  const int tiles_x = (p.cols + 63) / 64, tiles = tiles_x * ((p.rows + 63) / 64);
  tc::dep_launch();
  tc::dep_wait();
  if ((int)blockIdx.x >= tiles) return;
  __shared__ float tile[64][65];
  const float lr = a.lr_device != nullptr ? *a.lr_device : a.lr, theta = p.terms[3 * kMostSteps] * (1.f / kUnit);
  const float keep = 1.f - lr * a.decay, move = p.update ? -lr * p.rate * theta : theta;
  const int x = (threadIdx.x & 7) * 8, y0 = threadIdx.x >> 3;
  auto read = [&](int64_t i, float(&v)[8]) {
    float l[8];
    read_eight(p.hi, CPAB_F16, i, v);
    read_eight(p.lo, CPAB_F16, i, l);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += l[j];
  };
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int r0 = t / tiles_x * 64, c0 = t % tiles_x * 64;
    if (p.turned) {
#pragma unroll
      for (int y = y0; y < 64; y += 32) {
        float v[8] = {};
        if (c0 + y < p.cols && r0 + x < p.rows) read((int64_t)(c0 + y) * p.pitch + r0 + x, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[x + j][y] = v[j];
      }
      __syncthreads();
    }
#pragma unroll
    for (int y = y0; y < 64; y += 32) {
      if (r0 + y >= p.rows || c0 + x >= p.cols) continue;
      const int64_t i = (int64_t)(r0 + y) * p.cols + c0 + x;
      float v[8];
      if (p.turned) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[y][x + j];
      } else {
        read((int64_t)(r0 + y) * p.pitch + c0 + x, v);
      }
      if (p.vectors && c0 + x + 8 <= p.cols) {
        float old[8] = {};
        if (p.update) read_eight(p.out, p.dtype, i, old);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p.update ? fmaf(keep, old[j], move * v[j]) : move * v[j];
        if (p.dtype == CPAB_F32) {
          write_eight(static_cast<float *>(p.out) + i, v);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = p.dtype == CPAB_F16 ? pack_pair<__half>(v[2 * j], v[2 * j + 1])
                                       : pack_pair<__nv_bfloat16>(v[2 * j], v[2 * j + 1]);
          *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + x + j < p.cols)
            write_as(p.out, p.dtype, i + j,
                     p.update ? fmaf(keep, read_as(p.out, p.dtype, i + j), move * v[j]) : move * v[j]);
      }
    }
    if (p.turned) __syncthreads();
  }
}

// ---- the products ------------------------------------------------------------------

enum Phase { kGram, kSquare, kUpdate };

struct PhaseGroup {
  CUtensorMap a[2], b[2];          // first halves and remainders of the operands
  const __half *read[2];           // A (kSquare) or X (kUpdate)
  __half *write[2];                // A, B or the next X
  int64_t read_pitch, read_plane, write_pitch, write_plane;
  int m, n;                        // of the result
  int steps;                       // stages of 64 summed
  int tiles_m, tiles_n, end;       // tiles of one matrix; end of the group's in the launch
  int write_lo;
  const float *terms;              // of the set's first matrix, kTerms apart
  int splits, total;               // kGram: the sum over `total` stages in so many parts of `steps`,
  float *parts;                    // whose results go here as float32 (null: one part)
};
struct PhaseArgs {
  PhaseGroup g[kGroups];
  int groups, step;
  tc::Waits waits;
};

// What the tensor cores cut off a sum has one sign: 1.5e-5 of the sum at most over kLongest
// stages of halves, beside 2^-12 of its operands, but at 2^18 summed the result of 64 copies of
// a 1700 x 4096 matrix side by side was 2.4e-3 larger than one's.  X X^T of more stages (LONG,
// kernels of their own) therefore adds segments of kLongest in registers (2.3e-5; 1000 x
// 20000 680 us either way).
constexpr int kLongest = 128;

template <int PHASE, int PARTS, int CTAS, int BN, bool LONG>
struct Schulz {
  static constexpr int kCtas = CTAS, kBN = BN, kAcc = 2, kParts = PARTS;
  static constexpr int kChunk = PARTS == 2 && BN == 256 ? 16 : 32;
  static constexpr int kSegment = PARTS == 2 ? 4 : LONG ? kLongest : 0;
  static constexpr bool kScaled = false, kBMn = PHASE >= kUpdate, kSymmetric = PHASE <= kSquare;
  static constexpr int kBM = 128 * CTAS, kAcross = kBM / BN;
  static_assert(kBM % BN == 0, "tiles of symmetric results begin on the diagonal");
  struct alignas(16) Shared {};
  struct Tile {
    int m0, n0, steps, z, g;
    int k0, part;         // first stage and place of a part of the sum
    bool mirror, edge;  // stored turned too; some of it on or under the diagonal
  };
  const PhaseArgs &p;

  __device__ const tc::Waits &waits() const { return p.waits; }
  __device__ int tiles() const { return p.g[p.groups - 1].end; }
  __device__ Tile tile(int i) const {
    int g = 0, begin = 0;
    while (i >= p.g[g].end) begin = p.g[g++].end;
    const PhaseGroup &q = p.g[g];
    i -= begin;
    Tile t;
    t.g = g, t.steps = q.steps, t.k0 = 0, t.part = 0;
    if (kSymmetric) {  // rows of tiles, each from the diagonal on
      const int per = q.tiles_m * q.tiles_n - kAcross * (q.tiles_m * (q.tiles_m - 1) / 2);
      t.z = i / per, i %= per;
      int row = 0;
      for (int n = q.tiles_n; i >= n; n -= kAcross) i -= n, ++row;
      t.m0 = row * kBM, t.n0 = (row * kAcross + i) * BN;
      t.mirror = kAcross > 1 || i > 0, t.edge = kAcross > 1 && i < kAcross;
      if (PHASE == kGram && q.splits > 1) {
        t.part = t.z, t.z /= q.splits;
        t.k0 = (t.part - t.z * q.splits) * q.steps, t.steps = min(q.steps, q.total - t.k0);
      }
    } else {
      const int per = q.tiles_m * q.tiles_n;
      t.z = i / per, i %= per;
      t.m0 = i % q.tiles_m * kBM, t.n0 = i / q.tiles_m * BN, t.mirror = t.edge = false;
    }
    return t;
  }
  __device__ void warm(const Tile &t) const {
    const PhaseGroup &q = p.g[t.g];
    if (threadIdx.x < PARTS) tc::prefetch_map(&q.a[threadIdx.x]), tc::prefetch_map(&q.b[threadIdx.x]);
    tc::touch(q.read[0]), tc::touch(q.read[1]), tc::touch(q.write[0]), tc::touch(q.write[1]), tc::touch(q.terms);
    tc::touch(q.read_plane), tc::touch(q.write_plane), tc::touch(q.write_lo), tc::touch(p.step);
  }
  __device__ void load(const Tile &t, int k, uint32_t sa, uint32_t sb, uint32_t bar, uint32_t rank) const {
    const PhaseGroup &q = p.g[t.g];
    const int at = (t.k0 + k) * 64, n = t.n0 + rank * (BN / CTAS);
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
      tc::tile_load<CTAS>(sa + h * tc::kAHalf, &q.a[h], bar, at, t.m0 + rank * 128, t.z);
      const uint32_t to = sb + h * (BN / CTAS * 128);
#pragma unroll
      for (int c = 0; c < BN / CTAS; c += 64) {  // boxes of 64 rows
        if constexpr (kBMn) tc::tile_load<CTAS>(to + c * 128, &q.b[h], bar, n + c, at, t.z);
        else tc::tile_load<CTAS>(to + c * 128, &q.b[h], bar, at, n + c, t.z);
      }
    }
  }
  __device__ uint32_t stage_bytes() const { return CTAS * tc::CoreShape<Schulz>::kStageBytes; }
  __device__ void begin(const Tile &, Shared &, int) const {}

  // A's or X's halves in the place of what is stored.  (Read when a chunk is stored and
  // not one ahead, their latency alone was half of an update's time.)
  struct Ahead {
    uint32_t hi[PHASE == kGram ? 1 : kChunk / 2], lo[PHASE == kGram ? 1 : kChunk / 2];
    float mine, product;  // coefficients of it and of the product
  };
  __device__ Ahead ahead(const Tile &t, int row, int c) const {
    Ahead w = {};
    w.product = 1.f / kUnit;
    if constexpr (PHASE != kGram) {
      const PhaseGroup &q = p.g[t.g];
      const float *terms = q.terms + t.z * kTerms + 3 * p.step;
      w.mine = terms[PHASE == kSquare ? 1 : 0];
      if (PHASE == kSquare) w.product *= terms[2];
      const int col = t.n0 + c;
      const int64_t at = t.z * q.read_plane + row * q.read_pitch + col;
#pragma unroll
      for (int k = 0; k < kChunk; k += 16) {
        uint32_t h[8] = {}, l[8] = {};
        if (row < q.m && col + k < q.n) {  // (rows are padded to 16)
          tc::load_sector(q.read[0] + at + k, h);
          tc::load_sector(q.read[1] + at + k, l);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) w.hi[k / 2 + j] = h[j], w.lo[k / 2 + j] = l[j];
      }
    }
    return w;
  }
  __device__ void store(const Tile &t, const Shared &, int row, int c, const float *acc, const Ahead &w) const {
    const PhaseGroup &q = p.g[t.g];
    if (PHASE == kGram && q.splits > 1) {
      float *to = q.parts + t.part * q.write_plane + row * q.write_pitch + t.n0 + c;
#pragma unroll
      for (int k = 0; k < kChunk; k += 8) {
        uint32_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __float_as_uint(acc[k + j] * w.product);
        if (row < q.m && t.n0 + c + k < q.n) tc::store_sector(to + k, x);
      }
      return;
    }
    __half *hi = q.write[0] + t.z * q.write_plane, *lo = q.write[1] + t.z * q.write_plane;
    const int odd = threadIdx.x & 1;
#pragma unroll
    for (int k = 0; k < kChunk; k += 16) {
      const int col = t.n0 + c + k;
      if (col >= q.n) return;
      uint32_t h[8], l[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a = acc[k + 2 * j] * w.product, b = acc[k + 2 * j + 1] * w.product;
        if constexpr (PHASE != kGram) {
          const float2 x = unpack_pair<__half>(w.hi[k / 2 + j]), y = unpack_pair<__half>(w.lo[k / 2 + j]);
          a = fmaf(w.mine, x.x + y.x, a), b = fmaf(w.mine, x.y + y.y, b);
        }
        h[j] = pack_pair<__half>(a, b);
        const float2 x = unpack_pair<__half>(h[j]);
        l[j] = pack_pair<__half>(a - x.x, b - x.y);
      }
      // A value and its mirror image come from one sum: what lies under the diagonal is
      // not stored from here.
      const int rows0 = row - (int)(threadIdx.x & 31);
      if (t.edge && col < rows0 + 32) {
        if (col + 16 <= rows0) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int column = col + j;
          if (row >= q.m || column >= q.n || column < row) continue;
          const __half x = __ushort_as_half((uint16_t)(h[j >> 1] >> (16 * (j & 1))));
          const __half y = __ushort_as_half((uint16_t)(l[j >> 1] >> (16 * (j & 1))));
          const int64_t at = row * q.write_pitch + column, to = column * q.write_pitch + row;
          hi[at] = x, hi[to] = x;
          if (q.write_lo) lo[at] = y, lo[to] = y;
        }
        continue;
      }
      // (what lies past a row's end, up to the next multiple of 16, is never read as a value)
      if (row < q.m) {
        const int64_t at = row * q.write_pitch + col;
        tc::store_sector(hi + at, h);
        if (q.write_lo) tc::store_sector(lo + at, l);
      }
      if (t.mirror) {
        // Neighbouring rows' threads swap, so that each stores two rows of one column.
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t oh = __shfl_xor_sync(~0u, h[j], 1), ol = __shfl_xor_sync(~0u, l[j], 1);
          const uint32_t th = odd ? __byte_perm(oh, h[j], 0x7632) : __byte_perm(h[j], oh, 0x5410);
          const uint32_t tl = odd ? __byte_perm(ol, l[j], 0x7632) : __byte_perm(l[j], ol, 0x5410);
          const int column = col + 2 * j + odd;
          if (column < q.n && row < q.m) {
            const int64_t to = (int64_t)column * q.write_pitch + (row & ~1);
            *reinterpret_cast<uint32_t *>(hi + to) = th;
            if (q.write_lo) *reinterpret_cast<uint32_t *>(lo + to) = tl;
          }
        }
      }
    }
  }
};

template <int PHASE, int PARTS, int CTAS, int BN, bool LONG>
__global__ void __launch_bounds__(tc::kCoreThreads, 1)
    k_schulz(const __grid_constant__ PhaseArgs a) {
  tc::core(Schulz<PHASE, PARTS, CTAS, BN, LONG>{a});
}

template <int PHASE, int PARTS, int CTAS, int BN>
cudaError_t launch_phase_as(PhaseArgs &a, const int *batch, cudaStream_t s) {
  using S = tc::CoreShape<Schulz<PHASE, PARTS, CTAS, BN, false>>;  // (as large with segments)
  auto *kernel = k_schulz<PHASE, PARTS, CTAS, BN, false>;
  if constexpr (PHASE == kGram && PARTS == 1) {
    for (int g = 0; g < a.groups; ++g)
      if (a.g[g].steps > kLongest) kernel = k_schulz<PHASE, PARTS, CTAS, BN, true>;
  }
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (e != cudaSuccess) return e;
  int64_t tiles = 0;
  for (int g = 0; g < a.groups; ++g) {
    PhaseGroup &q = a.g[g];
    constexpr int kBM = 128 * CTAS;
    q.tiles_m = (q.m + kBM - 1) / kBM, q.tiles_n = (q.n + BN - 1) / BN;
    int64_t per = (int64_t)q.tiles_m * q.tiles_n;
    if (PHASE <= kSquare) per -= kBM / BN * ((int64_t)q.tiles_m * (q.tiles_m - 1) / 2);
    if (PHASE == kGram) per *= q.splits;
    tiles += per * batch[g];
    if (tiles >= int64_t(1) << 30) return cudaErrorInvalidValue;
    q.end = (int)tiles;
  }
  return tc::launch(kernel, (unsigned)(CTAS * std::min<int64_t>(tiles, device_info().sm_count / CTAS)), tc::kCoreThreads,
                    S::kBytes, CTAS, s, a);
}

// A of the parts of its sum, added in order: tiles of 64 x 64 on and above the
// diagonal, each stored twice.
__global__ void __launch_bounds__(256) k_join(const __grid_constant__ PhaseArgs a) {
  int g = 0, z = blockIdx.y;
  tc::dep_launch();
  tc::dep_wait();
  // (the groups' matrices one after another; `end` counts those of groups in parts)
  while (z >= a.g[g].end) z -= a.g[g++].end;
  const PhaseGroup &q = a.g[g];
  const int side = (q.m + 63) / 64;
  int row = 0, i = blockIdx.x;
  if (i >= side * (side + 1) / 2) return;
  for (int n = side; i >= n; --n) i -= n, ++row;
  const int r0 = row * 64, c0 = (row + i) * 64;
  __shared__ float tile[64][65];
  const int x = (threadIdx.x & 7) * 8, y0 = threadIdx.x >> 3;
#pragma unroll
  for (int y = y0; y < 64; y += 32) {
    float v[8] = {};
    if (r0 + y < q.m && c0 + x < q.m) {  // (rows are padded to 16)
      const float *from = q.parts + (int64_t)z * q.splits * q.write_plane + (r0 + y) * q.write_pitch + c0 + x;
      float p[8][8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < q.splits) read_eight(from + k * q.write_plane, CPAB_F32, 0, p[k]);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < q.splits) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += p[k][j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) tile[y][x + j] = v[j];
  }
  __syncthreads();
  __half *hi = q.write[0] + z * q.write_plane, *lo = q.write[1] + z * q.write_plane;
#pragma unroll
  for (int y = y0; y < 64; y += 32) {
    float v[8];
    if (r0 + y < q.m && c0 + x < q.m) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i == 0 && x + j < y ? tile[x + j][y] : tile[y][x + j];
      store_eight(hi, lo, (r0 + y) * q.write_pitch + c0 + x, v);
    }
    if (i > 0 && c0 + y < q.m && r0 + x < q.m) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tile[x + j][y];
      store_eight(hi, lo, (c0 + y) * q.write_pitch + r0 + x, v);
    }
  }
}

// Joins what kGram left in parts (nothing, where it left none).
cudaError_t launch_join(const PhaseArgs &grams, const int *batch, cudaStream_t s) {
  PhaseArgs a = grams;
  int matrices = 0, tiles = 0;
  for (int g = 0; g < a.groups; ++g) {
    a.g[g].end = a.g[g].splits > 1 ? batch[g] : 0;
    if (a.g[g].splits == 1) continue;
    const int side = (a.g[g].m + 63) / 64;
    matrices += batch[g], tiles = std::max(tiles, side * (side + 1) / 2);
  }
  if (matrices == 0) return cudaSuccess;
  return tc::launch(k_join, dim3((unsigned)tiles, (unsigned)matrices), 256, 0, 1, s, a);
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
  float *terms, *parts;
  int splits;
};
// Parts that the sums of X X^T are cut into where tiles are few and the sums long: as
// many as there are blocks for, of at least four stages.  Five steps of 256 x 4096: 169 us,
// in one part 278; 100 x 4000 float32 144 and 249; 1024 x 1024 207 and 221.
int splits_of(const std::vector<Set> &sets, const Set &set) {
  int64_t tiles = 0;
  for (const Set &s : sets) {
    const int64_t t = (s.m() + 127) / 128;
    tiles += t * (t + 1) / 2 * s.batch;
  }
  const int64_t stages = (set.n() + 63) / 64;
  const int64_t parts = std::min<int64_t>({8, device_info().sm_count / std::max<int64_t>(1, tiles), stages / 4});
  if (parts < 2) return 1;
  const int64_t each = (stages + parts - 1) / parts;
  return (int)((stages + each - 1) / each);
}
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
    const int splits = splits_of(sets, s);
    float *parts = splits > 1 ? reinterpret_cast<float *>(take(4 * splits * s.a_halves())) : nullptr;
    if (places != nullptr) (*places)[i].terms = terms, (*places)[i].parts = parts, (*places)[i].splits = splits;
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

// Tiles of 128 x 64 or 128 x 128, or 256 x 256 by a pair of blocks, by the time that the
// waves of tiles should take (as tile_of in product.cu).
template <int PHASE, int PARTS>
cudaError_t launch_phase(PhaseArgs &a, const int *batch, cudaStream_t s) {
  const int64_t sms = device_info().sm_count;
  const int rows[3] = {128, 128, 256}, columns[3] = {64, 128, 256};
  // (narrow tiles on the diagonal are stored element by element)
  const float launch[3] = {PHASE <= kSquare ? 6.5f : 4.f, 5.f, 7.f}, wave[3] = {0.5f, 1.f, 2.f};
  const float step[3] = {PARTS == 2 ? 0.36f : 0.2f, PARTS == 2 ? 0.5f : 0.25f, PARTS == 2 ? 0.85f : 0.33f};
  int best = 0;
  float least = 0.f;
  for (int k = 0; k < 3; ++k) {
    int64_t tiles = 0;
    double work = 0;
    for (int g = 0; g < a.groups; ++g) {
      const PhaseGroup &q = a.g[g];
      const int64_t tm = (q.m + rows[k] - 1) / rows[k], tn = (q.n + columns[k] - 1) / columns[k];
      const int64_t per = (tm * tn - (PHASE <= kSquare ? rows[k] / columns[k] * (tm * (tm - 1) / 2) : 0)) * batch[g] * (PHASE == kGram ? q.splits : 1);
      tiles += per, work += (double)per * (wave[k] + step[k] * (float)q.steps);
    }
    const int64_t slots = std::max<int64_t>(1, k == 2 ? sms / 2 : sms), waves = (tiles + slots - 1) / slots;
    const float t = launch[k] + (float)(work / (double)tiles * (double)waves);
    if (k == 0 || t < least) best = k, least = t;
  }
  switch (best) {
    case 2: return launch_phase_as<PHASE, PARTS, 2, 256>(a, batch, s);
    case 1: return launch_phase_as<PHASE, PARTS, 1, 128>(a, batch, s);
    default: return launch_phase_as<PHASE, PARTS, 1, 64>(a, batch, s);
  }
}

// The products of at most kGroups sets, all of one kind.
template <int PARTS>
cudaError_t schulz_as(const std::vector<Set> &sets, const std::vector<Places> &places, int steps, cudaStream_t s) {
  int batch[kGroups];
  PhaseArgs a;
  const int groups = (int)sets.size();
  a.groups = groups, a.waits = tc::waits();
  for (int g = 0; g < groups; ++g) batch[g] = sets[g].batch;
  for (int step = 0; step < steps; ++step) {
    const int now = step & 1;
    a.step = step;
    bool ok = true;
    cudaError_t e;
    for (int g = 0; g < groups; ++g) {
      const Set &t = sets[g];
      const Places &w = places[g];
      PhaseGroup &q = a.g[g];
      for (int h = 0; h < 2; ++h) {
        ok = ok && map_of(&q.a[h], w.x[now][h], t.n(), t.m(), t.batch, t.x_pitch(), 128);
        ok = ok && map_of(&q.b[h], w.x[now][h], t.n(), t.m(), t.batch, t.x_pitch(), 64);
        q.read[h] = nullptr, q.write[h] = w.a[h];
      }
      q.terms = w.terms;
      q.write_pitch = t.a_pitch(), q.write_plane = t.m() * t.a_pitch();
      q.m = q.n = t.m(), q.total = (t.n() + 63) / 64, q.write_lo = 1;
      q.splits = w.splits, q.parts = w.parts, q.steps = (q.total + q.splits - 1) / q.splits;
    }
    if (!ok) return cudaErrorInvalidValue;
    if ((e = launch_phase<kGram, PARTS>(a, batch, s)) != cudaSuccess) return e;
    if ((e = launch_join(a, batch, s)) != cudaSuccess) return e;
    for (int g = 0; g < groups; ++g) {
      const Set &t = sets[g];
      const Places &w = places[g];
      PhaseGroup &q = a.g[g];
      for (int h = 0; h < 2; ++h) {
        ok = ok && map_of(&q.a[h], w.a[h], t.m(), t.m(), t.batch, t.a_pitch(), 128);
        ok = ok && map_of(&q.b[h], w.a[h], t.m(), t.m(), t.batch, t.a_pitch(), 64);
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
    e = launch_phase<kUpdate, PARTS>(a, batch, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t schulz(const std::vector<Set> &sets, const std::vector<Places> &places, int steps, cudaStream_t s) {
  return sets[0].parts() == 2 ? schulz_as<2>(sets, places, steps, s) : schulz_as<1>(sets, places, steps, s);
}

// Launches what reads the matrices in.
cudaError_t prepare(const std::vector<Prepared> &list, double momentum, int nesterov, int steps, const double *c,
                    double eps, cudaStream_t s) {
  for (size_t first = 0; first < list.size(); first += kPrepared) {
    const int n = (int)std::min<size_t>(kPrepared, list.size() - first);
    PrepareArgs a;
    int64_t most = 0, tiles = 0;
    for (int i = 0; i < n; ++i) {
      a.m[i] = list[first + i];
      a.m[i].vectors = reinterpret_cast<uintptr_t>(a.m[i].grad) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(a.m[i].momentum) % 16 == 0;
      most = std::max(most, (int64_t)a.m[i].rows * a.m[i].cols);
      tiles = std::max(tiles, (int64_t)((a.m[i].rows + 63) / 64) * ((a.m[i].cols + 63) / 64));
    }
    a.momentum = (float)momentum, a.rest = (float)(1.0 - momentum), a.nesterov = nesterov, a.steps = steps, a.eps = eps, a.a = c[0], a.b = c[1], a.c = c[2];
    const int partials = (int)std::min<int64_t>(kPartials, (most + 2047) / 2048);
    cudaError_t e = tc::launch(k_direction, dim3(partials, n), 256, 0, 1, s, a);
    if (e == cudaSuccess)
      e = tc::launch(k_normalise, dim3((unsigned)std::min<int64_t>(tiles, 65535), n), 256, 0, 1, s, a, partials);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Launches what writes the results.
cudaError_t finish(const std::vector<Finished> &list, double lr, const float *lr_device, double decay, cudaStream_t s) {
  for (size_t first = 0; first < list.size(); first += kPrepared) {
    const int n = (int)std::min<size_t>(kPrepared, list.size() - first);
    FinishArgs a;
    int64_t tiles = 0;
    for (int i = 0; i < n; ++i) {
      Finished &m = a.m[i] = list[first + i];
      m.vectors = aligned_to(m.out, m.cols, dtype_size(m.dtype), 16);
      tiles = std::max(tiles, (int64_t)((m.rows + 63) / 64) * ((m.cols + 63) / 64));
    }
    a.lr = (float)lr, a.decay = (float)decay, a.lr_device = lr_device;
    const cudaError_t e =
        tc::launch(k_finish, dim3((unsigned)std::min<int64_t>(tiles, 65535), n), 256, 0, 1, s, a);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// ---- small matrices ------------------------------------------------------------------
//
// A matrix of few rows stays in shared memory through all steps, its columns spread
// over the blocks of a cluster: one launch in place of 18.  Each block forms its columns' part of X X^T; the blocks add the parts
// of one share each, in order, and hand the sums to all; each squares a share of the
// rows of A and hands B to all; each updates its own columns.  All as pairs of halves.

constexpr int kSmallThreads = 512, kSmallWarps = kSmallThreads / 32;
constexpr int kSmallRows = 128;
constexpr int kSmallUnits = 3;    // 16 x 32 results a warp holds
constexpr int kSmallSums = 9;     // times four sums a thread holds
constexpr int kSmallBytes = 220 * 1024;

struct Small {
  const void *grad;
  float *momentum;
  void *out;
  int rows, cols, dtype, update;
  float rate;
};
struct SmallArgs {
  Small m[kMatrices];
  int64_t stride;        // > 0: matrix z is m[0]'s, z * stride elements on
  float momentum, rest, lr, decay;
  const float *lr_device;
  int nesterov, steps;
  double eps, a, b, c;
};

// Sizes of a matrix's parts in a cluster of `blocks`.
struct SmallShape {
  int m, n, rows, columns;  // rows padded to 16, columns of a block padded to 16
  __host__ __device__ SmallShape(int rows_, int cols, int blocks) {
    m = rows_ < cols ? rows_ : cols, n = rows_ < cols ? cols : rows_;
    rows = (m + 15) / 16 * 16;
    columns = ((n + blocks - 1) / blocks + 15) / 16 * 16;
  }
  // (8 halves more than a row's: the eight rows of a matrix load lie in different banks)
  __host__ __device__ int a_pitch() const { return rows + 8; }
  __host__ __device__ int x_pitch() const { return columns + 8; }
  __host__ __device__ int bytes() const { return rows * (a_pitch() + x_pitch()) * 4; }
  bool fits(int blocks) const {
    const int r = rows / 16, wide = (rows + 31) / 32;
    return m <= kSmallRows && bytes() <= kSmallBytes && r * ((columns + 31) / 32) <= kSmallUnits * kSmallWarps &&
           (r + blocks - 1) / blocks * wide <= kSmallUnits * kSmallWarps &&
           (r + blocks - 1) / blocks * 4 * a_pitch() <= kSmallSums * kSmallThreads;
  }
};

__device__ __forceinline__ void load_matrices(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Pairs of halves in shared memory: `lo` lies `skip` bytes behind.
struct Halves {
  uint32_t hi, skip;
  int pitch;
  __device__ uint32_t at(int row, int column) const { return hi + (uint32_t)(row * pitch + column) * 2; }
};

// acc = A[row0.., :K] B: 16 rows and 32 columns (the second 16 where `both`); B's rows
// are its columns' (B^T as it lies), or with TURNED the summed ones.
template <bool TURNED>
__device__ __forceinline__ void unit(const Halves &A, const Halves &B, int row0, int col0, int K, bool both, int lane,
                                     float (&acc)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  const uint32_t from = A.at(row0 + (lane & 15), (lane >> 4) * 8);
  const uint32_t with = TURNED ? B.at(lane & 15, col0 + (lane >> 4) * 8)
                               : B.at(col0 + (lane & 7) + ((lane >> 4) << 3), ((lane >> 3) & 1) * 8);
  const uint32_t along = (TURNED ? 16 * B.pitch : 16) * 2, second = both ? (TURNED ? 16 : 16 * B.pitch) * 2 : 0;
#pragma unroll 1
  for (int k = 0; k < K / 16; ++k) {
    uint32_t ah[4], al[4], bh[2][4], bl[2][4];
    load_matrices(from + 32 * k, ah);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // (where there is no second half, the first again)
      const uint32_t b = with + along * k + second * h;
      if (TURNED) {
        load_matrices_turned(b + B.skip, bl[h]);
        load_matrices_turned(b, bh[h]);
      } else {
        load_matrices(b + B.skip, bl[h]);
        load_matrices(b, bh[h]);
      }
    }
    load_matrices(from + 32 * k + A.skip, al);
    // (one sum's three products four instructions apart)
#pragma unroll
    for (int i = 0; i < 4; ++i) mma_16816(acc[i], ah, bl[i >> 1][2 * (i & 1)], bl[i >> 1][2 * (i & 1) + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) mma_16816(acc[i], ah, bh[i >> 1][2 * (i & 1)], bh[i >> 1][2 * (i & 1) + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) mma_16816(acc[i], al, bh[i >> 1][2 * (i & 1)], bh[i >> 1][2 * (i & 1) + 1]);
  }
}

__device__ __forceinline__ float4 load_peer(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ double load_peer_double(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_peer(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void store_peer(uint32_t addr, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ uint32_t load_word(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_word(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// Two neighbours' value, and their halves.
__device__ __forceinline__ float2 value_of(const Halves &h, int row, int column) {
  const float2 x = unpack_pair<__half>(load_word(h.at(row, column)));
  const float2 y = unpack_pair<__half>(load_word(h.at(row, column) + h.skip));
  return make_float2(x.x + y.x, x.y + y.y);
}
__device__ __forceinline__ void halves_of(float a, float b, uint32_t *hi, uint32_t *lo) {
  *hi = pack_pair<__half>(a, b);
  const float2 x = unpack_pair<__half>(*hi);
  *lo = pack_pair<__half>(a - x.x, b - x.y);
}

__global__ void __launch_bounds__(kSmallThreads, 1) k_schulz_small(const __grid_constant__ SmallArgs a) {
  extern __shared__ __align__(16) uint8_t small_smem[];
  __shared__ double part[kSmallWarps], mine;
  __shared__ float terms[kTerms];
  const int blocks = tc::cluster_blocks(), rank = (int)tc::cluster_rank();
  const int z = blockIdx.x / blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Small p = a.m[a.stride > 0 ? 0 : z];
  if (a.stride > 0) {
    const int64_t skip = z * a.stride * (p.dtype == CPAB_F32 ? 4 : 2);
    p.grad = static_cast<const char *>(p.grad) + skip, p.out = static_cast<char *>(p.out) + skip;
  }
  const SmallShape t(p.rows, p.cols, blocks);
  const bool turned = p.rows > p.cols;
  const int n0 = rank * t.columns, own = max(0, min(t.columns, t.n - n0));  // this block's columns
  const uint32_t base = tc::smem_u32(small_smem);
  const Halves R = {base, (uint32_t)(t.rows * t.a_pitch() * 2), t.a_pitch()};
  const Halves X = {base + 2 * R.skip, (uint32_t)(t.rows * t.x_pitch() * 2), t.x_pitch()};
  tc::dep_launch();
  tc::dep_wait();

  // What goes in: element e of this block's part, in memory's order.
  const int inner = turned ? t.m : own, count = t.m * own;
  auto place = [&](int e, int *row, int *column) {
    const int x = e % inner, y = e / inner;
    *row = turned ? x : y, *column = turned ? y : x;
    return turned ? (int64_t)(n0 + y) * p.cols + x : (int64_t)y * p.cols + n0 + x;
  };
  auto direction_of = [&](int64_t i, float m) {
    const float g = read_as(p.grad, p.dtype, i);
    return p.momentum == nullptr ? g : a.nesterov ? a.rest * g + a.momentum * m : m;
  };
  double sum = 0;
  for (int e = threadIdx.x; e < count; e += kSmallThreads) {
    int row, column;
    const int64_t i = place(e, &row, &column);
    float m = 0.f;
    if (p.momentum != nullptr) {
      m = a.momentum * p.momentum[i] + a.rest * read_as(p.grad, p.dtype, i);
      p.momentum[i] = m;
    }
    const double u = direction_of(i, m);
    sum += u * u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) part[warp] = sum;
  for (uint32_t w = threadIdx.x; w < X.skip / 2; w += kSmallThreads) store_word(X.hi + 4 * w, 0);  // (padding is 0)
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < kSmallWarps; ++w) sum += part[w];
    mine = sum;
  }
  tc::cluster_sync();
  sum = 0;
  for (int c = 0; c < blocks; ++c) sum += load_peer_double(tc::mapa(tc::smem_u32(&mine), c));
  const double norm = sqrt(sum), theta = first_theta(norm, a.eps), scale = (double)kUnit / ((norm + a.eps) * theta);
  if (threadIdx.x == 0) write_terms(terms, theta, a.a, a.b, a.c, a.steps);
  for (int e = threadIdx.x; e < count; e += kSmallThreads) {
    int row, column;
    const int64_t i = place(e, &row, &column);
    const float v = (float)((double)direction_of(i, p.momentum != nullptr ? p.momentum[i] : 0.f) * scale);
    const __half h = __float2half_rn(v);
    __half *to = reinterpret_cast<__half *>(small_smem + 2 * R.skip) + row * X.pitch + column;
    *to = h;
    to[X.skip / 2] = __float2half_rn(v - __half2float(h));
  }
  __syncthreads();

  const int row_blocks = t.rows / 16, wide = (t.rows + 31) / 32;
  // This block's share of A's and B's rows, and the fours of their elements.
  const int share0 = rank * row_blocks / blocks, shares = (rank + 1) * row_blocks / blocks - share0;
  const int fours = shares * 4 * R.pitch;
  const int fr = lane >> 2, fc = 2 * (lane & 3);                           // a fragment's row and column
  for (int step = 0; step < a.steps; ++step) {
    // The columns' part of X X^T, in float32 where A will lie.
    for (int u = warp; u < row_blocks * wide; u += kSmallWarps) {
      const int row = u / wide * 16, col = u % wide * 32;
      const bool both = col + 16 < t.rows;
      float acc[4][4];
      unit<false>(X, X, row, col, t.columns, both, lane, acc);
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        if (f >= 2 && !both) break;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<float2 *>(small_smem + ((row + fr + 8 * h) * R.pitch + col + 8 * f + fc) * 4) =
              make_float2(acc[f][2 * h] * (1.f / kUnit), acc[f][2 * h + 1] * (1.f / kUnit));
      }
    }
    tc::cluster_sync();
    float4 v[kSmallSums];
#pragma unroll
    for (int k = 0; k < kSmallSums; ++k) {
      const int q = threadIdx.x + k * kSmallThreads;
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (q < fours) {
        const uint32_t from = base + (uint32_t)(share0 * 16 * R.pitch + 4 * q) * 4;
        // (all blocks' parts asked for before the first is added)
        float4 x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < blocks) x[c] = load_peer(tc::mapa(from, c));
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < blocks) v[k].x += x[c].x, v[k].y += x[c].y, v[k].z += x[c].z, v[k].w += x[c].w;
      }
    }
    tc::cluster_sync();
#pragma unroll
    for (int k = 0; k < kSmallSums; ++k) {
      const int q = threadIdx.x + k * kSmallThreads;
      if (q < fours) {
        uint2 hi, lo;
        halves_of(v[k].x, v[k].y, &hi.x, &lo.x);
        halves_of(v[k].z, v[k].w, &hi.y, &lo.y);
        const uint32_t to = R.hi + (uint32_t)(share0 * 16 * R.pitch + 4 * q) * 2;
        for (int c = 0; c < blocks; ++c) {
          const uint32_t peer = tc::mapa(to, c);
          store_peer(peer, hi);
          store_peer(peer + R.skip, lo);
        }
      }
    }
    tc::cluster_sync();
    // This block's rows of B = b A + c A A.
    float acc[kSmallUnits][4][4];
    const float ta = terms[3 * step], tb = terms[3 * step + 1], product = terms[3 * step + 2] * (1.f / kUnit);
#pragma unroll
    for (int k = 0; k < kSmallUnits; ++k) {
      const int u = warp + k * kSmallWarps;
      if (u < shares * wide) {
        const int row = (share0 + u / wide) * 16, col = u % wide * 32;
        unit<false>(R, R, row, col, t.rows, col + 16 < t.rows, lane, acc[k]);
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (f >= 2 && col + 16 >= t.rows) break;
            const float2 w = value_of(R, row + fr + 8 * h, col + 8 * f + fc);
            acc[k][f][2 * h] = tb * w.x + product * acc[k][f][2 * h];
            acc[k][f][2 * h + 1] = tb * w.y + product * acc[k][f][2 * h + 1];
          }
      }
    }
    tc::cluster_sync();
#pragma unroll
    for (int k = 0; k < kSmallUnits; ++k) {
      const int u = warp + k * kSmallWarps;
      if (u < shares * wide) {
        const int row = (share0 + u / wide) * 16, col = u % wide * 32;
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (f >= 2 && col + 16 >= t.rows) break;
            uint32_t hi, lo;
            halves_of(acc[k][f][2 * h], acc[k][f][2 * h + 1], &hi, &lo);
            const uint32_t to = R.at(row + fr + 8 * h, col + 8 * f + fc);
            store_word(to, hi);
            store_word(to + R.skip, lo);
          }
      }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < fours; q += kSmallThreads) {  // (16 bytes: eight halves or remainders)
      const int half = fours / 2;
      const uint32_t at = (uint32_t)(share0 * 16 * R.pitch * 2 + 16 * (q < half ? q : q - half)) + (q < half ? 0 : R.skip);
      const uint4 w = *reinterpret_cast<const uint4 *>(small_smem + at);
      for (int c = 0; c < blocks; ++c)
        if (c != rank) store_peer(tc::mapa(base + at, c), w);
    }
    tc::cluster_sync();
    // X <- a X + B X, own columns.
    const int across = (t.columns + 31) / 32;
#pragma unroll
    for (int k = 0; k < kSmallUnits; ++k) {
      const int u = warp + k * kSmallWarps;
      if (u < row_blocks * across) {
        const int row = u / across * 16, col = u % across * 32;
        unit<true>(R, X, row, col, t.rows, col + 16 < t.columns, lane, acc[k]);
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (f >= 2 && col + 16 >= t.columns) break;
            const float2 w = value_of(X, row + fr + 8 * h, col + 8 * f + fc);
            acc[k][f][2 * h] = ta * w.x + acc[k][f][2 * h] * (1.f / kUnit);
            acc[k][f][2 * h + 1] = ta * w.y + acc[k][f][2 * h + 1] * (1.f / kUnit);
          }
      }
    }
    __syncthreads();
    const bool end = step + 1 == a.steps;
    const float lr = a.lr_device != nullptr ? *a.lr_device : a.lr;
    const float final_theta = terms[3 * kMostSteps] * (1.f / kUnit);
    const float keep = 1.f - lr * a.decay, move = p.update ? -lr * p.rate * final_theta : final_theta;
#pragma unroll
    for (int k = 0; k < kSmallUnits; ++k) {
      const int u = warp + k * kSmallWarps;
      if (u < row_blocks * across) {
        const int row = u / across * 16, col = u % across * 32;
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (f >= 2 && col + 16 >= t.columns) break;
            const int r = row + fr + 8 * h, c = col + 8 * f + fc;
            if (!end) {
              uint32_t hi, lo;
              halves_of(acc[k][f][2 * h], acc[k][f][2 * h + 1], &hi, &lo);
              store_word(X.at(r, c), hi);
              store_word(X.at(r, c) + X.skip, lo);
              continue;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (r >= t.m || c + j >= own) continue;
              const int64_t i = turned ? (int64_t)(n0 + c + j) * p.cols + r : (int64_t)r * p.cols + n0 + c + j;
              const float o = move * acc[k][f][2 * h + j];
              write_as(p.out, p.dtype, i, p.update ? fmaf(keep, read_as(p.out, p.dtype, i), o) : o);
            }
          }
      }
    }
    __syncthreads();
  }
}

// The cluster for matrices of these shapes: the smallest that holds each, and twice
// that while blocks are few and columns many; 0: some matrix is too large.
int small_cluster(const Small *m, int shapes, int64_t count) {
  for (int blocks = 1; blocks <= 8; blocks *= 2) {
    int columns = 0;
    bool ok = true;
    for (int i = 0; i < shapes; ++i) {
      const SmallShape t(m[i].rows, m[i].cols, blocks);
      ok = ok && t.fits(blocks);
      columns = std::max(columns, t.columns);
    }
    if (ok && (blocks == 8 || columns <= 32 || 2 * blocks * count > device_info().sm_count)) return blocks;
    if (ok && blocks < 8) {
      bool next = true;
      for (int i = 0; i < shapes; ++i) next = next && SmallShape(m[i].rows, m[i].cols, 2 * blocks).fits(2 * blocks);
      if (!next) return blocks;
    }
  }
  return 0;
}

// Five steps by one launch and by a launch for each product (us, float32): 64 x 64 49,
// 49 x 2048 90, 128 x 128 80, 128 x 300 104, 128 x 1000 143; 130 x 260 119, 192 x 192 130.
// What the blocks hand each other (8 bytes a clock) grows with the rows' square.
bool is_small(int64_t rows, int64_t columns) {
  const int64_t m = std::min(rows, columns), n = std::max(rows, columns);
  return m <= kSmallRows && n <= 1 << 16 && (m <= 64 || m * n <= 1 << 16) &&
         SmallShape((int)rows, (int)columns, 8).fits(8);
}

cudaError_t launch_small(const SmallArgs &a, int shapes, int64_t count, cudaStream_t s) {
  const int blocks = small_cluster(a.m, shapes, count);
  int bytes = 0;
  for (int i = 0; i < shapes; ++i) bytes = std::max(bytes, SmallShape(a.m[i].rows, a.m[i].cols, blocks).bytes());
  const cudaError_t e = cudaFuncSetAttribute(k_schulz_small, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmallBytes);
  if (e != cudaSuccess) return e;
  return tc::launch(k_schulz_small, (unsigned)(blocks * count), kSmallThreads, bytes, blocks, s, a);
}

constexpr int64_t kMostRows = 1 << 20;

// No exception leaves a C entry (the lists may ask for more memory than there is).
template <typename F>
int guarded(const char *what, F f) {
  try {
    return f();
  } catch (const std::exception &e) {
    return report_error(CPAB_ERR_SIZE, "%s: %s", what, e.what());
  }
}

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
  if (is_small(rows, columns)) return 0;
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
  if (x == nullptr || out == nullptr) return report_error(CPAB_ERR_ARG, "%s", "orthogonalize: null pointer");
  if (tc::gave_up()) return tc::report_gave_up("orthogonalize");
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (is_small(rows, columns)) {
    SmallArgs a = {};
    a.m[0] = {x, nullptr, out, (int)rows, (int)columns, dtype, 0, 0.f};
    a.stride = rows * columns, a.steps = steps, a.eps = eps;
    a.a = coefficients[0], a.b = coefficients[1], a.c = coefficients[2];
    return launch_status(launch_small(a, 1, batch, s), "orthogonalize");
  }
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256)
    return report_error(CPAB_ERR_ARG, "%s", "orthogonalize: a null workspace, or one off 256 bytes");
  return guarded("orthogonalize", [&]() -> int {
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
    cudaError_t e = prepare(list, 0.0, 0, steps, coefficients, eps, s);
    if (e == cudaSuccess) e = schulz(sets, places, steps, s);
    std::vector<Finished> results((size_t)batch);
    for (int64_t z = 0; z < batch; ++z) {
      const int64_t at = z * t.m() * t.x_pitch();
      results[z] = {places[0].x[steps & 1][0] + at, places[0].x[steps & 1][1] + at, places[0].terms + z * kTerms,
                    static_cast<char *>(out) + z * rows * columns * dtype_size(dtype), t.x_pitch(), 1.f, (int)rows,
                    (int)columns, dtype, t.turned(), 0};
    }
    if (e == cudaSuccess) e = finish(results, 0.0, nullptr, 0.0, s);
    return launch_status(e, "orthogonalize");
  });
}

namespace cpab {
namespace {

// The tensors of one sequence of launches: sets of one shape and type, and the
// tensors of each in turn.
struct Sequence {
  std::vector<Set> sets;
  std::vector<int> tensors;
};

// Whether a tensor's step is taken by the kernel for small matrices: not where others
// go through the products as pairs of halves anyway, whose launches it joins.
struct Split {
  bool joined = false;
  Split(const cpab_muon_tensor *tensors, int count) {
    for (int i = 0; i < count && !joined; ++i) {
      const cpab_muon_tensor &t = tensors[i];
      joined = t.rows > 0 && t.columns > 0 && !is_small(t.rows, t.columns) &&
               Set{(int)t.rows, (int)t.columns, t.dtype, 1}.parts() == 2;
    }
  }
  bool small(const cpab_muon_tensor &t) const { return !joined && is_small(t.rows, t.columns); }
};

std::vector<Sequence> sequences(const cpab_muon_tensor *tensors, int count) {
  const Split split(tensors, count);
  std::vector<Set> shapes;
  std::vector<std::vector<int>> members;
  for (int i = 0; i < count; ++i) {
    const cpab_muon_tensor &t = tensors[i];
    if (t.rows == 0 || t.columns == 0 || split.small(t)) continue;
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
  // (steps of one matrix at a time would race)
  std::vector<const void *> seen;
  for (int i = 0; i < count; ++i)
    if (tensors[i].rows > 0 && tensors[i].columns > 0) seen.push_back(tensors[i].param), seen.push_back(tensors[i].momentum);
  std::sort(seen.begin(), seen.end());
  if (std::adjacent_find(seen.begin(), seen.end()) != seen.end()) return "a parameter or momentum given twice";
  // (the momentum is written before the gradient is read for the second time)
  std::vector<const void *> momenta;
  for (int i = 0; i < count; ++i)
    if (tensors[i].rows > 0 && tensors[i].columns > 0) momenta.push_back(tensors[i].momentum);
  std::sort(momenta.begin(), momenta.end());
  for (int i = 0; i < count; ++i)
    if (tensors[i].rows > 0 && tensors[i].columns > 0 && std::binary_search(momenta.begin(), momenta.end(), tensors[i].grad))
      return "a gradient that is a momentum";
  return nullptr;
}

}  // namespace
}  // namespace cpab

extern "C" int64_t cpab_b200_muon_workspace(const cpab_muon_tensor *tensors, int count) {
  int64_t most = 0;
  guarded("muon", [&]() -> int {
    if (check_tensors(tensors, count) != nullptr) return CPAB_ERR_ARG;
    for (const Sequence &q : sequences(tensors, count))
      most = std::max(most, place(q.sets, (int64_t)q.tensors.size(), nullptr, nullptr, nullptr));
    return CPAB_OK;
  });
  return most;
}

extern "C" int cpab_b200_muon(const cpab_muon_tensor *tensors, int count, double lr, const float *lr_device,
                              double momentum, int nesterov, double weight_decay, int steps,
                              const double *coefficients, double eps, int adjust, void *workspace,
                              cpab_stream_t stream) {
  if (coefficients == nullptr) return report_error(CPAB_ERR_ARG, "%s", "muon: null coefficients");
  return guarded("muon", [&]() -> int {
    const char *why = check_tensors(tensors, count);
    if (why == nullptr) why = check_steps(steps, coefficients, eps);
    if (why == nullptr && adjust != 0 && adjust != 1) why = "adjust must be 0 or 1";
    if (why != nullptr) return report_error(CPAB_ERR_ARG, "muon: %s", why);
    const std::vector<Sequence> list = sequences(tensors, count);
    if (!list.empty() && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256))
      return report_error(CPAB_ERR_ARG, "%s", "muon: null workspace, or one off 256 bytes");
    if (tc::gave_up()) return tc::report_gave_up("muon");
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    auto rate = [&](int64_t rows, int64_t columns) {
      return (float)(adjust ? 0.2 * std::sqrt((double)std::max(rows, columns))
                            : std::sqrt(std::max(1.0, (double)rows / (double)columns)));
    };
    const Split split(tensors, count);
    SmallArgs small = {};
    small.momentum = (float)momentum, small.rest = (float)(1.0 - momentum), small.lr = (float)lr, small.decay = (float)weight_decay, small.lr_device = lr_device;
    small.nesterov = nesterov, small.steps = steps, small.eps = eps;
    small.a = coefficients[0], small.b = coefficients[1], small.c = coefficients[2];
    for (int i = 0, n = 0; i <= count; ++i) {
      if (n > 0 && (n == kMatrices || i == count)) {
        if ((e = launch_small(small, n, n, s)) != cudaSuccess) return launch_status(e, "muon");
        n = 0;
      }
      if (i == count) break;
      const cpab_muon_tensor &t = tensors[i];
      if (t.rows > 0 && t.columns > 0 && split.small(t))
        small.m[n++] = {t.grad, t.momentum, t.param, (int)t.rows, (int)t.columns, t.dtype, 1, rate(t.rows, t.columns)};
    }
    for (const Sequence &q : list) {
      std::vector<Places> places;
      double *partials;
      place(q.sets, (int64_t)q.tensors.size(), static_cast<char *>(workspace), &places, &partials);
      std::vector<Prepared> in;
      std::vector<Finished> out;
      for (size_t g = 0; g < q.sets.size(); ++g) {
        const Set &t = q.sets[g];
        for (int z = 0; z < t.batch; ++z) {
          const int k = (int)in.size();
          const cpab_muon_tensor &m = tensors[q.tensors[k]];
          const Places &w = places[g];
          const int64_t at = z * t.m() * t.x_pitch();
          in.push_back({m.grad, m.momentum, w.x[0][0] + at, w.x[0][1] + at, partials + k * kPartials, w.terms + z * kTerms,
                        t.x_pitch(), t.rows, t.cols, t.dtype, t.turned()});
          out.push_back({w.x[steps & 1][0] + at, w.x[steps & 1][1] + at, w.terms + z * kTerms, m.param, t.x_pitch(),
                         rate(t.rows, t.cols), t.rows, t.cols, t.dtype, t.turned(), 1});
        }
      }
      if ((e = prepare(in, momentum, nesterov, steps, coefficients, eps, s)) != cudaSuccess) break;
      if ((e = schulz(q.sets, places, steps, s)) != cudaSuccess) break;
      if ((e = finish(out, lr, lr_device, weight_decay, s)) != cudaSuccess) break;
    }
    return launch_status(e, "muon");
  });
}
