// The product kernel's skeleton: a persistent block (or pair of blocks that share
// one tile of 256 rows) walks tiles of C = A B^T; one warp fetches operand tiles
// into a ring of stages, one issues the matrix instructions, two bring scale words (idle
// without), eight move the accumulators from tensor memory to registers (each a quarter of the
// block's rows and half of the columns), hand the accumulator back at once, and give
// the values to the policy.
//
// The policy P says what is multiplied:
//   kCtas, kBN        blocks to a tile (128 rows each; 1 or 2), its columns
//   kScaled           e4m3 codes with e8m0 scales (128 codes a step), else halves (64)
//   kParts            2: operands are sums of two halves; a stage holds both, and
//                     takes part x part of all but the remainders' product
//   kBMn              B's rows run along the other axis than the summed one
//   kAcc              accumulators in turn
//   kChunk            columns that store takes at a time: 16 or 32
//   kSegment          stages to an accumulator, whose sums are then added in
//                     registers (0: a tile's all).  The tensor cores cut, not round,
//                     what a float32 sum cannot hold, so an error of up to 2^-24 of
//                     the sum a step piles up where a tile has hundreds of steps
//   Shared            what its epilogue keeps in shared memory
//   const Waits &waits()            how long a wait may last, and whom to tell
//   int tiles()                     tiles of this launch
//   Tile tile(int i)                {m0, n0, steps, ...}
//   warm(tile)                      touches its arguments
//   load(tile, step, a, b, bar, rank)    issues the copies of one stage; the second
//                     parts lie kAHalf and kBHalf bytes behind the first
//   stage_bytes()                   bytes that a stage's copies bring, to all blocks
//   scales_a(tile, rank, row, group, words), scales_b(tile, row, group, words)
//                     asks for a row's scales of 8 steps, four to a word (kScaled);
//   one_a(), one_b(), words_of_one(words)  whether a row has one scale, and the words of
//                     that one, once all rows' are asked for
//   begin(tile, shared, thread)     before a tile's accumulators are waited for
//   Ahead, ahead(tile, row, column)  what store reads besides, asked for a chunk early
//   store(tile, shared, row, column, values, ahead)  kChunk values of this thread's row;
//                     the warp's rows are 32 in order
#pragma once

#include "tensor_core.cuh"

namespace cpab {
namespace tc {

constexpr int kCoreThreads = 384;
constexpr int kEpilogueThreads = 256;
constexpr int kAHalf = 128 * 128;  // bytes of one part of A a block holds per stage

// The epilogue's warps alone.
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory"); }

template <class P>
struct CoreShape {
  static constexpr int kBHalf = P::kBN / P::kCtas * 128;  // bytes of one part of B a block holds
  static constexpr int kStageBytes = P::kParts * (kAHalf + kBHalf);
  // Scale words: a chunk is those of 128 rows and four steps (512 bytes, four columns
  // of tensor memory); a slot holds 8 steps', in shared memory and in tensor memory
  // alike.
  static constexpr int kScaleChunks = P::kScaled ? 1 + (P::kBN + 127) / 128 : 0;
  static constexpr int kScaleSlots = 2;
  static constexpr int kSlotBytes = 2 * kScaleChunks * 512, kSlotColumns = 2 * kScaleChunks * 4;
  static constexpr int kScaleBytes = kScaleSlots * kSlotBytes;
  static constexpr int kFixed = 1024 /* alignment */ + 512 /* barriers */ + kScaleBytes + (int)sizeof(typename P::Shared);
  static constexpr int kRoom = 227 * 1024 - kFixed;
  static constexpr int kStages = kRoom / kStageBytes > 8 ? 8 : kRoom / kStageBytes;
  static constexpr int kBytes = kFixed + kStages * kStageBytes;
  static constexpr int kScaleColumn = P::kAcc * P::kBN;  // first tensor-memory column of the scales
  static constexpr int kColumnsUsed = kScaleColumn + kScaleSlots * kSlotColumns;
  static constexpr int kColumns = kColumnsUsed <= 128 ? 128 : kColumnsUsed <= 256 ? 256 : 512;
  static_assert(sizeof(typename P::Shared) % 16 == 0, "barriers lie behind it");
  static_assert(kStages >= 3 && kColumnsUsed <= 512, "a tile too large");
  static_assert(kStageBytes % 1024 == 0, "swizzle atoms");
};

struct CoreBarriers {
  uint64_t full[8], empty[8], scale_full[2], scale_empty[2], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int gave_up;
};

// N columns from tensor memory; NaN where a wait ran out and the tile was given up.
template <int N>
__device__ __forceinline__ void read_accumulators(bool ok, uint32_t addr, float (&v)[N]) {
  if (ok) {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_load(addr + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
    tmem_load_wait();
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = __uint_as_float(0x7FFFFFFFu);
  }
}

template <class P>
__device__ __forceinline__ void core(const P &p) {
  using S = CoreShape<P>;
  constexpr int C = P::kCtas;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *scales = smem + S::kStages * S::kStageBytes;
  auto *shared = reinterpret_cast<typename P::Shared *>(scales + S::kScaleBytes);
  auto *bars = reinterpret_cast<CoreBarriers *>(reinterpret_cast<uint8_t *>(shared) + sizeof(typename P::Shared));
  const uint32_t stage0 = smem_u32(smem), scale0 = smem_u32(scales);
  const uint32_t full = smem_u32(bars->full), empty = smem_u32(bars->empty);
  const uint32_t sfull = smem_u32(bars->scale_full), sempty = smem_u32(bars->scale_empty);
  const uint32_t afull = smem_u32(bars->acc_full), aempty = smem_u32(bars->acc_empty);
  constexpr int kLength = P::kSegment > 0 ? P::kSegment : 1 << 30;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = C == 2 ? cluster_rank() : 0;

  dep_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) bar_init(full + 8 * i, 1), bar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bar_init(sfull + 8 * i, 2 * C), bar_init(sempty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) bar_init(afull + 8 * i, 1), bar_init(aempty + 8 * i, 8 * C);
    bars->gave_up = 0;
    bar_init_fence();
  }
  if (warp == 2) tmem_alloc<C>(smem_u32(&bars->tmem), S::kColumns);
  fence_before();
  if constexpr (C == 2) cluster_sync();
  else __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(~0u, *reinterpret_cast<volatile uint32_t *>(&bars->tmem), 0);
  volatile int *gave_up = &bars->gave_up;
  const int tiles = p.tiles(), first = blockIdx.x / C, stride = gridDim.x / C;
  // What the launch itself brings (arguments, tensor maps) is fetched while the
  // kernel before still runs.
  const auto first_tile = p.tile(first);
  p.warm(first_tile);
  const bool go = p.waits().longest > 0;
  dep_wait();

  // The pair's shared barriers are the first block's.
  const uint32_t full0 = C == 2 ? mapa(full, 0) : full;

  if (warp == 0) {
    int s = 0, phase = 0;
    bool ok = go;
    for (int i = first; i < tiles && ok; i += stride) {
      const auto t = i == first ? first_tile : p.tile(i);
      for (int k = 0; k < t.steps; ++k) {
        ok = bar_wait_warp(empty + 8 * s, phase ^ 1, p.waits());
        if (!ok) break;
        if (elect()) {
          if (rank == 0) bar_expect(full + 8 * s, p.stage_bytes());
          const uint32_t a = stage0 + s * S::kStageBytes;
          p.load(t, k, a, a + P::kParts * kAHalf, full0 + 8 * s, rank);
        }
        __syncwarp();
        if (++s == S::kStages) s = 0, phase ^= 1;
      }
    }
    if (!ok) *gave_up = 1;
  } else if (warp == 1) {
    if (rank == 0) {
      int s = 0, phase = 0, sc = 0, sphase = 0, acc = 0, aphase = 0;
      bool ok = go;
      for (int i = first; i < tiles && ok; i += stride) {
        const auto t = i == first ? first_tile : p.tile(i);
        for (int k = 0; k < t.steps; ++k) {
          const bool fresh = k % kLength == 0;
          if (fresh && !(ok = bar_wait_warp(aempty + 8 * acc, aphase ^ 1, p.waits()))) break;
          if constexpr (P::kScaled) {
            if ((k & 7) == 0) {
              if ((k > 0 || i != first) && ++sc == S::kScaleSlots) sc = 0, sphase ^= 1;
              if (!(ok = bar_wait_warp(sfull + 8 * sc, sphase, p.waits()))) break;
              fence_after();
              const uint32_t from = scale0 + sc * S::kSlotBytes, to = tmem + S::kScaleColumn + sc * S::kSlotColumns;
              const int chunks = min(2, (t.steps - k + 3) >> 2) * S::kScaleChunks;
              if (elect()) {
                for (int c = 0; c < chunks; ++c) scales_to_tmem<C>(to + 4 * c, plain_desc(from + 512 * c));
                mma_commit<C>(sempty + 8 * sc);
              }
              __syncwarp();
            }
          }
          if (!(ok = bar_wait_warp(full + 8 * s, phase, p.waits()))) break;
          fence_after();
          const bool last = k + 1 == t.steps || (k + 1) % kLength == 0;
          const uint32_t d = tmem + acc * P::kBN;
          const uint32_t a = stage0 + s * S::kStageBytes, b = a + P::kParts * kAHalf;
          const uint64_t da = swizzled_desc(a), db = swizzled_desc(b, P::kBMn ? 8192 : 16);
          const uint32_t words = tmem + S::kScaleColumn + sc * S::kSlotColumns + ((k & 7) >> 2) * S::kScaleChunks * 4;
          if (elect()) {
            // (the small products first, while the sum is small)
#pragma unroll
            for (int part = P::kParts == 2 ? 2 : 0; part >= 0; --part) {
              const uint64_t pa = da + (part == 2 ? kAHalf >> 4 : 0), pb = db + (part == 1 ? S::kBHalf >> 4 : 0);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const bool add = !fresh || j > 0 || part != (P::kParts == 2 ? 2 : 0);
                if constexpr (P::kScaled) {
                  // (the descriptor's scale bytes are those of this step of the four)
                  mma_mx<C>(d, pa + 2 * j, pb + 2 * j, idesc_mx(128 * C, P::kBN, 0) | ((k & 3) << 4) | ((k & 3) << 29),
                            words, words + 4, add);
                } else {
                  mma_f16<C>(d, pa + 2 * j, pb + (P::kBMn ? 128 : 2) * j, idesc_f16(128 * C, P::kBN, P::kBMn), add);
                }
              }
            }
            mma_commit<C>(empty + 8 * s);
            if (last) mma_commit<C>(afull + 8 * acc);
          }
          __syncwarp();
          if (++s == S::kStages) s = 0, phase ^= 1;
          if (last && ++acc == P::kAcc) acc = 0, aphase ^= 1;
        }
      }
      if (!ok) *gave_up = 1;
    }
  } else if (warp < 4) {
    if constexpr (P::kScaled) {
      // Warp 2 brings A's words (the first chunk of each four steps), warp 3 B's.
      constexpr int kB = S::kScaleChunks - 1;
      int sc = 0, sphase = 0;
      bool ok = go;
      for (int i = first; i < tiles && ok; i += stride) {
        const auto t = i == first ? first_tile : p.tile(i);
        for (int g = 0; 8 * g < t.steps && ok; ++g) {
          uint32_t w[kB][4][2];  // [chunk][row lane + 32 j][word]
#pragma unroll
          for (int c = 0; c < kB; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (warp == 3) p.scales_b(t, 128 * c + lane + 32 * j, g, w[c][j]);
              else if (c == 0) p.scales_a(t, rank, lane + 32 * j, g, w[c][j]);
            }
          if (warp == 3 ? p.one_b() : p.one_a()) {
#pragma unroll
            for (int c = 0; c < kB; ++c)
#pragma unroll
              for (int j = 0; j < 4; ++j) p.words_of_one(w[c][j]);
          }
          ok = bar_wait_warp(sempty + 8 * sc, sphase ^ 1, p.waits());
          uint8_t *to = scales + sc * S::kSlotBytes + 16 * lane + (warp == 3 ? 512 : 0);
#pragma unroll
          for (int c = 0; c < kB; ++c) {
            if ((warp == 2 && c > 0) || !ok) break;  // (a slot that is not free may still be read)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              *reinterpret_cast<uint4 *>(to + 512 * (q * S::kScaleChunks + c)) =
                  make_uint4(w[c][0][q], w[c][1][q], w[c][2][q], w[c][3][q]);
          }
          proxy_fence();
          __syncwarp();
          if (lane == 0 && ok) {
            if constexpr (C == 2) bar_arrive_cluster(mapa(sfull + 8 * sc, 0));
            else bar_arrive(sfull + 8 * sc);
          }
          if (++sc == S::kScaleSlots) sc = 0, sphase ^= 1;
        }
      }
      if (!ok) *gave_up = 1;
    }
  } else {
    constexpr int kHalf = P::kBN / 2;
    // Where another accumulator is free the values are taken 32 at a time, else all
    // at once, so that the accumulator is free early.
    constexpr int kHold = P::kSegment > 0 || P::kAcc == 1 ? kHalf : 32;
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    int acc = 0, aphase = 0;
    bool ok = go;
    for (int i = first; i < tiles; i += stride) {
      const auto t = i == first ? first_tile : p.tile(i);
      p.begin(t, *shared, threadIdx.x - 128);
      const int row = t.m0 + (int)rank * 128 + quarter * 32 + lane;
      const int segments = P::kSegment > 0 ? (t.steps + kLength - 1) / kLength : 1;
      float v[kHold];
      typename P::Ahead now = p.ahead(t, row, half * kHalf);
      for (int g = 0; g < segments; ++g) {
        ok = ok && bar_wait_warp(afull + 8 * acc, aphase, p.waits());
        fence_after();
        const uint32_t d = tmem + acc * P::kBN + half * kHalf + ((uint32_t)(quarter * 32) << 16);
        if constexpr (kHold < kHalf) {
#pragma unroll 1
          for (int c = 0; c < kHalf; c += kHold) {
            read_accumulators(ok, d + c, v);
#pragma unroll
            for (int j = 0; j < kHold; j += P::kChunk) {
              const int column = half * kHalf + c + j;
              const typename P::Ahead next = p.ahead(t, row, c + j + P::kChunk < kHalf ? column + P::kChunk : column);
              p.store(t, *shared, row, column, v + j, now);
              now = next;
            }
          }
        } else if (P::kSegment == 0 || g == 0) {
          read_accumulators(ok, d, v);
        } else {
#pragma unroll
          for (int c = 0; c < kHalf; c += 32) {
            float w[32];
            read_accumulators(ok, d + c, w);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[c + j] += w[j];
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0 && ok) {
          if constexpr (C == 2) bar_arrive_cluster(mapa(aempty + 8 * acc, 0));
          else bar_arrive(aempty + 8 * acc);
        }
        if (++acc == P::kAcc) acc = 0, aphase ^= 1;
      }
      if constexpr (kHold == kHalf) {
#pragma unroll
        for (int c = 0; c < kHalf; c += P::kChunk) {
          const typename P::Ahead next = p.ahead(t, row, half * kHalf + (c + P::kChunk < kHalf ? c + P::kChunk : c));
          p.store(t, *shared, row, half * kHalf + c, v + c, now);
          now = next;
        }
      }
    }
    if (!ok) *gave_up = 1;
  }

  __syncwarp();
  __syncthreads();
  if (*gave_up) {
    // Copies in flight land before the block ends.
    if (threadIdx.x == 0 && p.waits().gave_up != nullptr) {
      *static_cast<volatile int *>(p.waits().gave_up) = 1;
      __threadfence_system();
    }
    if (threadIdx.x == 0)
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  fence_before();
  if constexpr (C == 2) cluster_sync();
  else __syncthreads();
  fence_after();
  if (warp == 2) tmem_free<C>(tmem, S::kColumns);
}

}  // namespace tc
}  // namespace cpab
