// Tensor-core products on sm_100a: barriers, tile copies, tensor memory and
// matrix instructions as PTX, for product.cu and muon.cu.
//
// A tile of operand lies in shared memory as rows of 128 bytes, eight rows to a
// swizzle atom of 1024 bytes (the tile copies write it so), and a matrix
// instruction takes 32 bytes of each row: 32 codes of 8 bits or 16 halves.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cpab {
namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ---- barriers ----------------------------------------------------------------

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The address of block `rank`'s copy of a shared address in this cluster, and an
// arrival there.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// How long a wait of these kernels may last (nanoseconds; 0: what waits gives up at once)
// and the word that is set where one ran out, in memory that the host reads too (or null).
struct Waits {
  uint64_t longest;
  int *gave_up;
};

// Waits for the phase of the given parity.  Every wait of these kernels ends: after
// `longest` (two seconds by default; a tile's whole sum, the longest in earnest, takes 0.4
// us for each 128 codes or 64 halves, milliseconds at most) the caller gives its work up.
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const Waits &waits) {
  for (int i = 0; i < 16; ++i)
    if (bar_try(bar, parity)) return true;
  const uint64_t begin = nanoseconds();
  do {
    if (bar_try(bar, parity)) return true;
  } while (nanoseconds() - begin < waits.longest);
  return false;
}
// The same for a whole warp, with one answer.
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, const Waits &waits) {
  return __all_sync(~0u, bar_wait(bar, parity, waits));
}

// One lane of a whole warp.  (Copies and matrix instructions take their operands from
// the warp's uniform registers: warps that issue them run their loops whole and elect
// a lane for the issue alone.  With loops of lane 0 a matrix instruction took twice
// its time: 8192 x 8192 x 8192 codes 482 us.)
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_blocks() {
  int n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// Orders this thread's writes to shared memory before later reads of the tile
// copies and matrix instructions.
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Programmatic launch: the next kernel of the stream may begin while this one
// ends; what it reads of this one's results it reads after dep_wait, and with ordinary
// loads: read-only ones (__ldg, ld.global.nc) are for memory that nothing writes while
// the kernel runs, and it runs while this one writes.
__device__ __forceinline__ void dep_launch() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- tile copies ---------------------------------------------------------------

// Copies the box at (x, y, z) of a tensor to this block's shared memory; its bytes
// count on `bar`, which with CTAS == 2 may be the other block's of the pair.
template <int CTAS>
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  if constexpr (CTAS == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Keeps a load whose value nothing needs.
template <typename T>
__device__ __forceinline__ void touch(const T &v) {
  if constexpr (sizeof(T) == 8) asm volatile("" ::"l"(v));
  else asm volatile("" ::"r"(v));
}

// ---- tensor memory -------------------------------------------------------------

// (one whole warp; with CTAS == 2 one of each block of the pair)
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 "tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::"r"(slot), "r"(columns) : "memory");
  else
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                 "tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::"r"(slot), "r"(columns) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: v[j] is column addr + j of the thread's row.
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
// 32 bytes at once (a whole sector), aligned to 32.
__device__ __forceinline__ void store_sector(void *p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void load_sector(const void *p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p) : "memory");
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- matrix instructions ---------------------------------------------------------

// Shared-memory descriptor.  K-major (rows of 128 bytes along the summed axis,
// swizzled): atoms of eight rows 1024 bytes apart; the distance in the other
// direction is not used.  MN-major (64 halves of the other axis to a row): atoms
// of eight summed indices 1024 bytes apart, the next 64 halves `lead` bytes on.
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t addr, uint32_t lead = 16) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Plain (no swizzle) 8-row groups of 16-byte rows, 128 bytes apart: scale words.
__device__ __forceinline__ uint64_t plain_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}

// Instruction descriptors: float32 accumulators, M x N (M of both blocks of a
// pair); halves, B as given (mn: 64 halves of N to a row); e4m3 codes with e8m0 scales,
// byte `sf` of each scale word.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__host__ __device__ constexpr uint32_t idesc_mx(int M, int N, int sf) {
  return ((uint32_t)sf << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) |
         ((uint32_t)sf << 29);
}

template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (CTAS == 2)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       bool add) {
  if constexpr (CTAS == 2)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(sfa), "r"(sfb) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(sfa), "r"(sfb) : "memory");
}
// 128 scale words (32 rows of 16 bytes; word w of row i is that of operand row
// 32 w + i) to four columns of tensor memory, for every quarter of the lanes; with
// CTAS == 2 in both blocks, each from its own shared memory.
template <int CTAS>
__device__ __forceinline__ void scales_to_tmem(uint32_t d, uint64_t desc) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(d), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(d), "l"(desc) : "memory");
}
// One arrival on `bar` (with CTAS == 2 on that of both blocks) when this thread's
// matrix instructions so far are done.
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// A launch in clusters of `cluster` blocks that may begin while the stream's last
// kernel ends (a kernel so launched calls dep_wait before it touches memory).
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned block, size_t shared, unsigned cluster, cudaStream_t s,
                   const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3(block), cfg.dynamicSmemBytes = shared, cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// What a launch on the current device passes on, and whether a kernel of an earlier one
// gave up waiting there (once for each time; the answer to the call is then reported as
// CPAB_ERR_WAIT).  Defined in product.cu.
Waits waits();
bool gave_up();
int report_gave_up(const char *what);

}  // namespace tc

// A tensor map of `rows` rows of `columns` elements (`pitch` bytes apart), `batch`
// of them (`plane` bytes apart), whose boxes of 128 bytes x box_rows arrive
// swizzled; elements outside read 0.  Defined in product.cu; false: refused.
bool make_tile_map(CUtensorMap *map, bool halves, const void *base, int64_t columns, int64_t rows, int64_t batch,
                   int64_t pitch, int64_t plane, int box_rows);

}  // namespace cpab
