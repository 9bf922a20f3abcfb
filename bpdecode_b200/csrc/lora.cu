// Low-rank adapters of many requests beside a projection that they share:
//
//   y[t, n] = sum_k x[t, k] W[n, k] + s_a sum_j (sum_k x[t, k] A_a[j, k]) B_a[n, j]
//
// with a = ids[t], no adapter where ids[t] is outside [0, num_adapters).
//
// Two launches. shrink_kernel computes S[t, j] = s_a sum_k x[t, k] A_a[j, k].
// project_kernel is one tcgen05 product: a tile of 128 outputs (the rows of W,
// the M side) by up to 256 rows of x (the N side) is accumulated in tensor
// memory over the inner elements, and the adapters are further steps of the
// same accumulation: B_a's tile times S, with S zero in the rows that have
// another adapter. Few rows are bound by reading W, which every row shares and
// which is read once; the adapters' steps then cost what reading B_a costs.
//
// The rows of S that a step covers are an item: a run of 16-row blocks that one
// adapter's rows lie in, with zeros in the rows of others. An item has a row
// for every kReach of its blocks at least, so a batch of single tokens has one
// item for each adapter, a prompt's runs have one each, and rows far apart one
// each; they need not be sorted. A matrix instruction over few rows costs
// nearly what one over 128 costs (about 87 cycles at 16 rows), which is why
// items are wide rather than exact: with 16-row items alone, 256 rows with 24
// adapters took 226 us at 65,536 outputs, against 161 so (154 in pairs, see below).
//
// Tiles of 256 rows are bound by what an SM loads, 48 KB for every 64 inner
// elements. Two CTAs then work as a pair (cta_group::2): an instruction of the
// first multiplies 256 outputs by 256 rows, each CTA has its own 128 outputs of
// W and half of the rows of x, and both accumulate their outputs for all rows.
// The first CTA's barriers count the loads of both, the adapters' too: all of them
// are tensor copies, which alone may be counted in another CTA.
//
// S is held as the sum of 16-bit values, each the rounding of what those before
// it left off: two of them keep 2^-17 of it in bf16 (one would cost 2^-9 of the
// adapter's part), and an fp32 result has a third. In fp16 two keep 2^-22 of it,
// but nothing below 2^-25, where fp16 ends: 2^-22 of S from 1/8 on.
//
// The matrix unit cuts its sums off to fp32 at every step, always towards zero:
// 4.4e-6 of the result at 4096 inner elements, and growing with them. A 16-bit
// result does not see that. An fp32 result is therefore accumulated 512 inner
// elements at a time, and these sums are added up in registers (5e-7, as fp32
// arithmetic has it).
//
// Times in these comments are of calls that follow one another on the same
// operands, a few at a time: what fits in L2 is there, and clocks are high. With
// caches flushed, or for seconds on end, they are larger (4096 rows by 4096 x 8192,
// 8 adapters of rank 64: 207 us here, 242 in a long run).
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"

namespace bpd {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kTileN = 128;        // outputs of a tile: the M of the matrix instruction
constexpr int kStepK = 64;         // inner elements of a step: one 128-byte swizzled row
constexpr int kBlock = 16;         // rows of x of a block
constexpr int kRankStep = 32;      // inner elements of an adapter's step, at most
constexpr int kMaxItems = 8;       // items of an adapters' step, at most
constexpr int kGroup = 8;           // steps that an fp32 result is accumulated over at once
constexpr int kReach = 4;          // blocks that an item spans for each row that it has, at most
// Tiles of rows up to which S is gathered row by row beside the product: with
// more, products of all of a block's adapters in front of it take less (750 rows
// by 4096 x 8192, 8 adapters of rank 64: 61 us, gathered 79; 4096 rows: 201, 217),
// with fewer, more (500 rows, 24 of rank 16: 66, gathered 52).
constexpr int kGatherTiles = 2;
constexpr int kMaxSplit = 8;       // CTAs of a cluster that share one tile's inner elements
constexpr int kThreads = 192;      // loads, products, four warps that write
constexpr int kShrinkThreads = 256;
constexpr uint64_t kGiveUpNs = 4000000000ull;  // a wait this long ends with an error

// A wait that gave up leaves its mark here (bpd_lora_take_error).
__device__ uint32_t g_error;

struct LoraArgs {
  const void* x;
  int64_t x_stride;
  int32_t T, K, N;
  const void* a;
  const void* b;
  const float* scale;
  int32_t adapters, rank;
  const void* ids;
  int32_t ids64;
  void* out;
  int64_t out_stride;
  // workspace: the items of each tile of rows
  int32_t* count;       // [row tiles]
  uint2* items;         // [row tiles, tile]: adapter; first block of S << 9 | its first block << 5
                        // | its blocks
  uint8_t* low;         // [row tiles, most_blocks, rank * parts * 32 bytes]: S of the items' blocks
  int32_t tile;         // rows that a tile has room for
  int32_t step;         // rows of a tile: as many in each, in whole blocks
  int32_t most_blocks;  // of S, of a tile's items
  int32_t row_tiles, out_tiles;
  int32_t parts;        // 16-bit values that make up one of S
  int32_t pair;         // CTAs that share the product's instructions: 1 or 2
  int32_t fp32;         // whether the result is
};

__device__ __forceinline__ int32_t adapter_of(const LoraArgs& g, int32_t t) {
  if (t >= g.T) return -1;
  const int64_t id = g.ids64 ? static_cast<const int64_t*>(g.ids)[t]
                             : static_cast<const int32_t*>(g.ids)[t];
  return id >= 0 && id < g.adapters ? static_cast<int32_t>(id) : -1;
}

// ---------------------------------------------------------------------------
// PTX

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// As bar_try, for what the cluster's other CTAs arrived for.
__device__ __forceinline__ bool bar_try_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// False where the wait gave up.
template <typename There>
__device__ __forceinline__ bool wait_for(There&& there) {
  if (there()) return true;
  const uint64_t start = now_ns();
  while (!there())
    if (now_ns() - start > kGiveUpNs) return false;
  return true;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  return wait_for([&] { return bar_try(bar, parity); });
}
template <int PAIR>
__device__ __forceinline__ bool bar_wait_free(uint32_t bar, uint32_t parity) {
  return wait_for(
      [&] { return PAIR == 2 ? bar_try_cluster(bar, parity) : bar_try(bar, parity); });
}
// The barrier at the same place in the cluster's CTA `rank`.
__device__ __forceinline__ void bar_arrive_at(uint32_t bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %0, %1;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar), "r"(rank)
      : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// A CTA's part of a pair's operands, counted by the first CTA's barrier.
__device__ __forceinline__ void load_box_for(uint32_t dst, const CUtensorMap* map, int32_t x,
                                             int32_t y, uint32_t first_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y),
      "r"(first_bar)
      : "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void load_bulk(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst), "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// One instruction of this CTA (PAIR 1) or of both CTAs of a pair, each with its
// own operands at these places: 128 outputs each, half of the rows of x each.
template <int PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (PAIR == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// Arrives where all instructions so far are through: in every CTA of the pair,
// or in this one.
template <int PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (PAIR == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar), "h"(static_cast<uint16_t>(3))
        : "memory");
}
template <int PAIR>
__device__ __forceinline__ void mma_commit_here(uint32_t bar) {
  if constexpr (PAIR == 1)
    mma_commit<1>(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// 16 bytes of the shared memory of the cluster's CTA `rank`; read behind a
// cluster barrier and before the next, where nothing writes them.
__device__ __forceinline__ float4 peer_float4(uint32_t own, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(own), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a));
  return v;
}
// 16 columns of this warp's 32 lanes of tensor memory.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory operand descriptors (K-major): rows of 128 swizzled bytes in
// groups of eight, or 8 x 16-byte core matrices, `lead` bytes from one to the
// next along K and 128 along the rows.
__device__ __forceinline__ uint64_t desc_swizzled(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_plain(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (uint64_t(lead >> 4) << 16) |
         (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}

// Instruction descriptor: fp32 accumulator, both operands of type T and
// K-major, M = 128 outputs for each CTA.
template <typename T, int PAIR>
constexpr uint32_t instruction(uint32_t n) {
  const uint32_t f = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((n >> 3) << 17) | ((PAIR * kTileN >> 4) << 24);
}

// ---------------------------------------------------------------------------
// S. An item's rows are gathered, up to 16 of them, and multiplied by its
// adapter's A over all inner elements; the warps split over the inner elements,
// which a cluster splits further where there are few items. Bound by the latency
// of reading A and x (12 to 18 us alone: 64 to 256 rows, 24 adapters of 4096
// inner elements), and hidden behind the product's reading of W: a CTA is small
// enough (20 KB of shared memory) to stand beside one of the product's. The
// products go through mma.sync, whose rate is no limit here. The order of the
// inner elements within a step is permuted, alike in both operands, so that every
// load is 16 bytes.

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// Where an item of `blocks` keeps eight values of S of its row `row`, from the
// inner element `col`: [CTA of the pair][rank step][part][rank / 8][rows][8].
__device__ __forceinline__ uint8_t* place_of(const LoraArgs& g, uint8_t* low, int32_t blocks,
                                             int32_t row, int32_t col, int32_t which) {
  const int32_t rows = blocks * kBlock / g.pair, cta = row >= rows;
  const int32_t c = col / kRankStep * kRankStep, wide = min(kRankStep, g.rank - c);
  return low + (cta * g.rank * g.parts + c * g.parts + which * wide) * rows * 2 +
         ((col - c) >> 3) * rows * 16 + (row - cta * rows) * 16;
}
// Writes them: each 16-bit part is the rounding of what those before it left.
template <typename T>
__device__ __forceinline__ void put_low(const LoraArgs& g, uint8_t* low, int32_t blocks,
                                        int32_t row, int32_t col, float (&s)[8]) {
  for (int32_t which = 0; which < g.parts; ++which) {
    alignas(16) typename Dt<T>::Bits part_of[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      part_of[e] = Dt<T>::from_float_dev(s[e]);
      s[e] -= Dt<T>::to_float(part_of[e]);
    }
    *reinterpret_cast<uint4*>(place_of(g, low, blocks, row, col, which)) =
        *reinterpret_cast<uint4*>(part_of);
  }
}

// The items of a tile of rows, made by kShrinkThreads threads, one for each row.
struct Plan {
  alignas(16) int32_t ids[256];
  uint2 items[256];       // as in LoraArgs
  uint16_t members[256];  // rows of an item that are its adapter's
  int32_t warp_items[kShrinkThreads / 32], warp_blocks[kShrinkThreads / 32];
};

// How many there are; `own` is the adapter of this thread's row, `rows_in` the
// rows that have it, a bit each.
__device__ __forceinline__ int32_t plan_items(const LoraArgs& g, int32_t t0, Plan& sh,
                                              int32_t& own, uint32_t (&rows_in)[8]) {
  constexpr int kWarps = kShrinkThreads / 32;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  own = tid < g.step ? adapter_of(g, t0 + tid) : -1;
  sh.ids[tid] = own;
  __syncthreads();
  // The first row of each adapter finds the adapter's items: runs of blocks
  // that hold at least one of its rows for every kReach blocks.
  bool lead = own >= 0;
  int32_t found = 0, blocks = 0;
  auto each_item = [&](auto&& f) {
    int32_t start = -1, end = 0, rows = 0;
#pragma unroll
    for (int32_t b = 0; b < 16; ++b) {
      if (b % g.pair) continue;  // a pair has whole blocks of 32 rows, half of each in a CTA
      const int32_t here = __popc(g.pair == 2 ? rows_in[b >> 1]
                                              : (rows_in[b >> 1] >> ((b & 1) * 16)) & 0xFFFFu);
      if (here == 0) continue;
      if (start >= 0 && b + g.pair - start > kReach * (rows + here)) {
        f(start, end - start, rows);
        start = -1;
      }
      if (start < 0) {
        start = b;
        rows = 0;
      }
      end = b + g.pair;
      rows += here;
    }
    if (start >= 0) f(start, end - start, rows);
  };
  if (lead) {
#pragma unroll
    for (int32_t w = 0; w < 8; ++w) {
      uint32_t m = 0;
#pragma unroll
      for (int32_t j = 0; j < 32; j += 4) {
        const int4 v = *reinterpret_cast<const int4*>(&sh.ids[w * 32 + j]);
        m |= (v.x == own ? 1u : 0u) << j | (v.y == own ? 2u : 0u) << j |
             (v.z == own ? 4u : 0u) << j | (v.w == own ? 8u : 0u) << j;
      }
      rows_in[w] = m;
      if (w < warp) lead = lead && m == 0;
      if (w == warp) lead = lead && (m & ((1u << lane) - 1u)) == 0;
    }
    if (lead)
      each_item([&](int32_t, int32_t n, int32_t) {
        ++found;
        blocks += n;
      });
  }
  // where this thread's items go: the sums over the threads before it
  int32_t at_item = found, at_block = blocks;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int32_t i = __shfl_up_sync(kFull, at_item, o), b = __shfl_up_sync(kFull, at_block, o);
    if (lane >= o) {
      at_item += i;
      at_block += b;
    }
  }
  if (lane == 31) {
    sh.warp_items[warp] = at_item;
    sh.warp_blocks[warp] = at_block;
  }
  __syncthreads();
  int32_t total = 0;
  at_item -= found;
  at_block -= blocks;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      at_item += sh.warp_items[w];
      at_block += sh.warp_blocks[w];
    }
    total += sh.warp_items[w];
  }
  if (lead)
    each_item([&](int32_t start, int32_t n, int32_t rows) {
      sh.items[at_item] = make_uint2(static_cast<uint32_t>(own),
                                  static_cast<uint32_t>(at_block << 9 | start << 5 | n));
      sh.members[at_item++] = static_cast<uint16_t>(rows);
      at_block += n;
    });
  __syncthreads();
  return total;
}

template <typename T, int RS>
__global__ void __launch_bounds__(kShrinkThreads, 2)
    shrink_kernel(const LoraArgs g, const int32_t turns, const int32_t split) {
  using Bits = typename Dt<T>::Bits;
  constexpr int kWarps = kShrinkThreads / 32;
  constexpr int kRows = 16;  // of a unit
  constexpr int kSlots = std::min(kWarps, 4096 / (kRows * RS));  // parts that are added at once
  constexpr int kUnroll = RS == 16 ? 4 : RS == 32 ? 3 : 2;
  __shared__ Plan plan;
  __shared__ uint8_t list[256];      // the rows of this item in the tile
  __shared__ int32_t warp_rows[kWarps];
  __shared__ float sums[kSlots][kRows][RS];
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t kpart = blockIdx.x % split;
  const int32_t turn = blockIdx.x / split % turns, tile = blockIdx.x / split / turns;
  const int32_t t0 = tile * g.step;
  pdl_wait();
  pdl_trigger();  // what ran before has completed: x is there for the next kernel, too
  int32_t own;
  uint32_t rows_in[8];
  const int32_t total = plan_items(g, t0, plan, own, rows_in);
  if (turn == 0 && kpart == 0) {
    if (tid < total) g.items[static_cast<int64_t>(tile) * g.tile + tid] = plan.items[tid];
    if (tid == 0) g.count[tile] = total;
  }

  const int32_t part = warp + kpart * kWarps;
  // each part is a contiguous share of the inner elements, a multiple of 32
  const int32_t share = ((g.K + 31) / 32 + kWarps * split - 1) / (kWarps * split) * 32;
  const int32_t k0 = min(g.K, part * share), k1 = min(g.K, k0 + share);
  // units are counted through the items; this CTA takes every turns-th
  int32_t before = 0, next = turn;
  for (int32_t i = 0; i < total; ++i) {
    const int32_t units = (plan.members[i] + kRows - 1) / kRows, u0 = next - before;
    before += units;
    if (u0 >= units) continue;  // alike in all threads of the cluster
    const int32_t a = static_cast<int32_t>(plan.items[i].x);
    const int32_t n = plan.items[i].y & 31u, b0 = (plan.items[i].y >> 5) & 15u;
    uint8_t* low = g.low + (static_cast<int64_t>(tile) * g.most_blocks + (plan.items[i].y >> 9)) *
                               (g.rank * g.parts * 32);
    const float scale = g.scale[a];
    // the item's rows, in order
    const bool mine = own == a && tid >= b0 * kBlock && tid < (b0 + n) * kBlock;
    const uint32_t vote = __ballot_sync(kFull, mine);
    if (lane == 0) warp_rows[warp] = __popc(vote);
    __syncthreads();
    int32_t at = __popc(vote & ((1u << lane) - 1u));
    for (int32_t w = 0; w < warp; ++w) at += warp_rows[w];
    if (mine) list[at] = static_cast<uint8_t>(tid);
    __syncthreads();
    auto place = [&](int32_t row, int32_t col, int32_t which) {
      return place_of(g, low, n, row, col, which);
    };
    if (u0 == 0) {  // the rows between
      for (int32_t v = tid + kpart * kShrinkThreads; v < n * kBlock * (g.rank / 8);
           v += kShrinkThreads * split) {
        const int32_t row = v % (n * kBlock), col = v / (n * kBlock) * 8;
        if (plan.ids[b0 * kBlock + row] != a) {
          for (int32_t which = 0; which < g.parts; ++which)
            *reinterpret_cast<uint4*>(place(row, col, which)) = uint4{};
        }
      }
    }
    for (int32_t u = u0; u < units; u += turns, next += turns) {
      const int32_t m0 = u * kRows, have = min(kRows, plan.members[i] - m0);
      const int32_t r0 = lane >> 2, r1 = r0 + 8;  // this lane's two rows
      const bool in0 = r0 < have, in1 = r1 < have;
      const Bits* x0 = static_cast<const Bits*>(g.x) +
                       static_cast<int64_t>(t0 + (in0 ? list[m0 + r0] : 0)) * g.x_stride;
      const Bits* x1 = static_cast<const Bits*>(g.x) +
                       static_cast<int64_t>(t0 + (in1 ? list[m0 + r1] : 0)) * g.x_stride;
      for (int32_t c = 0; c < g.rank; c += RS) {
        const int32_t rc = min(RS, g.rank - c);
        const Bits* w = static_cast<const Bits*>(g.a) +
                        (static_cast<int64_t>(a) * g.rank + c + (lane >> 2)) * g.K;
        float acc[RS / 8][4] = {};
        for (int32_t k = k0; k < k1; k += 32 * kUnroll) {
          uint4 p[kUnroll], q[kUnroll], v[kUnroll][RS / 8];
#pragma unroll
          for (int s = 0; s < kUnroll; ++s) {
            const int32_t e = k + s * 32 + (lane & 3) * 8;
            const bool in = e < k1;
            p[s] = in && in0 ? *reinterpret_cast<const uint4*>(x0 + e) : uint4{};
            q[s] = in && in1 ? *reinterpret_cast<const uint4*>(x1 + e) : uint4{};
#pragma unroll
            for (int j = 0; j < RS / 8; ++j)
              v[s][j] = in && j * 8 < rc ? *reinterpret_cast<const uint4*>(
                                               w + static_cast<int64_t>(j) * 8 * g.K + e)
                                         : uint4{};
          }
#pragma unroll
          for (int s = 0; s < kUnroll; ++s)
#pragma unroll
            for (int j = 0; j < RS / 8; ++j) {
              mma_16816<T>(acc[j], p[s].x, q[s].x, p[s].y, q[s].y, v[s][j].x, v[s][j].y);
              mma_16816<T>(acc[j], p[s].z, q[s].z, p[s].w, q[s].w, v[s][j].z, v[s][j].w);
            }
        }
        // the parts meet in a fixed order, kSlots at a time
        for (int32_t round = 0; round < kWarps; round += kSlots) {
          const int32_t slot = warp - round;
          if (slot >= 0 && slot < kSlots) {
#pragma unroll
            for (int j = 0; j < RS / 8; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float& f = sums[slot][r0 + (e >> 1) * 8][j * 8 + (lane & 3) * 2 + (e & 1)];
                f = round == 0 ? acc[j][e] : f + acc[j][e];
              }
          }
          __syncthreads();
        }
        if constexpr (kSlots > 1) {
          for (int32_t e = tid; e < have * RS; e += kShrinkThreads) {
            float s = 0.0f;
#pragma unroll
            for (int p = 0; p < kSlots; ++p) s += sums[p][e / RS][e % RS];
            sums[0][e / RS][e % RS] = s;
          }
        }
        if (split > 1)
          cluster_sync();
        else
          __syncthreads();
        for (int32_t v = tid; v < have * (rc / 8); v += kShrinkThreads) {
          const int32_t r = v / (rc / 8), col = v % (rc / 8) * 8;
          if (split > 1 && r % split != kpart) continue;
          float s[8] = {};
          if (split > 1) {
            const uint32_t from = shared_addr(&sums[0][r][col]);
            float4 f[kMaxSplit], h[kMaxSplit];
#pragma unroll
            for (int p = 0; p < kMaxSplit; ++p) {
              f[p] = p < split ? peer_float4(from, p) : float4{};
              h[p] = p < split ? peer_float4(from + 16, p) : float4{};
            }
#pragma unroll
            for (int p = 0; p < kMaxSplit; ++p) {
              s[0] += f[p].x; s[1] += f[p].y; s[2] += f[p].z; s[3] += f[p].w;
              s[4] += h[p].x; s[5] += h[p].y; s[6] += h[p].z; s[7] += h[p].w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = sums[0][r][col + e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] *= scale;
          put_low<T>(g, low, n, list[m0 + r] - b0 * kBlock, c + col, s);
        }
        if (split > 1)
          cluster_sync();
        else
          __syncthreads();
      }
    }
  }
}

// ---------------------------------------------------------------------------
// S of prompts: 128 rows of x by the adapters that they have, up to 128 of their
// ranks at a time, as tcgen05 products whose D holds a row in each lane; a row
// keeps the columns of its own adapter. A cluster splits the inner elements.
// Bound by the loads of x and A and by what they wait for at first: 22 us alone
// for 4096 rows of 8 adapters of rank 64 (45 gathered), 25 at rank 128. Its CTAs
// leave no room for the product's, which begins as they end.

constexpr int kWideRows = 128;
constexpr int kWideRanks = 128;  // columns of D at a time
constexpr int kWideStageBytes = (kWideRows + kWideRanks) * kStepK * 2;
constexpr int kWideStages = 4;
constexpr int kWideBytes =
    kWideStages * kWideStageBytes + kWideRows * (kWideRanks + 4) * 4 + 1024;

struct WideShared {
  Plan plan;
  uint64_t full[kWideStages], empty[kWideStages], done[2], free[2], last;
  uint32_t tmem, failed;
  int32_t who[kWideRows];   // the adapters of these rows
  int32_t count[kWideRows / 32];
  int32_t item[kWideRows];  // of a row
  float scale[kWideRows];
};

template <typename T>
__global__ void __launch_bounds__(kShrinkThreads, 1)
    shrink_wide_kernel(const __grid_constant__ CUtensorMap amap,
                       const __grid_constant__ CUtensorMap xmap, const LoraArgs g,
                       const int32_t split) {
  extern __shared__ uint8_t dynamic[];
  __shared__ WideShared sh;
  const uint32_t ring = (shared_addr(dynamic) + 1023u) & ~1023u;
  const int32_t pitch = g.rank + 4;  // of a row's sums, 16-byte aligned
  const uint32_t sums = ring + kWideStages * kWideStageBytes;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t kpart = blockIdx.x % split, block = blockIdx.x / split;
  const int32_t halves = g.tile / kWideRows, tile = block / halves;
  const int32_t base = block % halves * kWideRows;  // of these rows in their tile
  const int32_t t0 = tile * g.step;
  const int32_t steps = (g.K + kStepK - 1) / kStepK;
  const int32_t s0 = static_cast<int32_t>(static_cast<int64_t>(steps) * kpart / split);
  const int32_t s1 = static_cast<int32_t>(static_cast<int64_t>(steps) * (kpart + 1) / split);
  if (tid == 0) {
    for (int i = 0; i < kWideStages; ++i) {
      bar_init(shared_addr(&sh.full[i]), 1);
      bar_init(shared_addr(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(shared_addr(&sh.done[i]), 1);
      bar_init(shared_addr(&sh.free[i]), 4);
    }
    bar_init(shared_addr(&sh.last), 1);
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     shared_addr(&sh.tmem)),
                 "n"(2 * kWideRanks)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  pdl_trigger();
  int32_t own;
  uint32_t rows_in[8];
  const int32_t total = plan_items(g, t0, sh.plan, own, rows_in);
  if (base == 0 && kpart == 0) {
    if (tid < total) g.items[static_cast<int64_t>(tile) * g.tile + tid] = sh.plan.items[tid];
    if (tid == 0) g.count[tile] = total;
  }
  // the adapters of these rows, in the order of their first rows
  const bool here = tid >= base && tid < base + kWideRows;
  bool lead = here && own >= 0;
  if (lead) {
#pragma unroll
    for (int32_t w = 0; w < 8; ++w) {
      if (w < base / 32) continue;
      if (w < warp) lead = lead && rows_in[w] == 0;
      if (w == warp) lead = lead && (rows_in[w] & ((1u << lane) - 1u)) == 0;
    }
  }
  const uint32_t vote = __ballot_sync(kFull, lead);
  if (here && lane == 0) sh.count[warp - base / 32] = __popc(vote);
  __syncthreads();
  int32_t adapters = 0;
#pragma unroll
  for (int w = 0; w < kWideRows / 32; ++w) adapters += sh.count[w];
  if (lead) {
    int32_t at = __popc(vote & ((1u << lane) - 1u));
    for (int32_t w = 0; w < warp - base / 32; ++w) at += sh.count[w];
    sh.who[at] = own;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  const int32_t most = kWideRanks / g.rank;  // adapters at a time
  const int32_t chunks = (adapters + most - 1) / most;
  // as the product, an fp32 result's sums of 512 inner elements at a time
  const int32_t group = g.fp32 ? kGroup : steps;
  bool ok = true;
  if (warp == 0) {
    int32_t stage = 0, issued = 0;
    uint32_t phase = 0;
    for (int32_t c = 0; c < chunks && ok; ++c) {
      const int32_t n = min(most, adapters - c * most);
      for (int32_t s = s0; s < s1; ++s) {
        ok = __all_sync(kFull, bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1));
        if (!ok) break;
        const uint32_t bar = shared_addr(&sh.full[stage]), at = ring + stage * kWideStageBytes;
        if (lane == 0) {
          bar_expect(bar, kWideRows * kStepK * 2 + n * g.rank * kStepK * 2);
          load_box(at, &xmap, s * kStepK, t0 + base, bar);
        }
        __syncwarp();
        if (lane < n)
          load_box(at + (kWideRows + lane * g.rank) * kStepK * 2, &amap, s * kStepK,
                   sh.who[c * most + lane] * g.rank, bar);
        ++issued;
        if (++stage == kWideStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && lane == 0) {
      sh.failed = 1;
      for (int32_t i = issued - min(issued, kWideStages); i < issued; ++i)
        bar_wait(shared_addr(&sh.full[i % kWideStages]), (i / kWideStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int32_t stage = 0, buffer = 0;
      uint32_t phase = 0, turn = 0;
      for (int32_t c = 0; c < chunks && ok; ++c) {
        const int32_t n = min(most, adapters - c * most);
        for (int32_t s = s0; s < s1; ++s) {
          const bool fresh = (s - s0) % group == 0;
          if (fresh) {
            if (!(ok = bar_wait(shared_addr(&sh.free[buffer]), turn ^ 1))) break;
          }
          if (!(ok = bar_wait(shared_addr(&sh.full[stage]), phase))) break;
          fence_after();
          const uint32_t at = ring + stage * kWideStageBytes;
          const uint64_t xd = desc_swizzled(at), ad = desc_swizzled(at + kWideRows * kStepK * 2);
#pragma unroll
          for (int k = 0; k < kStepK / 16; ++k)
            mma<1>(tmem + buffer * kWideRanks, xd + 2 * k, ad + 2 * k,
                   instruction<T, 1>(0) | (n * g.rank >> 3) << 17, k > 0 || !fresh);
          mma_commit<1>(shared_addr(&sh.empty[stage]));
          if (++stage == kWideStages) {
            stage = 0;
            phase ^= 1;
          }
          if (s + 1 == s1 || (s + 1 - s0) % group == 0) {
            mma_commit<1>(shared_addr(&sh.done[buffer]));
            buffer ^= 1;
            turn ^= buffer == 0;
          }
        }
      }
      if (!ok) {
        sh.failed = 1;
        mma_commit<1>(shared_addr(&sh.last));
        bar_wait(shared_addr(&sh.last), 0);
      }
    }
    __syncwarp();
  } else if (warp < 6) {
    const int32_t quarter = warp & 3, r = quarter * 32 + lane;
    const int32_t a = sh.plan.ids[base + r];
    int32_t slot = -1;
    if (a >= 0) {
      sh.scale[r] = g.scale[a];
      for (int32_t i = 0; i < adapters; ++i)
        if (sh.who[i] == a) slot = i;
      const int32_t at = (base + r) / kBlock;
      for (int32_t i = 0; i < total; ++i) {
        const uint2 item = sh.plan.items[i];
        if (item.x == static_cast<uint32_t>(a) &&
            static_cast<uint32_t>(at) - ((item.y >> 5) & 15u) < (item.y & 31u))
          sh.item[r] = i;
      }
    }
    int32_t buffer = 0;
    uint32_t turn = 0;
    for (int32_t c = 0; c < chunks && ok; ++c) {
      const int32_t n = min(most, adapters - c * most);
      for (int32_t s = s0; s < s1; s += group) {
        ok = __all_sync(kFull, bar_wait(shared_addr(&sh.done[buffer]), turn));
        if (!ok) {
          sh.failed = 1;
          break;
        }
        fence_after();
        for (int32_t i = 0; i < n; ++i) {
          const bool mine = slot == c * most + i;
          if (!__any_sync(kFull, mine)) continue;
          for (int32_t col = 0; col < g.rank; col += 16) {
            uint32_t v[16];
            tmem_load16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buffer * kWideRanks +
                            i * g.rank + col, v);
            if (!mine) continue;
            const uint32_t to = sums + (r * pitch + col) * 4;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              float f[4] = {};
              if (s > s0)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                             : "r"(to + e * 4)
                             : "memory");
              asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + e * 4),
                           "f"(f[0] + __uint_as_float(v[e])), "f"(f[1] + __uint_as_float(v[e + 1])),
                           "f"(f[2] + __uint_as_float(v[e + 2])),
                           "f"(f[3] + __uint_as_float(v[e + 3]))
                           : "memory");
            }
          }
        }
        fence_before();
        if (lane == 0) bar_arrive(shared_addr(&sh.free[buffer]));
        buffer ^= 1;
        turn ^= buffer == 0;
      }
    }
  } else {
    // the rows between an item's, of these 128: a warp takes whole items
    for (int32_t i = kpart * 2 + warp - 6; i < total; i += 2 * split) {
      const uint2 item = sh.plan.items[i];
      const int32_t n = item.y & 31u, b0 = (item.y >> 5) & 15u;
      if (sh.plan.members[i] == n * kBlock) continue;
      uint8_t* low = g.low + (static_cast<int64_t>(tile) * g.most_blocks + (item.y >> 9)) *
                                 (g.rank * g.parts * 32);
      const int32_t from = max(b0 * kBlock, base), to = min((b0 + n) * kBlock, base + kWideRows);
      for (int32_t row = from + lane; row < to; row += 32) {
        if (sh.plan.ids[row] == static_cast<int32_t>(item.x)) continue;
        for (int32_t which = 0; which < g.parts; ++which)
          for (int32_t col = 0; col < g.rank; col += 8)
            *reinterpret_cast<uint4*>(place_of(g, low, n, row - b0 * kBlock, col, which)) = uint4{};
      }
    }
  }
  __syncwarp();
  cluster_sync();
  // this CTA's share of the rows, summed over the cluster in its order
  for (int32_t v = tid; v < kWideRows / split * (g.rank / 8); v += kShrinkThreads) {
    const int32_t r = v / (g.rank / 8) * split + kpart, col = v % (g.rank / 8) * 8;
    const int32_t a = sh.plan.ids[base + r];
    if (a < 0) continue;
    const uint32_t from = sums + (r * pitch + col) * 4;
    float4 f[kMaxSplit], h[kMaxSplit];
#pragma unroll
    for (int p = 0; p < kMaxSplit; ++p) {
      f[p] = p < split ? peer_float4(from, p) : float4{};
      h[p] = p < split ? peer_float4(from + 16, p) : float4{};
    }
    float sum[8] = {};
#pragma unroll
    for (int p = 0; p < kMaxSplit; ++p) {
      sum[0] += f[p].x; sum[1] += f[p].y; sum[2] += f[p].z; sum[3] += f[p].w;
      sum[4] += h[p].x; sum[5] += h[p].y; sum[6] += h[p].z; sum[7] += h[p].w;
    }
    const float scale = sh.scale[r];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] *= scale;
    const uint2 item = sh.plan.items[sh.item[r]];
    uint8_t* low = g.low + (static_cast<int64_t>(tile) * g.most_blocks + (item.y >> 9)) *
                               (g.rank * g.parts * 32);
    put_low<T>(g, low, item.y & 31u, base + r - static_cast<int32_t>((item.y >> 5) & 15u) * kBlock,
               col, sum);
  }
  fence_before();
  cluster_sync();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(2 * kWideRanks));
  }
  if (tid == 0 && sh.failed) atomicExch(&g_error, 1u);
}

// ---------------------------------------------------------------------------
// The product.

template <int NT, int PAIR>
struct Shape {
  static constexpr int kWeightBytes = kTileN * kStepK * 2;
  // a stage holds a step's tiles of W and x, or at least one item of any size
  static constexpr int kStageBytes =
      std::max(kWeightBytes + NT / PAIR * kStepK * 2,
               kRankStep * (kTileN * 2 + NT / PAIR * (NT > 128 ? 4 : 6)));
  // leaves room for a CTA of shrink_kernel on the same SM
  static constexpr int kStages = (200 * 1024) / kStageBytes;
  static constexpr int kColumns = std::max(32, 2 * NT);  // tensor memory: two accumulators
  static constexpr int kBytes = kStages * kStageBytes + 1024;  // with room to align
};

constexpr int kMaxStages = 11;
constexpr uint32_t kEnd = 0;  // an empty step behind the last adapter of a tile

// An item of a step as the matrix instructions take it: operands, first column,
// instruction; how far S goes on for the next 16 inner elements.
struct __align__(16) Op {
  uint64_t b, low;
  uint32_t to, idesc, next, pad;
};

struct ProjectShared {
  uint64_t full[kMaxStages], empty[kMaxStages], done[2], free[2], last;
  uint32_t shape[kMaxStages];   // of an adapters' step: rank step << 8 | items; kEnd
  Op op[kMaxStages][kMaxItems];  // its items
  uint32_t tmem;
  uint32_t failed;
  // the items of the tile of rows, and the steps that they go in
  uint32_t adapter[256];
  uint32_t blocks[256];     // first block of S
  uint32_t plan[256];       // loads B << 31 | B << 20 | S << 9 (places) | first block << 5 | blocks
  uint16_t step[257];       // first item of each step
};

// What the product copies by tensor maps: W, x and, for a pair, B and S as rows
// of kFlatRow bytes. A copy of B has min(kRankStep, rank) inner elements of a tile
// of outputs, or 16 where some step has only that many; one of S has as many of
// 2, 4, 8 or 16 blocks, half of which are this CTA's rows.
constexpr int kFlatRow = 512;
struct ProjectMaps {
  CUtensorMap w, x, b, s[4];
};
__host__ __device__ constexpr int32_t flat_inner(int32_t rank) {
  return rank % kRankStep ? 16 : kRankStep;
}

template <typename T, typename O, int NT, int PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    project_kernel(const __grid_constant__ ProjectMaps maps, const LoraArgs g,
                   const int32_t split) {
  using S = Shape<NT, PAIR>;
  static_assert(S::kStages <= kMaxStages &&
                    (PAIR == 2 || S::kStages * S::kStageBytes >= NT * kTileN * 4),
                "barriers for each stage, room for a tile of sums");
  extern __shared__ uint8_t dynamic[];
  __shared__ ProjectShared sh;
  const uint32_t ring = (shared_addr(dynamic) + 1023u) & ~1023u;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr bool kGroups = std::is_same_v<O, float>;
  const int32_t part = split > 1 ? static_cast<int32_t>(blockIdx.x % split) : 0;
  // A pair has two tiles of outputs side by side, this CTA the cta-th; the first
  // CTA gives the instructions of both.
  const int32_t cta = PAIR == 2 ? static_cast<int32_t>(blockIdx.x & 1u) : 0;
  const int32_t tiles = g.row_tiles * ((g.out_tiles + PAIR - 1) / PAIR);
  const int32_t first = split > 1 ? blockIdx.x / split : blockIdx.x / PAIR;
  const int32_t stride = split > 1 ? tiles : gridDim.x / PAIR;  // a cluster of parts has one tile
  const int32_t steps = (g.K + kStepK - 1) / kStepK;
  const int32_t s0 = static_cast<int32_t>(static_cast<int64_t>(steps) * part / split);
  const int32_t s1 = static_cast<int32_t>(static_cast<int64_t>(steps) * (part + 1) / split);

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      bar_init(shared_addr(&sh.full[i]), 1);
      bar_init(shared_addr(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(shared_addr(&sh.done[i]), 1);
      bar_init(shared_addr(&sh.free[i]), 4 * PAIR);
    }
    bar_init(shared_addr(&sh.last), 1);
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       shared_addr(&sh.tmem)),
                   "n"(S::kColumns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       shared_addr(&sh.tmem)),
                   "n"(S::kColumns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  fence_before();
  __syncthreads();
  if (PAIR == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = sh.tmem;
  bool ok = true;
  // the rows that a tile has, in whole blocks
  auto columns = [&](int32_t rows) {
    return (min(g.step, g.T - rows * g.step) + PAIR * kBlock - 1) / (PAIR * kBlock) *
           (PAIR * kBlock);
  };

  if (warp == 0) {
    // --- loads ---------------------------------------------------------------
    if (!g.ids) pdl_wait();  // else what ran before the first kernel has completed
    bool waited = false;
    int32_t listed = -1, nsteps = 0;
    int32_t stage = 0;
    uint32_t phase = 0;
    int32_t issued = 0;
    auto next = [&] {
      ++issued;
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    };
    for (int32_t tile = first; tile < tiles && ok; tile += stride) {
      const int32_t rows = tile % g.row_tiles, outs = tile / g.row_tiles * PAIR + cta;
      for (int32_t s = s0; s < s1; ++s) {
        ok = __all_sync(kFull, bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1));
        if (!ok) break;
        if (lane == 0) {
          const uint32_t bar = shared_addr(&sh.full[stage]), at = ring + stage * S::kStageBytes;
          if constexpr (PAIR == 1) {
            bar_expect(bar, S::kWeightBytes + g.step * kStepK * 2);
            load_box(at, &maps.w, s * kStepK, outs * kTileN, bar);
            load_box(at + S::kWeightBytes, &maps.x, s * kStepK, rows * g.step, bar);
          } else {
            const uint32_t of_both = in_cta(bar, 0);
            if (cta == 0) bar_expect(bar, 2 * S::kWeightBytes + g.step * kStepK * 2);
            load_box_for(at, &maps.w, s * kStepK, outs * kTileN, of_both);
            load_box_for(at + S::kWeightBytes, &maps.x, s * kStepK,
                         rows * g.step + cta * (columns(rows) / 2), of_both);
          }
        }
        next();
      }
      if (!g.ids || !ok) continue;
      if (!waited) {
        pdl_wait();  // S is there
        waited = true;
      }
      if (listed != rows) {
        // A step takes as many items as fit: the ring is as long as the queue
        // of loads in front of HBM, so a step costs its share of that queue
        // however little it carries (one adapter a step: 0.7 us each). The
        // plan is made once for a tile of rows; places are in units of 32
        // bytes for each inner element of a step.
        listed = rows;
        const int32_t items = min(g.count[rows], NT);
        const int32_t p0 = items * part / split, p1 = items * (part + 1) / split;
        __syncwarp();
        for (int32_t i = p0 + lane; i < p1; i += 32) {
          const uint2 item = g.items[static_cast<int64_t>(rows) * NT + i];
          sh.adapter[i - p0] = item.x;
          sh.blocks[i - p0] = item.y >> 9;
          sh.plan[i - p0] = item.y & 511u;
        }
        __syncwarp();
        const int32_t room = S::kStageBytes / (32 * min(kRankStep, g.rank));
        int32_t n = 0, used = 0, b_at = 0;
        uint32_t last = ~0u;
        nsteps = 0;
        if (lane == 0) {
          for (int32_t i = 0; i < p1 - p0; ++i) {
            const uint32_t a = sh.adapter[i], item = sh.plan[i];
            const int32_t wide = (item & 31u) * g.parts / PAIR;
            if (i == 0 || n == kMaxItems || used + (a == last ? 0 : kTileN / 16) + wide > room) {
              sh.step[nsteps++] = static_cast<uint16_t>(i);
              n = used = 0;
              last = ~0u;
            }
            const bool load = a != last;
            if (load) {
              b_at = used;
              used += kTileN / 16;
            }
            sh.plan[i] = item | static_cast<uint32_t>(load) << 31 |
                         static_cast<uint32_t>(b_at) << 20 | static_cast<uint32_t>(used) << 9;
            used += wide;
            last = a;
            ++n;
          }
          sh.step[nsteps] = static_cast<uint16_t>(p1 - p0);
        }
        nsteps = __shfl_sync(kFull, nsteps, 0);
        __syncwarp();
      }
      // each lane starts the copies of one item
      for (int32_t c = 0; c < g.rank && ok; c += kRankStep) {
        const int32_t rc = min(kRankStep, g.rank - c);
        for (int32_t s = 0; s < nsteps; ++s) {
          const int32_t i0 = sh.step[s], n = sh.step[s + 1] - i0;
          const uint32_t at = ring + stage * S::kStageBytes;
          const uint32_t item = lane < n ? sh.plan[i0 + lane] : 0;
          const uint32_t wide = (item & 31u) * g.parts / PAIR;
          const bool load = item >> 31;
          int32_t units = lane < n ? wide + (load ? kTileN / 16 : 0) : 0;
#pragma unroll
          for (int o = kMaxItems / 2; o > 0; o >>= 1) units += __shfl_xor_sync(kFull, units, o);
          ok = __all_sync(kFull, bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1));
          if (!ok) break;
          const uint32_t blocks = item & 31u;
          const uint32_t bar = shared_addr(&sh.full[stage]);
          if (cta == 0) {  // who gives the instructions
            if (lane < n) {
              Op& op = sh.op[stage][lane];
              op.b = desc_plain(at + ((item >> 20) & 2047u) * rc * 32, kTileN * 16);
              op.low =
                  desc_plain(at + ((item >> 9) & 2047u) * rc * 32, blocks * kBlock * 16 / PAIR);
              op.to = ((item >> 5) & 15u) * kBlock;
              op.idesc = instruction<T, PAIR>(0) | (blocks * (kBlock >> 3)) << 17;
              op.next = blocks * kBlock * 2 / PAIR;
            }
            if (lane == 0)
              sh.shape[stage] = static_cast<uint32_t>(rc) << 8 | static_cast<uint32_t>(n);
            __syncwarp();
            if (lane == 0) bar_expect(bar, PAIR * units * rc * 32);
          }
          __syncwarp();
          if (lane < n) {
            const uint32_t to_b = at + ((item >> 20) & 2047u) * rc * 32;
            uint32_t to_s = at + ((item >> 9) & 2047u) * rc * 32;
            // bytes from the start of B and of S
            const int64_t from_b = ((static_cast<int64_t>(sh.adapter[i0 + lane]) * g.out_tiles +
                                     min(outs, g.out_tiles - 1)) * g.rank + c) * (kTileN * 2);
            const int64_t from_s =
                (static_cast<int64_t>(rows) * g.most_blocks + sh.blocks[i0 + lane]) *
                    (g.rank * g.parts * 32) + wide * (cta * g.rank + c) * 32;
            if constexpr (PAIR == 1) {
              if (load)
                load_bulk(to_b, static_cast<const uint8_t*>(g.b) + from_b, rc * kTileN * 2, bar);
              load_bulk(to_s, g.low + from_s, wide * rc * 32, bar);
            } else {
              const uint32_t of_both = in_cta(bar, 0);
              const int32_t inner = flat_inner(g.rank);
              int32_t row_b = static_cast<int32_t>(from_b / kFlatRow);
              int32_t row_s = static_cast<int32_t>(from_s / kFlatRow);
              for (int32_t k = 0; k < rc; k += inner) {
                if (load) load_box_for(to_b + k * kTileN * 2, &maps.b, 0, row_b, of_both);
                row_b += inner * kTileN * 2 / kFlatRow;
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                  if ((blocks >> (j + 1) & 1u) == 0) continue;
                  load_box_for(to_s, &maps.s[j], 0, row_s, of_both);
                  to_s += (inner * 64) << j;
                  row_s += (inner * 64 / kFlatRow) << j;
                }
              }
            }
          }
          next();
        }
      }
      if (ok) {
        ok = __all_sync(kFull, bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1));
        if (ok) {
          if (lane == 0 && cta == 0) {
            sh.shape[stage] = kEnd;
            bar_arrive(shared_addr(&sh.full[stage]));
          }
          next();
        }
      }
    }
    if (g.ids && !waited) pdl_wait();
    if (PAIR == 2) {  // the pair's instructions are through, and their arrivals here
      for (int i = 0; i < S::kStages && ok; ++i) {
        ok = __all_sync(kFull, bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1));
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && lane == 0) {
      // give up: wait for the copies that are still on their way
      sh.failed = 1;
      if (cta == 0) {
        const int32_t open = min(issued, S::kStages);
        for (int32_t i = issued - open; i < issued; ++i)
          bar_wait(shared_addr(&sh.full[i % S::kStages]), (i / S::kStages) & 1);
      }
    }
  } else if (warp == 1) {
    // --- products ------------------------------------------------------------
    if (lane == 0 && cta == 0) {
      int32_t stage = 0, buffer = 0;
      uint32_t phase = 0, turn = 0;
      for (int32_t tile = first; tile < tiles && ok; tile += stride) {
        if (!(ok = bar_wait_free<PAIR>(shared_addr(&sh.free[buffer]), turn ^ 1))) break;
        fence_after();
        uint32_t d = tmem + buffer * NT;
        const uint32_t wide = instruction<T, PAIR>(columns(tile % g.row_tiles));
        auto finish = [&] {
          mma_commit<PAIR>(shared_addr(&sh.empty[stage]));
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
          }
        };
        for (int32_t s = s0; s < s1; ++s) {
          if (kGroups && s > s0 && (s - s0) % kGroup == 0) {  // the other accumulator
            mma_commit<PAIR>(shared_addr(&sh.done[buffer]));
            buffer ^= 1;
            turn ^= buffer == 0;
            if (!(ok = bar_wait_free<PAIR>(shared_addr(&sh.free[buffer]), turn ^ 1))) break;
            fence_after();
            d = tmem + buffer * NT;
          }
          if (!(ok = bar_wait(shared_addr(&sh.full[stage]), phase))) break;
          fence_after();
          const uint32_t at = ring + stage * S::kStageBytes;
          const uint64_t wd = desc_swizzled(at), xd = desc_swizzled(at + S::kWeightBytes);
#pragma unroll
          for (int k = 0; k < kStepK / 16; ++k)
            mma<PAIR>(d, wd + 2 * k, xd + 2 * k, wide,
                      k > 0 || (kGroups ? (s - s0) % kGroup != 0 : s > s0));
          finish();
        }
        if (!ok) break;
        if (g.ids) {
          for (;;) {
            if (!(ok = bar_wait(shared_addr(&sh.full[stage]), phase))) break;
            fence_after();
            const uint32_t shape = sh.shape[stage];
            if (shape == kEnd) {
              finish();
              break;
            }
            const int32_t rc = shape >> 8, n = shape & 255;
            // One item after the other in a short loop: what this thread does between
            // instructions shows (64 rows by 128,256 to fp32: 205 us, 217 with a
            // branch for each half), and so does going from item to item for each
            // part (24 adapters of rank 64, 256 rows by 65,536: 226 us, 260 to 490).
            const int32_t halves = rc > 16 ? 2 : 1, count = g.parts * halves;
            for (int32_t i = 0; i < n; ++i) {
              Op op = sh.op[stage][i];
              for (int32_t p = 0; p < count; ++p) {
                mma<PAIR>(d + op.to, op.b + (p & (halves - 1)) * (kTileN * 2), op.low, op.idesc,
                          true);
                op.low += op.next;
              }
            }
            finish();
          }
          if (!ok) break;
        }
        mma_commit<PAIR>(shared_addr(&sh.done[buffer]));
        buffer ^= 1;
        turn ^= buffer == 0;
      }
      if (!ok) {
        sh.failed = 1;
        mma_commit_here<PAIR>(shared_addr(&sh.last));
        bar_wait(shared_addr(&sh.last), 0);
      }
    }
    __syncwarp();
  } else {
    // --- results -------------------------------------------------------------
    const int32_t quarter = warp & 3;  // the lanes of tensor memory that this warp may read
    const uint32_t mine = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    using OBits = typename Dt<O>::Bits;
    int32_t buffer = 0;
    uint32_t turn = 0;
    const int32_t groups = kGroups ? (s1 - s0 + kGroup - 1) / kGroup : 1;
    for (int32_t tile = first; tile < tiles && ok; tile += stride) {
      const int32_t rows = tile % g.row_tiles, outs = tile / g.row_tiles * PAIR + cta;
      const int32_t n = outs * kTileN + quarter * 32 + lane;
      OBits* out =
          static_cast<OBits*>(g.out) + static_cast<int64_t>(rows) * g.step * g.out_stride + n;
      const int32_t have = min(g.step, g.T - rows * g.step);
      // 16 rows of the tile: for the cluster's sum, [row][output] in shared memory
      auto put = [&](int32_t c, const float (&v)[16]) {
        if (split > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(
                             ring + ((c + i) * kTileN + quarter * 32 + lane) * 4),
                         "f"(v[i])
                         : "memory");
        } else if (n < g.N) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < have) out[(c + i) * g.out_stride] = Dt<O>::from_float_dev(v[i]);
        }
      };
      float sum[kGroups ? NT / 16 : 1][16];
      for (int32_t group = 0; group < groups; ++group) {
        ok = __all_sync(kFull, bar_wait(shared_addr(&sh.done[buffer]), turn));
        if (!ok) {
          sh.failed = 1;
          break;
        }
        fence_after();
        if constexpr (kGroups) {
#pragma unroll
          for (int c = 0; c < NT; c += 16) {
            if (c >= have) break;
            uint32_t v[16];
            tmem_load16(mine + buffer * NT + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              sum[c / 16][i] =
                  group == 0 ? __uint_as_float(v[i]) : sum[c / 16][i] + __uint_as_float(v[i]);
          }
        } else {
          for (int c = 0; c < have; c += 16) {
            uint32_t v[16];
            tmem_load16(mine + buffer * NT + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[0][i] = __uint_as_float(v[i]);
            put(c, sum[0]);
          }
        }
        fence_before();
        if (lane == 0) {
          if (cta == 0)
            bar_arrive(shared_addr(&sh.free[buffer]));
          else
            bar_arrive_at(shared_addr(&sh.free[buffer]), 0);
        }
        buffer ^= 1;
        turn ^= buffer == 0;
      }
      if constexpr (kGroups) {
        if (ok) {
#pragma unroll
          for (int c = 0; c < NT; c += 16)
            if (c < have) put(c, sum[c / 16]);
        }
      }
    }
  }
  __syncwarp();
  if (PAIR == 2) cluster_sync();  // nothing reads or arrives in the other CTA any more
  if (split > 1) {
    cluster_sync();
    // this CTA's share of the tile's rows, summed over the cluster in its order
    const int32_t rows = first % g.row_tiles, n = first / g.row_tiles * kTileN + lane * 4;
    const int32_t have = min(g.step, g.T - rows * g.step);
    using OBits = typename Dt<O>::Bits;
    OBits* out =
        static_cast<OBits*>(g.out) + static_cast<int64_t>(rows) * g.step * g.out_stride + n;
    for (int32_t r = part + split * warp; r < have; r += split * (kThreads / 32)) {
      float4 v[kMaxSplit];
#pragma unroll
      for (int p = 0; p < kMaxSplit; ++p)
        v[p] = p < split ? peer_float4(ring + (r * kTileN + lane * 4) * 4, p) : float4{};
      float y[4] = {};
#pragma unroll
      for (int p = 0; p < kMaxSplit; ++p) {
        y[0] += v[p].x;
        y[1] += v[p].y;
        y[2] += v[p].z;
        y[3] += v[p].w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < g.N) out[r * g.out_stride + i] = Dt<O>::from_float_dev(y[i]);
    }
    cluster_sync();
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    if constexpr (PAIR == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "n"(S::kColumns));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "n"(S::kColumns));
  }
  if (tid == 0 && sh.failed) atomicExch(&g_error, 1u);
}

// ---------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static std::atomic<EncodeFn> cached{nullptr};
  EncodeFn fn = cached.load(std::memory_order_relaxed);
  if (fn) return fn;
  void* p = nullptr;
  cudaDriverEntryPointQueryResult found;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) !=
          cudaSuccess ||
      found != cudaDriverEntryPointSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  fn = reinterpret_cast<EncodeFn>(p);
  cached.store(fn, std::memory_order_relaxed);
  return fn;
}

// A matrix [rows, cols] of 16-bit elements, read in boxes of `box` rows by 64.
bool matrix_map(CUtensorMap* map, EncodeFn encode, const void* base, bool bf16, int32_t rows,
                int32_t cols, int64_t stride, int32_t box) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t boxes[2] = {kStepK, static_cast<cuuint32_t>(box)}, unit[2] = {1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                const_cast<void*>(base), dims, strides, boxes, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// `rows` rows of kFlatRow bytes each, in boxes of `box` of them.
bool flat_map(CUtensorMap* map, EncodeFn encode, const void* base, int64_t rows, int32_t box) {
  const cuuint64_t dims[2] = {kFlatRow / 2, static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {kFlatRow};
  const cuuint32_t boxes[2] = {kFlatRow / 2, static_cast<cuuint32_t>(box)}, unit[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides,
                boxes, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of x of a tile: all of them where that is one tile, W is then read once.
// (An fp32 result keeps its sums in registers, which hold 128.)
int32_t row_tile(int32_t rows, bool fp32) {
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 || fp32 ? 128 : 256;
}

// Whether two CTAs share the instructions of tiles of 256 rows: each then loads
// half of x, which is most of what an SM loads of them (at 4096 x 65536, 256
// rows: 118 us in pairs, 135 alone; 4096 rows by 8192 outputs: 177, 188). With
// smaller tiles W is most of it, and pairs gain nothing (64 rows, 128,256
// outputs: 172, 169; 128 rows, 65,536 outputs: 102, 103). With adapters, whose
// first steps wait longer in a pair, only where SMs have more than one tile (86
// tiles of outputs, 24 adapters: 54 us in pairs, 48 alone; 512 tiles: 150, 161).
int32_t pair_of(int32_t nt, int64_t tiles, bool adapters) {
  return nt == 256 && tiles * (adapters ? 1 : 2) > sm_count() ? 2 : 1;
}

struct Workspace {
  int32_t most_blocks;
  size_t count, items, low, bytes;
};
Workspace workspace_of(int32_t rows, int32_t rank, int32_t adapters, bool fp32) {
  const int32_t nt = row_tile(rows, fp32);
  const size_t tiles = (static_cast<size_t>(rows) + nt - 1) / nt;
  Workspace w;
  w.most_blocks = std::min<int64_t>(kReach * nt, static_cast<int64_t>(nt / kBlock) *
                                                     std::max(adapters, 1));
  w.count = 0;
  w.items = align256(tiles * sizeof(int32_t));
  w.low = w.items + align256(tiles * nt * sizeof(uint2));
  w.bytes = w.low + align256(tiles * w.most_blocks * rank * 32 * (fp32 ? 3 : 2));
  return w;
}

template <typename T, typename O, int NT, int PAIR>
cudaError_t launch_tile(const ProjectMaps& maps, const LoraArgs& g, cudaStream_t st) {
  static std::atomic<bool> ready[64];
  using S = Shape<NT, PAIR>;
  auto kernel = project_kernel<T, O, NT, PAIR>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             S::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  const int64_t tiles = static_cast<int64_t>(g.row_tiles) * ((g.out_tiles + PAIR - 1) / PAIR);
  const int32_t sms = sm_count(), steps = (g.K + kStepK - 1) / kStepK;
  // Few tiles leave SMs idle: a cluster then shares a tile, each CTA with a
  // part of the inner elements.
  int32_t split = 1;
  while (PAIR == 1 && split < kMaxSplit && tiles * split * 2 <= sms && split * 2 <= steps)
    split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(
      split > 1 ? tiles * split : std::min<int64_t>(tiles, sms / PAIR) * PAIR));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = BPD_PDL ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split * PAIR;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split * PAIR > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, maps, g, split);
}

template <typename T, int RS>
cudaError_t launch_shrink_rank(const LoraArgs& g, int32_t turns, int32_t split, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(g.row_tiles * turns * split));
  cfg.blockDim = dim3(kShrinkThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = BPD_PDL ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  // The largest share of an SM's memory as shared memory, as the product needs
  // it: an SM that is set up otherwise takes none of its CTAs until this
  // kernel's are gone (64 rows, 4096 x 4096: 22 us instead of 17).
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev].load(std::memory_order_relaxed))) {
    e = cudaFuncSetAttribute(shrink_kernel<T, RS>,
                             cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, shrink_kernel<T, RS>, g, turns, split);
}

template <typename T>
cudaError_t launch_shrink_wide(const LoraArgs& g, const CUtensorMap& amap, const CUtensorMap& xmap,
                               cudaStream_t st) {
  static std::atomic<bool> ready[64];
  auto kernel = shrink_wide_kernel<T>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  const int32_t blocks = g.row_tiles * (g.tile / kWideRows), steps = (g.K + kStepK - 1) / kStepK;
  int32_t split = 1;
  while (split < kMaxSplit && blocks * split * 2 <= sm_count() && split * 8 <= steps) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * split));
  cfg.blockDim = dim3(kShrinkThreads);
  cfg.dynamicSmemBytes = kWideBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = BPD_PDL ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, amap, xmap, g, split);
}

template <typename T>
cudaError_t launch_shrink(const LoraArgs& g, cudaStream_t st) {
  // A tile's items go round its CTAs in turn, 16 rows at a time: as many CTAs as
  // that can come to. What is left of the SMs splits the inner elements.
  const int32_t turns = std::min(sm_count() / g.row_tiles,
                                 std::min(g.T, g.adapters + std::min(g.T, g.tile) / 16));
  int32_t split = 1;
  while (split < kMaxSplit && static_cast<int64_t>(g.row_tiles) * turns * split * 2 <= sm_count() &&
         split * 512 <= g.K)
    split *= 2;
  return g.rank <= 16   ? launch_shrink_rank<T, 16>(g, turns, split, st)
         : g.rank <= 32 ? launch_shrink_rank<T, 32>(g, turns, split, st)
                        : launch_shrink_rank<T, 64>(g, turns, split, st);
}

template <typename T, typename O>
cudaError_t launch_project(const ProjectMaps& maps, const CUtensorMap& amap,
                           const CUtensorMap& xrows, const LoraArgs& g, cudaStream_t st) {
  cudaError_t e = !g.ids                       ? cudaSuccess
                  : g.row_tiles > kGatherTiles ? launch_shrink_wide<T>(g, amap, xrows, st)
                                               : launch_shrink<T>(g, st);
  if (e == cudaSuccess) {
    switch (g.tile) {
      case 16: e = launch_tile<T, O, 16, 1>(maps, g, st); break;
      case 32: e = launch_tile<T, O, 32, 1>(maps, g, st); break;
      case 64: e = launch_tile<T, O, 64, 1>(maps, g, st); break;
      case 128: e = launch_tile<T, O, 128, 1>(maps, g, st); break;
      default:  // an fp32 result has tiles of up to 128 rows
        if constexpr (!std::is_same_v<O, float>)
          e = g.pair == 2 ? launch_tile<T, O, 256, 2>(maps, g, st)
                          : launch_tile<T, O, 256, 1>(maps, g, st);
    }
  }
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

extern "C" size_t bpd_lora_workspace_bytes(int32_t rows, int32_t rank, int32_t num_adapters,
                                           int32_t out_dtype) {
  return workspace_of(std::max(rows, 1), std::max(rank, 0), num_adapters, out_dtype == BPD_F32)
      .bytes;
}

extern "C" bpd_status bpd_lora_take_error(int32_t* error_out) {
  BPD_REQUIRE(error_out, "bpd_lora_take_error: null pointer");
  uint32_t v = 0;
  cudaError_t e = cudaDeviceSynchronize();  // streams that do not wait for the default one, too
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_error, sizeof(v));
  const uint32_t zero = 0;
  if (e == cudaSuccess && v) e = cudaMemcpyToSymbol(g_error, &zero, sizeof(zero));
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(BPD_ERR_CUDA, "bpd_lora_take_error: %s", cudaGetErrorString(e));
  }
  *error_out = static_cast<int32_t>(v);
  return BPD_OK;
}

extern "C" bpd_status bpd_lora_project(const void* x, int64_t x_stride, const void* weight,
                                       int64_t weight_stride, int32_t dtype, int32_t rows,
                                       int32_t in_features, int32_t out_features, const void* a,
                                       const void* b, const float* scale, int32_t num_adapters,
                                       int32_t rank, const void* ids, int32_t ids_int64, void* out,
                                       int32_t out_dtype, int64_t out_stride, void* workspace,
                                       void* stream) {
  const char* what = "bpd_lora_project";
  BPD_REQUIRE(rows >= 0 && in_features > 0 && out_features > 0, "%s: bad sizes", what);
  BPD_REQUIRE(dtype == BPD_BF16 || dtype == BPD_F16, "%s: unsupported dtype %d", what, dtype);
  BPD_REQUIRE(out_dtype == dtype || out_dtype == BPD_F32, "%s: unsupported output dtype %d", what,
              out_dtype);
  if (rows == 0) return BPD_OK;
  BPD_REQUIRE(x && weight && out, "%s: null pointer", what);
  BPD_REQUIRE(in_features % 8 == 0, "%s: in_features must be a multiple of 8", what);
  BPD_REQUIRE(aligned16(x) && aligned16(weight) && x_stride % 8 == 0 && weight_stride % 8 == 0,
              "%s: rows of x and weight must start on 16-byte boundaries", what);
  BPD_REQUIRE(x_stride >= in_features && weight_stride >= in_features &&
                  out_stride >= out_features, "%s: row stride too small", what);
  if (ids) {
    BPD_REQUIRE(num_adapters >= 0, "%s: bad sizes", what);
    if (num_adapters == 0) ids = nullptr;
  }
  if (ids) {
    BPD_REQUIRE(a && b && scale && workspace, "%s: null pointer", what);
    BPD_REQUIRE(rank > 0 && rank % 16 == 0 && rank <= BPD_LORA_MAX_RANK,
                "%s: rank must be a multiple of 16, at most %d", what, BPD_LORA_MAX_RANK);
    BPD_REQUIRE(aligned16(a) && aligned16(b) && aligned16(workspace),
                "%s: adapters and workspace must be 16-byte aligned", what);
    if (num_adapters > (1 << 28))
      return fail(BPD_ERR_CAPACITY, "%s: too many adapters", what);
  }
  const bool fp32 = out_dtype == BPD_F32;
  const int32_t nt = row_tile(rows, fp32);
  const int32_t row_tiles = (rows - 1) / nt + 1, out_tiles = (out_features - 1) / kTileN + 1;
  if (static_cast<int64_t>(row_tiles) * out_tiles > INT_MAX / 2)
    return fail(BPD_ERR_CAPACITY, "%s: too many tiles", what);
  // As many rows in every tile, and no more loaded: 300 rows by 4096 x 65,536 with 24
  // adapters take 196 us as 160 and 140 rows, 198 where 256 are loaded for each, and
  // 229 as 256 and 44.
  const int32_t step = std::min(nt, (rows + row_tiles * 32 - 1) / (row_tiles * 32) * 32);
  const Workspace w = workspace_of(rows, rank, num_adapters, fp32);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int32_t parts = fp32 && dtype == BPD_BF16 ? 3 : 2;
  int32_t pair = pair_of(nt, static_cast<int64_t>(row_tiles) * out_tiles, ids != nullptr);
  // rows of B and of S as a pair copies them
  const int64_t flat_b = static_cast<int64_t>(num_adapters) * out_tiles * rank * (kTileN * 2) /
                         kFlatRow;
  const int64_t flat_s = static_cast<int64_t>(row_tiles) * w.most_blocks * rank * parts * 32 /
                         kFlatRow;
  if (ids && std::max(flat_b, flat_s) > INT_MAX) pair = 1;
  const EncodeFn encode = encoder();
  if (!encode) return fail(BPD_ERR_CUDA, "%s: the driver has no tensor maps", what);
  ProjectMaps maps{};
  CUtensorMap amap{}, xrows{};
  const bool bf16 = dtype == BPD_BF16;
  if (!matrix_map(&maps.w, encode, weight, bf16, out_features, in_features, weight_stride, kTileN) ||
      !matrix_map(&maps.x, encode, x, bf16, rows, in_features, x_stride, step / pair))
    return fail(BPD_ERR_INVALID, "%s: strides too large for a tensor map", what);
  if (ids && row_tiles > kGatherTiles) {
    if (static_cast<int64_t>(num_adapters) * rank > INT_MAX)
      return fail(BPD_ERR_CAPACITY, "%s: too many adapters", what);
    if (!matrix_map(&amap, encode, a, bf16, num_adapters * rank, in_features, in_features, rank) ||
        !matrix_map(&xrows, encode, x, bf16, rows, in_features, x_stride, kWideRows))
      return fail(BPD_ERR_INVALID, "%s: strides too large for a tensor map", what);
  }
  if (ids && pair == 2) {
    const int32_t inner = flat_inner(rank);
    bool made = flat_map(&maps.b, encode, b, flat_b, inner * kTileN * 2 / kFlatRow);
    for (int j = 0; j < 4; ++j)
      made = made && flat_map(&maps.s[j], encode, ws + w.low, flat_s, (inner * 64 / kFlatRow) << j);
    if (!made) return fail(BPD_ERR_INVALID, "%s: adapters too large for a tensor map", what);
  }
  const LoraArgs g{x, x_stride, rows, in_features, out_features, a, b, scale, num_adapters, rank,
                   ids, ids_int64, out, out_stride,
                   reinterpret_cast<int32_t*>(ws + w.count),
                   reinterpret_cast<uint2*>(ws + w.items), ws + w.low, nt, step, w.most_blocks,
                   row_tiles,
                   out_tiles, parts, pair, fp32};
  cudaStream_t st = as_stream(stream);
  auto launch = [&](auto in, auto result) {
    return launch_project<decltype(in), decltype(result)>(maps, amap, xrows, g, st);
  };
  const cudaError_t e = bf16 ? fp32 ? launch(__nv_bfloat16{}, float{})
                                    : launch(__nv_bfloat16{}, __nv_bfloat16{})
                        : fp32 ? launch(__half{}, float{})
                               : launch(__half{}, __half{});
  return e == cudaSuccess ? BPD_OK : fail(BPD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
