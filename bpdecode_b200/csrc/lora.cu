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
// S goes into those steps in blocks of 16 rows, the smallest N of the matrix
// unit at M = 128 (of 64 for prompts): a (block, adapter) pair exists only
// where one of the block's rows has that adapter, so there are at most as many
// pairs as rows, whatever their order. Rows need not be sorted.
//
// S is held as the sum of two 16-bit values (its rounding, and what that left
// off): together 2^-17 of it in bf16, 2^-22 in fp16, so an fp32 result keeps
// what fp32 sums have. One 16-bit value would cost 2^-9 of the adapter's part.
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
constexpr int kRankStep = 64;      // inner elements of an adapter's step, at most
constexpr int kMaxPairs = 32;      // pairs of an adapters' step, at most
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
  // workspace: the pairs of each tile of rows, in the order of their adapters
  int32_t* count;    // [row tiles]
  uint32_t* pairs;   // [row tiles, most_pairs]: adapter << 4 | block
  uint8_t* low;      // [row tiles, most_pairs, rank * block * 4 bytes]: S of a pair's rows
  int32_t tile, block;  // rows of a tile and of a block
  int32_t most_pairs;   // of a tile
  int32_t row_tiles, out_tiles;
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
// False where the wait gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  if (bar_try(bar, parity)) return true;
  const uint64_t start = now_ns();
  while (!bar_try(bar, parity))
    if (now_ns() - start > kGiveUpNs) return false;
  return true;
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void load_bulk(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst), "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
      "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
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
// K-major, M = 128.
template <typename T>
constexpr uint32_t instruction(uint32_t n) {
  const uint32_t f = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((n >> 3) << 17) | ((kTileN >> 4) << 24);
}

// ---------------------------------------------------------------------------
// S. A few CTAs for each block of rows share the adapters that the block has:
// BLOCK rows of x by the adapter's A over all inner elements, the warps split
// over 16-row groups and over the inner elements. Bound by the latency of
// reading A, and hidden behind the product's reading of W: a CTA is small
// enough (18 KB of shared memory) to stand beside one of the product's. The
// products go through mma.sync, whose rate is no limit here. The order of the
// inner elements within a step is permuted, alike in both operands, so that
// every load is 16 bytes.

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

// CTAs of a block: as many as it can have adapters, or few where the rows are
// a prompt's and come in runs.
template <int BLOCK>
constexpr int kShrinkCtas = BLOCK == 16 ? 16 : 4;

template <typename T, int BLOCK, int RS>
__global__ void __launch_bounds__(kShrinkThreads, 2) shrink_kernel(const LoraArgs g) {
  using Bits = typename Dt<T>::Bits;
  constexpr int kGroups = BLOCK / 16;                     // 16-row groups of a block
  constexpr int kParts = kShrinkThreads / 32 / kGroups;   // parts of the inner elements
  constexpr int kSlots = std::min(kParts, 4096 / (BLOCK * RS));  // parts that are added at once
  constexpr int kUnroll = RS == 16 ? 4 : RS == 32 ? 3 : 2;
  __shared__ int32_t ids[256];
  __shared__ uint8_t leads[256];
  __shared__ float sums[kSlots][BLOCK][RS];
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t turn = blockIdx.x % kShrinkCtas<BLOCK>;
  const int32_t r0 = blockIdx.x / kShrinkCtas<BLOCK> * BLOCK;  // the block's first row
  const int32_t tile = r0 / g.tile, t0 = tile * g.tile, b0 = r0 - t0;
  pdl_wait();
  pdl_trigger();  // what ran before has completed: x is there for the next kernel, too
  if (tid < g.tile) ids[tid] = adapter_of(g, t0 + tid);
  __syncthreads();
  // the first row of each adapter in its block
  bool lead = tid < g.tile && ids[tid] >= 0;
  if (lead)
    for (int32_t j = tid / BLOCK * BLOCK; j < tid; ++j) lead = lead && ids[j] != ids[tid];
  leads[tid] = lead;
  const int32_t total = __syncthreads_count(lead);
  if (b0 == 0 && turn == 0 && tid == 0) g.count[tile] = total;

  const int32_t group = warp % kGroups, part = warp / kGroups;
  const int32_t i0 = b0 + group * 16 + (lane >> 2);  // this lane's two rows in the tile
  const Bits* x0 = static_cast<const Bits*>(g.x) + static_cast<int64_t>(t0 + i0) * g.x_stride;
  const Bits* x1 = x0 + 8 * g.x_stride;
  // each part is a contiguous share of the inner elements, a multiple of 32
  const int32_t share = ((g.K + 31) / 32 + kParts - 1) / kParts * 32;
  const int32_t k0 = min(g.K, part * share), k1 = min(g.K, k0 + share);
  int32_t seen = 0;
  for (int32_t i = b0; i < b0 + BLOCK; ++i) {
    if (!leads[i] || seen++ % kShrinkCtas<BLOCK> != turn) continue;  // alike in all threads
    const int32_t a = ids[i];
    const int32_t at_pair = __syncthreads_count(
        lead && (ids[tid] < a || (ids[tid] == a && tid / BLOCK < b0 / BLOCK)));
    const int64_t pair = static_cast<int64_t>(tile) * g.most_pairs + at_pair;
    if (tid == 0)
      g.pairs[pair] = (static_cast<uint32_t>(a) << 4) | static_cast<uint32_t>(b0 / BLOCK);
    const bool in0 = ids[i0] == a, in1 = ids[i0 + 8] == a;
    const float scale = g.scale[a];
    for (int32_t c = 0; c < g.rank; c += RS) {
      const int32_t rc = min(RS, g.rank - c);
      const Bits* w = static_cast<const Bits*>(g.a) +
                      (static_cast<int64_t>(a) * g.rank + c + (lane >> 2)) * g.K;
      float acc[RS / 8][4] = {};
      for (int32_t k = k0; k < k1; k += 32 * kUnroll) {
        uint4 u[kUnroll], v[kUnroll], q[kUnroll][RS / 8];
#pragma unroll
        for (int s = 0; s < kUnroll; ++s) {
          const int32_t at = k + s * 32 + (lane & 3) * 8;
          const bool in = at < k1;
          u[s] = in && in0 ? *reinterpret_cast<const uint4*>(x0 + at) : uint4{};
          v[s] = in && in1 ? *reinterpret_cast<const uint4*>(x1 + at) : uint4{};
#pragma unroll
          for (int j = 0; j < RS / 8; ++j)
            q[s][j] = in && j * 8 < rc
                          ? *reinterpret_cast<const uint4*>(w + static_cast<int64_t>(j) * 8 * g.K + at)
                          : uint4{};
        }
#pragma unroll
        for (int s = 0; s < kUnroll; ++s)
#pragma unroll
          for (int j = 0; j < RS / 8; ++j) {
            mma_16816<T>(acc[j], u[s].x, v[s].x, u[s].y, v[s].y, q[s][j].x, q[s][j].y);
            mma_16816<T>(acc[j], u[s].z, v[s].z, u[s].w, v[s].w, q[s][j].z, q[s][j].w);
          }
      }
      // the parts meet in a fixed order, kSlots at a time
      for (int32_t round = 0; round < kParts; round += kSlots) {
        if (part >= round && part < round + kSlots) {
          float(*to)[RS] = sums[part - round];
          const int32_t row = group * 16 + (lane >> 2);
#pragma unroll
          for (int j = 0; j < RS / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& f = to[row + (e >> 1) * 8][j * 8 + (lane & 3) * 2 + (e & 1)];
              f = round == 0 ? acc[j][e] : f + acc[j][e];
            }
        }
        __syncthreads();
      }
      // the operand's layout: [rank / 8][rows][8], first the rounded values, then the rests
      Bits* low = reinterpret_cast<Bits*>(g.low + (pair * g.rank + c) * (BLOCK * 4));
      for (int32_t e = tid; e < BLOCK * rc; e += kShrinkThreads) {
        const int32_t row = (e >> 3) % BLOCK, col = e / (8 * BLOCK) * 8 + (e & 7);
        float s = 0.0f;
#pragma unroll
        for (int p = 0; p < kSlots; ++p) s += sums[p][row][col];
        s = ids[b0 + row] == a ? s * scale : 0.0f;
        const Bits hi = Dt<T>::from_float_dev(s);
        low[e] = hi;
        low[BLOCK * rc + e] = Dt<T>::from_float_dev(s - Dt<T>::to_float(hi));
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// The product.

template <int NT, int BLOCK>
struct Shape {
  static constexpr int kWeightBytes = kTileN * kStepK * 2;
  // a stage holds a step's rows of x, or the pairs of an adapter's step
  static constexpr int kRowBytes = std::max(NT * kStepK * 2, BLOCK * kRankStep * 4);
  static constexpr int kStageBytes = kWeightBytes + kRowBytes;
  // leaves room for a CTA of shrink_kernel on the same SM
  static constexpr int kStages = (200 * 1024) / kStageBytes;
  static constexpr int kColumns = std::max(32, 2 * NT);  // tensor memory: two accumulators
  static constexpr int kBytes = kStages * kStageBytes + 1024;  // with room to align
};

constexpr int kMaxStages = 10;
constexpr uint32_t kEnd = 0;  // an empty step behind the last adapter of a tile

struct ProjectShared {
  uint64_t full[kMaxStages], empty[kMaxStages], done[2], free[2], last;
  uint32_t shape[kMaxStages];   // of an adapters' step: rank step << 8 | pairs; kEnd
  uint8_t pair[kMaxStages][kMaxPairs];  // its pairs: adapter of the step << 4 | block
  uint32_t tmem;
  uint32_t failed;
  uint32_t list[256];
};

template <typename T, typename O, int NT, int BLOCK>
__global__ void __launch_bounds__(kThreads, 1)
    project_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                   const LoraArgs g, const int32_t split) {
  using S = Shape<NT, BLOCK>;
  extern __shared__ uint8_t dynamic[];
  __shared__ ProjectShared sh;
  const uint32_t ring = (shared_addr(dynamic) + 1023u) & ~1023u;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t part = split > 1 ? static_cast<int32_t>(blockIdx.x % split) : 0;
  const int32_t tiles = g.row_tiles * g.out_tiles;
  const int32_t first = split > 1 ? blockIdx.x / split : blockIdx.x;
  const int32_t stride = split > 1 ? tiles : gridDim.x;  // a cluster has one tile
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
      bar_init(shared_addr(&sh.free[i]), 4);
    }
    bar_init(shared_addr(&sh.last), 1);
    sh.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     shared_addr(&sh.tmem)),
                 "n"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  bool ok = true;

  if (warp == 0) {
    // --- loads ---------------------------------------------------------------
    if (!g.ids) pdl_wait();  // else what ran before the first kernel has completed
    bool waited = false;
    int32_t listed = -1, pairs = 0;
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
      const int32_t rows = tile % g.row_tiles, outs = tile / g.row_tiles;
      if (lane == 0) {
        for (int32_t s = s0; s < s1; ++s) {
          if (!(ok = bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1))) break;
          const uint32_t bar = shared_addr(&sh.full[stage]), at = ring + stage * S::kStageBytes;
          bar_expect(bar, S::kWeightBytes + NT * kStepK * 2);
          load_box(at, &wmap, s * kStepK, outs * kTileN, bar);
          load_box(at + S::kWeightBytes, &xmap, s * kStepK, rows * NT, bar);
          next();
        }
      }
      ok = __shfl_sync(kFull, ok, 0);
      if (!g.ids || !ok) continue;
      if (!waited) {
        pdl_wait();  // S is there
        waited = true;
      }
      if (listed != rows) {
        pairs = min(g.count[rows], g.most_pairs);
        __syncwarp();
        for (int32_t i = lane; i < pairs; i += 32)
          sh.list[i] = g.pairs[static_cast<int64_t>(rows) * g.most_pairs + i];
        __syncwarp();
        listed = rows;
      }
      if (lane == 0) {
        // A step takes as many pairs as fit: the ring is as long as the queue
        // of loads in front of HBM, so a step costs its share of that queue
        // however little it carries (one adapter a step: 0.7 us each).
        const int32_t p0 = pairs * part / split, p1 = pairs * (part + 1) / split;
        for (int32_t c = 0; c < g.rank && ok; c += kRankStep) {
          const int32_t rc = min(kRankStep, g.rank - c);
          const int32_t adapters = kRankStep / rc;
          const int32_t most = min(kMaxPairs, S::kRowBytes / (rc * BLOCK * 4));
          for (int32_t p = p0; p < p1;) {
            if (!(ok = bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1))) break;
            const uint32_t bar = shared_addr(&sh.full[stage]), at = ring + stage * S::kStageBytes;
            int32_t n = 0, met = 0;
            uint32_t last = 0;
            for (; n < most && p + n < p1; ++n) {
              const uint32_t pair = sh.list[p + n], a = pair >> 4;
              if (met == 0 || a != last) {
                if (met == adapters) break;
                ++met;
                last = a;
              }
              sh.pair[stage][n] = static_cast<uint8_t>((met - 1) << 4 | (pair & 15u));
            }
            sh.shape[stage] = static_cast<uint32_t>(rc) << 8 | static_cast<uint32_t>(n);
            bar_expect(bar, met * rc * kTileN * 2 + n * rc * BLOCK * 4);
            for (int32_t i = 0, m = -1; i < n; ++i) {
              const uint32_t a = sh.list[p + i] >> 4;
              if (i == 0 || a != last) {
                last = a;
                load_bulk(at + ++m * rc * kTileN * 2,
                          static_cast<const uint8_t*>(g.b) +
                              ((static_cast<int64_t>(a) * g.out_tiles + outs) * g.rank + c) *
                                  (kTileN * 2),
                          rc * kTileN * 2, bar);
              }
              // pairs that follow one another in memory, too, where rank is one step
              if (rc != g.rank)
                load_bulk(at + S::kWeightBytes + i * rc * BLOCK * 4,
                          g.low + ((static_cast<int64_t>(rows) * g.most_pairs + p + i) * g.rank + c) *
                                      (BLOCK * 4),
                          rc * BLOCK * 4, bar);
            }
            if (rc == g.rank)
              load_bulk(at + S::kWeightBytes,
                        g.low + (static_cast<int64_t>(rows) * g.most_pairs + p) * g.rank *
                                    (BLOCK * 4),
                        n * rc * BLOCK * 4, bar);
            next();
            p += n;
          }
        }
        if (ok && (ok = bar_wait(shared_addr(&sh.empty[stage]), phase ^ 1))) {
          sh.shape[stage] = kEnd;
          bar_arrive(shared_addr(&sh.full[stage]));
          next();
        }
      }
      ok = __shfl_sync(kFull, ok, 0);
    }
    if (g.ids && !waited) pdl_wait();
    if (!ok && lane == 0) {
      // give up: wait for the copies that are still on their way
      sh.failed = 1;
      const int32_t open = min(issued, S::kStages);
      for (int32_t i = issued - open; i < issued; ++i)
        bar_wait(shared_addr(&sh.full[i % S::kStages]), (i / S::kStages) & 1);
    }
  } else if (warp == 1) {
    // --- products ------------------------------------------------------------
    if (lane == 0) {
      int32_t stage = 0, buffer = 0;
      uint32_t phase = 0, turn = 0;
      for (int32_t tile = first; tile < tiles && ok; tile += stride) {
        if (!(ok = bar_wait(shared_addr(&sh.free[buffer]), turn ^ 1))) break;
        fence_after();
        const uint32_t d = tmem + buffer * NT;
        auto finish = [&] {
          mma_commit(shared_addr(&sh.empty[stage]));
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
          }
        };
        for (int32_t s = s0; s < s1; ++s) {
          if (!(ok = bar_wait(shared_addr(&sh.full[stage]), phase))) break;
          fence_after();
          const uint32_t at = ring + stage * S::kStageBytes;
          const uint64_t wd = desc_swizzled(at), xd = desc_swizzled(at + S::kWeightBytes);
#pragma unroll
          for (int k = 0; k < kStepK / 16; ++k)
            mma(d, wd + 2 * k, xd + 2 * k, instruction<T>(NT), s > s0 || k > 0);
          finish();
        }
        if (!ok) break;
        if (g.ids) {
          for (;;) {
            if (!(ok = bar_wait(shared_addr(&sh.full[stage]), phase))) break;
            fence_after();
            const uint32_t at = ring + stage * S::kStageBytes;
            const uint32_t shape = sh.shape[stage];
            if (shape == kEnd) {
              finish();
              break;
            }
            const int32_t rc = shape >> 8, n = shape & 255;
            for (int32_t i = 0; i < n; ++i) {
              const uint32_t pair = sh.pair[stage][i];
              const uint32_t to = d + (pair & 15u) * BLOCK;
              const uint32_t b = at + (pair >> 4) * rc * kTileN * 2;
              const uint32_t low = at + S::kWeightBytes + i * rc * BLOCK * 4;
              for (int32_t half = 0; half < 2; ++half)
                for (int32_t k = 0; k < rc; k += 16)
                  mma(to, desc_plain(b + k * kTileN * 2, kTileN * 16),
                      desc_plain(low + half * rc * BLOCK * 2 + k * BLOCK * 2, BLOCK * 16),
                      instruction<T>(BLOCK), true);
            }
            finish();
          }
          if (!ok) break;
        }
        mma_commit(shared_addr(&sh.done[buffer]));
        buffer ^= 1;
        turn ^= buffer == 0;
      }
      if (!ok) {
        sh.failed = 1;
        mma_commit(shared_addr(&sh.last));
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
    for (int32_t tile = first; tile < tiles; tile += stride) {
      const int32_t rows = tile % g.row_tiles, outs = tile / g.row_tiles;
      ok = bar_wait(shared_addr(&sh.done[buffer]), turn);
      if (!__all_sync(kFull, ok)) {
        ok = false;
        sh.failed = 1;
        break;
      }
      fence_after();
      const int32_t n = outs * kTileN + quarter * 32 + lane;
      OBits* out = static_cast<OBits*>(g.out) + static_cast<int64_t>(rows) * NT * g.out_stride + n;
      const int32_t have = min(NT, g.T - rows * NT);
      for (int32_t c = 0; c < NT; c += 16) {
        uint32_t v[16];
        tmem_load16(mine + buffer * NT + c, v);
        if (split > 1) {
          // [row][output] in shared memory, for the cluster's sum
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(
                             ring + ((c + i) * kTileN + quarter * 32 + lane) * 4),
                         "r"(v[i])
                         : "memory");
        } else if (n < g.N) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < have)
              out[(c + i) * g.out_stride] = Dt<O>::from_float_dev(__uint_as_float(v[i]));
        }
      }
      fence_before();
      if (lane == 0) bar_arrive(shared_addr(&sh.free[buffer]));
      buffer ^= 1;
      turn ^= buffer == 0;
    }
  }
  __syncwarp();
  if (split > 1) {
    cluster_sync();
    // this CTA's share of the tile's rows, summed over the cluster in its order
    const int32_t rows = first % g.row_tiles, n = first / g.row_tiles * kTileN + lane * 4;
    const int32_t have = min(NT, g.T - rows * NT);
    using OBits = typename Dt<O>::Bits;
    OBits* out = static_cast<OBits*>(g.out) + static_cast<int64_t>(rows) * NT * g.out_stride + n;
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
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

// Rows of x of a tile: all of them where that is one tile, W is then read once.
int32_t row_tile(int32_t rows) {
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
}

// Rows of a pair. Wide ones need fewer, fuller matrix instructions (a prompt's
// rows come in runs of one adapter); narrow ones carry fewer zeros where every
// row may have an adapter of its own, as in a batch of single tokens.
int32_t block_of(int32_t rows, int32_t adapters) { return rows > 256 && adapters <= 64 ? 64 : 16; }

struct Workspace {
  int32_t block, most_pairs;
  size_t count, pairs, low, bytes;
};
Workspace workspace_of(int32_t rows, int32_t rank, int32_t adapters) {
  const int32_t nt = row_tile(rows);
  const size_t tiles = (static_cast<size_t>(rows) + nt - 1) / nt;
  Workspace w;
  w.block = block_of(rows, adapters);
  w.most_pairs = nt / w.block * std::min(w.block, std::max(adapters, 1));
  w.count = 0;
  w.pairs = align256(tiles * sizeof(int32_t));
  w.low = w.pairs + align256(tiles * w.most_pairs * sizeof(uint32_t));
  w.bytes = w.low + align256(tiles * w.most_pairs * rank * w.block * 4);
  return w;
}

template <typename T, typename O, int NT, int BLOCK>
cudaError_t launch_tile(const CUtensorMap& wmap, const CUtensorMap& xmap, const LoraArgs& g,
                        cudaStream_t st) {
  static std::atomic<bool> ready[64];
  auto kernel = project_kernel<T, O, NT, BLOCK>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Shape<NT, BLOCK>::kBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  const int64_t tiles = static_cast<int64_t>(g.row_tiles) * g.out_tiles;
  const int32_t sms = sm_count(), steps = (g.K + kStepK - 1) / kStepK;
  // Few tiles leave SMs idle: a cluster then shares a tile, each CTA with a
  // part of the inner elements.
  int32_t split = 1;
  while (split < kMaxSplit && tiles * split * 2 <= sms && split * 2 <= steps) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(split > 1 ? tiles * split
                                                     : std::min<int64_t>(tiles, sms)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Shape<NT, BLOCK>::kBytes;
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
  return cudaLaunchKernelEx(&cfg, kernel, wmap, xmap, g, split);
}

template <typename T, int BLOCK>
cudaError_t launch_shrink(const LoraArgs& g, cudaStream_t st) {
  const dim3 grid((g.T + BLOCK - 1) / BLOCK * kShrinkCtas<BLOCK>), block(kShrinkThreads);
  return g.rank <= 16   ? launch_pdl(shrink_kernel<T, BLOCK, 16>, grid, block, 0, st, g)
         : g.rank <= 32 ? launch_pdl(shrink_kernel<T, BLOCK, 32>, grid, block, 0, st, g)
                        : launch_pdl(shrink_kernel<T, BLOCK, 64>, grid, block, 0, st, g);
}

template <typename T, typename O>
cudaError_t launch_project(const CUtensorMap& wmap, const CUtensorMap& xmap, const LoraArgs& g,
                           cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (g.ids) e = g.block == 64 ? launch_shrink<T, 64>(g, st) : launch_shrink<T, 16>(g, st);
  if (e != cudaSuccess) return e;
  switch (g.tile) {
    case 16: e = launch_tile<T, O, 16, 16>(wmap, xmap, g, st); break;
    case 32: e = launch_tile<T, O, 32, 16>(wmap, xmap, g, st); break;
    case 64: e = launch_tile<T, O, 64, 16>(wmap, xmap, g, st); break;
    case 128: e = launch_tile<T, O, 128, 16>(wmap, xmap, g, st); break;
    default:
      e = g.block == 64 ? launch_tile<T, O, 256, 64>(wmap, xmap, g, st)
                        : launch_tile<T, O, 256, 16>(wmap, xmap, g, st);
  }
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

extern "C" size_t bpd_lora_workspace_bytes(int32_t rows, int32_t rank, int32_t num_adapters) {
  return workspace_of(std::max(rows, 1), std::max(rank, 0), num_adapters).bytes;
}

extern "C" bpd_status bpd_lora_take_error(int32_t* error_out) {
  BPD_REQUIRE(error_out, "bpd_lora_take_error: null pointer");
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_error, sizeof(v));
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
  const int32_t nt = row_tile(rows);
  const int32_t row_tiles = (rows - 1) / nt + 1, out_tiles = (out_features - 1) / kTileN + 1;
  if (static_cast<int64_t>(row_tiles) * out_tiles > INT_MAX / 2)
    return fail(BPD_ERR_CAPACITY, "%s: too many tiles", what);
  const EncodeFn encode = encoder();
  if (!encode) return fail(BPD_ERR_CUDA, "%s: the driver has no tensor maps", what);
  CUtensorMap wmap, xmap;
  const bool bf16 = dtype == BPD_BF16;
  if (!matrix_map(&wmap, encode, weight, bf16, out_features, in_features, weight_stride, kTileN) ||
      !matrix_map(&xmap, encode, x, bf16, rows, in_features, x_stride, nt))
    return fail(BPD_ERR_INVALID, "%s: strides too large for a tensor map", what);
  const Workspace w = workspace_of(rows, rank, num_adapters);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const LoraArgs g{x, x_stride, rows, in_features, out_features, a, b, scale, num_adapters, rank,
                   ids, ids_int64, out, out_stride,
                   reinterpret_cast<int32_t*>(ws + w.count),
                   reinterpret_cast<uint32_t*>(ws + w.pairs), ws + w.low, nt, w.block,
                   w.most_pairs, row_tiles, out_tiles};
  cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (bf16)
    e = out_dtype == BPD_F32 ? launch_project<__nv_bfloat16, float>(wmap, xmap, g, st)
                             : launch_project<__nv_bfloat16, __nv_bfloat16>(wmap, xmap, g, st);
  else
    e = out_dtype == BPD_F32 ? launch_project<__half, float>(wmap, xmap, g, st)
                             : launch_project<__half, __half>(wmap, xmap, g, st);
  return e == cudaSuccess ? BPD_OK : fail(BPD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
