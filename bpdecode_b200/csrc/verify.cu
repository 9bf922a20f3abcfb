// Verification of drafted tokens against the target's probabilities, from
// random numbers that the caller gives, under each request's grammar.
//
// Request b brings len drafts d_0 .. d_{len-1} and len + 1 rows of logits x_i.
// Row i is masked by the allow bits of the state that the first i drafts lead
// to. With m = max x_i, w = exp((x_i - m) / T), Z = sum w and p = w / Z:
//
//   accept d_i             iff  u_i * q_i[d_i] < p[d_i]
//   the first not accepted: argmax over t of max(p[t] - q_i[t], 0) / e[t]
//   none left (i == len):   argmax over t of p[t] / e[t]
//
// where e is exponential noise (argmax of p / e is a draw from p: the first of
// independent exponential clocks with rates p) and q_i the distribution that
// draft i was drawn from; without probabilities q_i is all on d_i. T <= 0 is
// greedy: d_i is accepted iff it is the first maximal token, which also
// replaces it.
//
// One cluster of CTAs works through one request, position after position, so
// rows behind the first refused draft are never read. Each CTA scans a slice
// of the row once in 16-byte vectors, with a running maximum and sum, leaving
// out vectors whose tokens are all rejected; the slices' (m, argmax, s) meet
// through distributed shared memory in a fixed order, so a result does not
// depend on timing. Behind the last draft the race runs in that same pass, on
// x / T - log e, which needs neither m nor Z. A row whose draft was refused is
// scanned a second time (from L2) with the noise and the draft's
// probabilities. What a thread finds best is then scored again with full
// precision, so that only scores within one thread are compared in fast
// arithmetic.
#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"

namespace bpd {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxCluster = 8;
// Bytes of shared memory for each thread's loads on their way: eight vectors of
// logits, or four with their noise, or two with noise and probabilities.
constexpr int kRingBytes = 192;
#ifndef LB
#define LB 4
#endif
constexpr int kCtasPerSm = LB;
constexpr float kLog2e = 1.4426950408889634f;

struct VerifyArgs {
  const void* src;
  int64_t src_stride, src_total;
  const int64_t* src_rows;
  const void* drafts;
  int64_t draft_stride;
  int32_t drafts64;
  const int32_t* lens;
  const void* probs;
  int32_t probs_dtype;
  int64_t probs_stride, probs_total;
  const int64_t* prob_rows;
  const float* uniforms;
  int64_t uniform_stride;
  const float* noise;
  int64_t noise_stride;
  const float* temperature;
  float temperature_all;
  int32_t batch, K, V;
  int32_t* pool;
  const int64_t* slots;
  const int32_t* path;
  const uint32_t* bits;
  int32_t wstride;
  const int32_t* tok_next;
  int32_t num_states;
  int64_t* tokens;
  int32_t* counts;
  float* logprobs;
  int32_t* next_out;
  int32_t write_back;
  int32_t window;  // positions that are scanned before the cluster meets
};

// What a slice of a row comes to: its maximum, the first index that has it
// (-1: nothing allowed), and the sum of exp((x - m) / T).
struct Slice {
  float m;
  int32_t idx;
  float s;
};

// A position: what its decision needs, and what came of it.
struct Position {
  float xd, qd, uniform;  // the draft's logit (-inf: rejected) and probability
  int32_t draft;          // -1: none, or no token of the vocabulary
  float m, s;             // the whole row's
  int32_t idx, accept;
};

struct Shared {
  uint4 lanes[256];  // for each byte of allow bits, the 16-bit lanes that it keeps
  uint64_t warp_key[kVerifyWarps];
  float warp_sum[kVerifyWarps];
  uint64_t race[2];  // of two races in turn
  uint32_t bar;      // of a race: what no thread needs to look below
  Slice slice[BPD_MAX_DRAFTS + 1];
  Position position[BPD_MAX_DRAFTS + 1];
  int32_t state[BPD_MAX_DRAFTS + 1];
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// A barrier over the cluster's threads (over the CTA's where it has one CTA).
template <int C>
__device__ __forceinline__ void cluster_barrier() {
  if constexpr (C == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  }
}

// The address of `p` (this CTA's shared memory) in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t peer_shared(const void* p, uint32_t rank) {
  uint32_t a;
  const uint32_t own = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(own), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t peer_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t peer_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// The inverse of order_key.
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's allow bits: every token (no grammar), a row of bits, or nothing.
struct Allow {
  const uint32_t* row;  // NULL: see `any`
  bool any;
  __device__ __forceinline__ bool has(int32_t t) const {
    return row ? ((__ldg(row + (t >> 5)) >> (t & 31)) & 1u) : any;
  }
  // the bits of N tokens from t on, all of them inside the vocabulary
  template <int N>
  __device__ __forceinline__ uint32_t bits(int32_t t) const {
    constexpr uint32_t all = (1u << N) - 1u;
    if (!row) return any ? all : 0u;
    const int32_t w = t >> 5, sh = t & 31;
    const uint32_t lo = __ldg(row + w), hi = sh + N > 32 ? __ldg(row + w + 1) : 0u;
    return __funnelshift_r(lo, hi, sh) & all;
  }
};

// A row of logits as 16-byte vectors: `head` tokens, `vecs` vectors, a tail.
template <typename T>
struct Row {
  static constexpr int kEpv = Dt<T>::kPerVec;
  using Bits = typename Dt<T>::Bits;
  const Bits* p;
  int32_t head, vecs, V;
  __device__ Row(const void* row, int32_t V_) : p(static_cast<const Bits*>(row)), V(V_) {
    const uintptr_t off = reinterpret_cast<uintptr_t>(row) & 15u;
    head = min(V, static_cast<int32_t>((16u - off) & 15u) / static_cast<int32_t>(sizeof(Bits)));
    vecs = (V - head) / kEpv;
  }
  __device__ __forceinline__ float at(int64_t t) const { return Dt<T>::to_float(p[t]); }
  __device__ __forceinline__ int32_t token(int32_t vec) const { return head + vec * kEpv; }
  __device__ __forceinline__ const Bits* vec_at(int32_t j) const { return p + token(j); }
  // the token outside the vectors that this thread looks at, or -1
  __device__ __forceinline__ int32_t edge(bool first, bool last) const {
    const int32_t i = threadIdx.x, tail = head + vecs * kEpv;
    if (first && i < head) return i;
    if (last && i >= 32 && i - 32 < V - tail) return tail + i - 32;
    return -1;
  }
};

// exp((x - m) / T) where x is not NaN and m the row's maximum: 1 at the
// maximum itself, which may be +inf, 0 at -inf.
__device__ __forceinline__ float weight(float x, float m, float inv) {
  if (x == m) return 1.0f;
  return x > -INFINITY ? expf((x - m) * inv) : 0.0f;
}

template <typename T>
__device__ __forceinline__ float load_logit(const void* row, int64_t t) {
  return Dt<T>::to_float(static_cast<const typename Dt<T>::Bits*>(row)[t]);
}

__device__ __forceinline__ float load_prob(const void* row, int32_t dtype, int64_t t) {
  if (dtype == BPD_F32) return static_cast<const float*>(row)[t];
  if (dtype == BPD_BF16) return load_logit<__nv_bfloat16>(row, t);
  return load_logit<__half>(row, t);
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ uint4 shared_vec(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

// This thread's places in the ring: 16 bytes beside its neighbours'.
constexpr uint32_t kPlane = kVerifyThreads * 16;

// N consecutive floats from p on, to the planes from `dst` on.
template <int N>
__device__ __forceinline__ void copy_floats(uint32_t dst, const float* p, bool aligned) {
  if (aligned) {
#pragma unroll
    for (int i = 0; i < N; i += 4) copy_async<16>(dst + i / 4 * kPlane, p + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) copy_async<4>(dst + i / 4 * kPlane + i % 4 * 4, p + i);
  }
}
template <int N>
__device__ __forceinline__ void read_floats(uint32_t src, float (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint4 v = shared_vec(src + i / 4 * kPlane);
    out[i] = __uint_as_float(v.x);
    out[i + 1] = __uint_as_float(v.y);
    out[i + 2] = __uint_as_float(v.z);
    out[i + 3] = __uint_as_float(v.w);
  }
}

// A row of the draft's probabilities (p == NULL: none).
struct Given {
  const void* p;
  int32_t dtype;
  bool aligned;  // its vectors begin where the logits' do, on as many bytes as a copy has
  // N probabilities from token t on, on their way to the planes from dst on
  // (fp32: always; 16 bits: where aligned)
  template <int N>
  __device__ __forceinline__ void copy(uint32_t dst, int32_t t) const {
    if (!p) return;
    if (dtype == BPD_F32)
      copy_floats<N>(dst, static_cast<const float*>(p) + t, aligned);
    else if (aligned)
      copy_async<N * 2>(dst, static_cast<const uint16_t*>(p) + t);
  }
  template <int N>
  __device__ __forceinline__ void read(uint32_t src, int32_t t, float (&out)[N]) const {
    if (!p) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = 0.0f;
      return;
    }
    if (dtype == BPD_F32) {
      read_floats<N>(src, out);
      return;
    }
    uint32_t w[N / 2];
    if (aligned) {
      const uint4 v = shared_vec(src);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = vec_word(v, i);
    } else {
      const uint16_t* h = static_cast<const uint16_t*>(p) + t;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        w[i] = __ldg(h + 2 * i) | static_cast<uint32_t>(__ldg(h + 2 * i + 1)) << 16;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint16_t u = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
      out[i] = dtype == BPD_BF16 ? Dt<__nv_bfloat16>::to_float(u) : Dt<__half>::to_float(u);
    }
  }
};

// A warp's share of a row: every `step`-th block of 128 vectors from `first` on.
struct Share {
  int32_t first, step;
  bool head, tail;  // whether this CTA looks at the tokens before, behind the vectors
};
constexpr int kRounds = 4;  // of a warp in a block, a vector for each lane

// Streams a warp's share of a row through shared memory, DEPTH vectors on
// their way for each thread at any time: start(slot, vector) begins the copies
// of a vector that keeps a token, use(slot, vector, keep) takes it (also where
// none is kept and nothing was copied). Registers
// hold none of what is on its way (kept in registers, two rounds ahead, the
// same loop ran at a third of the rate). A lane reads 32 allow bits of a block,
// a block ahead of the copies, and the others take theirs from it. A thread
// reads what it copied itself, so there is no barrier.
template <typename T, int DEPTH, typename Start, typename Use>
__device__ __forceinline__ void stream(const Row<T>& row, const Allow& ok, const Share& share,
                                       Start&& start, Use&& use) {
  constexpr int kEpv = Row<T>::kEpv;
  constexpr int kLanes = 32 / kEpv;       // vectors, and lanes, of a word of bits
  constexpr int kAhead = DEPTH / kRounds; // whole blocks that a copy is ahead
  constexpr uint32_t kAllBits = (1u << kEpv) - 1u;
  static_assert(DEPTH == 2 || DEPTH % kRounds == 0, "copies run two rounds or whole blocks ahead");
  const int32_t lane = threadIdx.x & 31;
  const int32_t blocks = (row.vecs + 127) / 128;
  const int32_t words = (row.V + 31) / 32, shift = row.head & 31;
  auto bits = [&](int32_t b) -> uint32_t {
    if (b >= blocks) return 0u;
    if (!ok.row) return ok.any ? ~0u : 0u;
    const int32_t w = (row.head >> 5) + b * (4 * kEpv) + (lane & (4 * kEpv - 1));
    const uint32_t lo = w < words ? __ldg(ok.row + w) : 0u;
    const uint32_t hi = shift && w + 1 < words ? __ldg(ok.row + w + 1) : 0u;
    return __funnelshift_r(lo, hi, shift);
  };
  auto keep_of = [&](uint32_t word, int32_t j, int32_t q) -> uint32_t {
    const uint32_t w = __shfl_sync(kFull, word, q * kEpv + lane / kLanes);
    return j < row.vecs ? (w >> (lane % kLanes * kEpv)) & kAllBits : 0u;
  };
  // words[i]: the bits of the i-th block from the one in use on
  uint32_t word[kAhead + 2];
#pragma unroll
  for (int i = 0; i < kAhead + 2; ++i) word[i] = bits(share.first + i * share.step);
  int32_t b = share.first;
#pragma unroll
  for (int r = 0; r < DEPTH; ++r) {
    const int32_t j = (b + r / kRounds * share.step) * 128 + r % kRounds * 32 + lane;
    if (keep_of(word[r / kRounds], j, r % kRounds)) start(r, j);
    copy_commit();
  }
  int32_t slot0 = 0;
  for (; b < blocks; b += share.step) {
    const uint32_t behind = bits(b + (kAhead + 2) * share.step);
#pragma unroll
    for (int q = 0; q < kRounds; ++q) {
      const int32_t slot = DEPTH > kRounds ? slot0 + q : q & (DEPTH - 1);
      copy_wait<DEPTH - 1>();
      const int32_t j = b * 128 + q * 32 + lane;
      use(slot, j, keep_of(word[0], j, q));
      constexpr int kOver = DEPTH % kRounds;
      const int next = kAhead + (q + kOver) / kRounds, nq = (q + kOver) % kRounds;
      const int32_t nj = (b + next * share.step) * 128 + nq * 32 + lane;
      if (keep_of(word[next], nj, nq)) start(slot, nj);
      copy_commit();
    }
    if (DEPTH > kRounds) slot0 = (slot0 + kRounds) & (DEPTH - 1);
#pragma unroll
    for (int i = 0; i <= kAhead; ++i) word[i] = word[i + 1];
    word[kAhead + 1] = behind;
  }
  copy_wait<0>();
}

__device__ __forceinline__ uint64_t block_max(uint64_t k, Shared& sh) {
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  k = warp_max_u64(k);
  if (lane == 0) sh.warp_key[warp] = k;
  __syncthreads();
  k = warp_max_u64(sh.warp_key[lane & (kVerifyWarps - 1)]);
  return k;
}
// Between this and block_max there is a barrier in each call order used here.
__device__ __forceinline__ float block_sum(float s, Shared& sh) {
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  s = warp_sum(s);
  if (lane == 0) sh.warp_sum[warp] = s;
  __syncthreads();
  return warp_sum(lane < kVerifyWarps ? sh.warp_sum[lane] : 0.0f);
}

// Calls f for each token of this thread's share, one by one.
template <typename T, typename F>
__device__ __forceinline__ void each_token(const Row<T>& row, const Share& share, F&& f) {
  constexpr int kTokens = 128 * Row<T>::kEpv;
  const int32_t end = row.token(row.vecs);
  for (int32_t b = share.first; b * 128 < row.vecs; b += share.step)
    for (int32_t i = threadIdx.x & 31; i < kTokens && row.token(b * 128) + i < end; i += 32)
      f(row.token(b * 128) + i);
  const int32_t t = row.edge(share.head, share.tail);
  if (t >= 0) f(t);
}

// The sum of a slice whose maximum is m, by its definition: infinities share
// the weight, NaN has none.
template <typename T>
__device__ __noinline__ float sum_by_definition(const Row<T> row, const Allow ok, const Share share,
                                                float m, float inv) {
  float s = 0.0f;
  each_token(row, share, [&](int32_t t) {
    if (ok.has(t)) s += weight(fmaxf(row.at(t), -INFINITY), m, inv);
  });
  return s;
}

// `v` with -inf in the lanes that `keep` leaves out.
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& v, uint32_t keep, const Shared& sh) {
  if constexpr (sizeof(typename Dt<T>::Bits) == 4) {
    return make_uint4(keep & 1 ? v.x : 0xFF800000u, keep & 2 ? v.y : 0xFF800000u,
                      keep & 4 ? v.z : 0xFF800000u, keep & 8 ? v.w : 0xFF800000u);
  } else {
    constexpr uint32_t kNone = std::is_same_v<T, __half> ? 0xFC00FC00u : 0xFF80FF80u;
    const uint4 k = sh.lanes[keep];
    return make_uint4((v.x & k.x) | (kNone & ~k.x), (v.y & k.y) | (kNone & ~k.y),
                      (v.z & k.z) | (kNone & ~k.z), (v.w & k.w) | (kNone & ~k.w));
  }
}

// The largest element of a vector; NaN only where there is nothing else.
template <typename T>
__device__ __forceinline__ float vec_top(const uint4& v) {
  if constexpr (sizeof(typename Dt<T>::Bits) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else if constexpr (std::is_same_v<T, __half>) {
    const __half2* p = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
    return fmaxf(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
}

// A race's threads share a bar, the best score any of them has found so far:
// with a bar of its own some lane of a warp nearly always has a new best to
// look at (45 instructions for each element, against 11). A score has to be
// over the bar less this much to be looked at, more than all roundings between
// them, so the winner always is, whatever the order in which the bar rises.
constexpr float kSlack = 1.0f - 3.0e-5f;
constexpr float kMostScore = 1.0e30f;  // a bar is no higher: noise near 0 is still compared

// Maximum, its first index (where `first_index`) and the sum over the CTA's
// share of a row. With RACE, this thread's
// best of exp(x / T) / noise goes to `best`, too (-1: none); sh.bar is then
// order_key(-inf) before the call.
//
// The sum is of exp2(x c - ref) with c = log2(e) / T and ref the rounded m c:
// one fused multiply-add for each element; what the rounding left off is put
// right once, at the end.
template <typename T, bool RACE>
__device__ __forceinline__ Slice scan_slice(const Row<T>& row, const Allow& ok,
                                            const Share& share, float inv, bool first_index,
                                            const float* noise,
                                            bool noise_aligned, int32_t& best, uint32_t ring, Shared& sh) {
  constexpr int kEpv = Row<T>::kEpv;
  const float c = inv * kLog2e;
  float m = -INFINITY, ref = 0.0f, s = 0.0f;
  float score = -INFINITY;  // log2 of this thread's best in the race
  int32_t idx = 0, from = 0;
  best = -1;
  constexpr int kDepth = RACE ? 4 : 8;
  constexpr uint32_t kSlot = (RACE ? 1 + kEpv / 4 : 1) * kPlane;
  static_assert(kDepth * kSlot <= kRingBytes * kVerifyThreads, "the ring holds every slot");
  auto start = [&](int32_t slot, int32_t j) {
    copy_async<16>(ring + slot * kSlot, row.vec_at(j));
    if constexpr (RACE)
      copy_floats<kEpv>(ring + slot * kSlot + kPlane, noise + row.token(j), noise_aligned);
  };
  auto use = [&](int32_t slot, int32_t j, uint32_t keep) {
    const uint4 v = masked<T>(shared_vec(ring + slot * kSlot), keep, sh);
    const float top = vec_top<T>(v);
    if (top > m) {
      const float to = top * c;
      s *= m > -INFINITY ? exp2_fast(ref - to) : 0.0f;
      ref = to;
      m = top;
      from = j;
    }
    float w[kEpv];  // ref is 0 as long as there is nothing but -inf: weights of 0
#pragma unroll
    for (int i = 0; i < kEpv; ++i) {
      w[i] = exp2_fast(fmaf(Dt<T>::to_float(vec_get<T>(v, i)), c, -ref));
      s += w[i];
    }
    if constexpr (RACE) {
      const float bar =
          exp2_fast(key_value(*const_cast<volatile uint32_t*>(&sh.bar)) - ref) * kSlack;
      float e[kEpv], over = 0.0f;
      read_floats<kEpv>(ring + slot * kSlot + kPlane, e);
#pragma unroll
      for (int i = 0; i < kEpv; ++i) over = fmaxf(over, fmaf(-bar, e[i], w[i]));
      if (over > 0.0f) {
#pragma unroll
        for (int i = 0; i < kEpv; ++i) {
          const float f = __log2f(w[i]) + ref - __log2f(e[i]);
          if (f > score && w[i] > 0.0f) {
            score = f;
            best = row.token(j) + i;
          }
        }
        const float rise = fminf(score, ref + __log2f(kMostScore));
        if (rise > -INFINITY) atomicMax(&sh.bar, order_key(rise));
      }
    }
  };
  stream<T, kDepth>(row, ok, share, start, use);
  if (first_index && m > -INFINITY) {
    // the first maximal token of the vector that had it
    const uint32_t keep = ok.template bits<kEpv>(row.token(from));
    for (int i = kEpv - 1; i >= 0; --i)
      if ((keep >> i) & 1u && row.at(row.token(from) + i) == m) idx = row.token(from) + i;
  }
  const int32_t t = row.edge(share.head, share.tail);
  if (t >= 0 && ok.has(t)) {
    const float x = fmaxf(row.at(t), -INFINITY);
    if (x > -INFINITY) {
      if (x > m || (x == m && t < idx)) idx = t;
      if (x > m) {
        const float to = x * c;
        s *= m > -INFINITY ? exp2_fast(ref - to) : 0.0f;
        ref = to;
        m = x;
      }
      const float w = exp2_fast(fmaf(x, c, -ref));
      s += w;
      if (RACE && __log2f(w) + ref - __log2f(noise[t]) > score) best = t;
    }
  }
  s *= exp2_fast(-fmaf(m, c, -ref));  // from ref to m c
  const uint64_t k =
      block_max(m > -INFINITY ? pack_arg(order_key(m), first_index ? idx : 0) : 0, sh);
  Slice out;
  out.idx = k ? unpack_idx(k) : -1;
  out.m = k ? key_value(static_cast<uint32_t>(k >> 32)) : -INFINITY;
  out.s = block_sum(m > -INFINITY ? s * exp2_fast((m - out.m) * c) : 0.0f, sh);
  // an infinite maximum, a NaN, or a temperature at either end of its range
  if (k && !(out.s < INFINITY)) {
    __syncthreads();
    out.s = block_sum(sum_by_definition<T>(row, ok, share, out.m, inv), sh);
  }
  return out;
}

__device__ __forceinline__ uint64_t race_key(float score, int32_t t) {
  return pack_arg(__float_as_uint(score > 0.0f ? score : 0.0f), t);
}

// The race of max(p - q, 0) / noise over the CTA's share of a row: (score,
// lowest index), 0 where nothing takes part; sh.bar is 0 before the call.
// `draft`: a token that takes no part (-1: none).
template <typename T>
__device__ uint64_t race_slice(const Row<T>& row, const Allow& ok, const Share& share, float inv,
                               float m, float rz, const float* noise, bool noise_aligned,
                               const Given& given, int32_t draft, uint32_t ring, Shared& sh) {
  constexpr int kEpv = Row<T>::kEpv;
  const float c = inv * kLog2e;
  // p - q with full precision, and its score
  auto exact = [&](int32_t t) -> uint64_t {
    if (t == draft || !ok.has(t)) return 0;
    float left = weight(fmaxf(row.at(t), -INFINITY), m, inv) * rz;
    if (given.p) left -= load_prob(given.p, given.dtype, t);
    return left > 0.0f ? race_key(left / noise[t], t) : 0;
  };
  uint64_t mine = 0;
  if (m < INFINITY && c < INFINITY) {
    float best = -1.0f;
    int32_t idx = -1;
    const float ref = m * c, fix = exp2_fast(-fmaf(m, c, -ref)) * rz;
    constexpr int kDepth = 2;
    constexpr uint32_t kNoise = kPlane, kGiven = kPlane * (1 + kEpv / 4),
                       kSlot = kPlane * (1 + kEpv / 2);
    static_assert(kDepth * kSlot <= kRingBytes * kVerifyThreads, "the ring holds every slot");
    auto start = [&](int32_t slot, int32_t j) {
      copy_async<16>(ring + slot * kSlot, row.vec_at(j));
      copy_floats<kEpv>(ring + slot * kSlot + kNoise, noise + row.token(j), noise_aligned);
      given.template copy<kEpv>(ring + slot * kSlot + kGiven, row.token(j));
    };
    auto use = [&](int32_t slot, int32_t j, uint32_t keep) {
      if (!keep) return;  // nothing was copied
      const int32_t t = row.token(j);
      if (static_cast<uint32_t>(draft - t) < static_cast<uint32_t>(kEpv))
        keep &= ~(1u << (draft - t));
      const uint4 x = masked<T>(shared_vec(ring + slot * kSlot), keep, sh);
      const float bar = __uint_as_float(*const_cast<volatile uint32_t*>(&sh.bar)) * kSlack;
      float left[kEpv], e[kEpv], over = 0.0f;
      given.template read<kEpv>(ring + slot * kSlot + kGiven, t, left);
      read_floats<kEpv>(ring + slot * kSlot + kNoise, e);
#pragma unroll
      for (int i = 0; i < kEpv; ++i) {
        const float w = exp2_fast(fmaf(Dt<T>::to_float(vec_get<T>(x, i)), c, -ref));
        left[i] = fmaf(w, fix, -left[i]);
        over = fmaxf(over, fmaf(-bar, e[i], left[i]));
      }
      if (over > 0.0f) {
#pragma unroll
        for (int i = 0; i < kEpv; ++i) {
          const float f = fmaxf(__fdividef(left[i], e[i]), 0.0f);
          if (left[i] > 0.0f && f > best) {
            best = f;
            idx = t + i;
          }
        }
        if (best > 0.0f) atomicMax(&sh.bar, __float_as_uint(fminf(best, kMostScore)));
      }
    };
    stream<T, kDepth>(row, ok, share, start, use);
    if (idx >= 0) mine = exact(idx);
    const int32_t t = row.edge(share.head, share.tail);
    if (t >= 0) {
      const uint64_t k = exact(t);
      mine = k > mine ? k : mine;
    }
  } else {
    each_token(row, share, [&](int32_t t) {
      const uint64_t k = exact(t);
      mine = k > mine ? k : mine;
    });
  }
  return block_max(mine, sh);
}

// The largest of the cluster's keys; every CTA brings its own in `slot`.
template <int C>
__device__ __forceinline__ uint64_t cluster_max(uint64_t k, uint64_t& slot) {
  if constexpr (C == 1) {
    return k;
  } else {
    const int32_t lane = threadIdx.x & 31;
    if (threadIdx.x == 0) slot = k;
    cluster_barrier<C>();
    return warp_max_u64(peer_u64(peer_shared(&slot, lane < C ? lane : 0)));
  }
}

template <typename T, int C>
__global__ void __launch_bounds__(kVerifyThreads, kCtasPerSm) verify_kernel(const VerifyArgs a) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  const uint32_t ring =
      static_cast<uint32_t>(__cvta_generic_to_shared(dynamic)) + threadIdx.x * 16;
  const uint32_t rank = C == 1 ? 0 : cluster_rank();
  const int32_t b = static_cast<int32_t>(blockIdx.x / C);
  const int32_t tid = threadIdx.x, lane = tid & 31;
  const int32_t K = a.K, V = a.V;
  pdl_wait();
  const int32_t len = a.lens ? a.lens[b] : K;
  const int64_t first = a.src_rows ? a.src_rows[b] : static_cast<int64_t>(b) * (K + 1);
  const int64_t pfirst = a.prob_rows ? a.prob_rows[b] : static_cast<int64_t>(b) * K;
  const int64_t slot = a.slots ? a.slots[b] : b;
  const bool idle = len < 0 || len > K || first < 0 || first > a.src_total - 1 - len ||
                    (a.probs && len > 0 && (pfirst < 0 || pfirst > a.probs_total - len));
  int64_t* tokens = a.tokens + static_cast<int64_t>(b) * (K + 1);
  float* logprobs = a.logprobs + static_cast<int64_t>(b) * (K + 1);
  if (idle) {  // the same for every CTA of the cluster
    if (rank == 0) {
      for (int32_t i = tid; i <= K; i += kVerifyThreads) {
        tokens[i] = -1;
        logprobs[i] = 0.0f;
      }
      if (tid == 0) {
        a.counts[b] = 0;
        if (a.next_out) a.next_out[b] = a.pool[slot];
      }
    }
    return;
  }
  const float heat = a.temperature ? a.temperature[b] : a.temperature_all;
  const bool greedy = !(heat > 0.0f);
  const float inv = greedy ? 1.0f : 1.0f / heat;
  const Share share{static_cast<int32_t>(rank) * kVerifyWarps + (tid >> 5), C * kVerifyWarps,
                    rank == 0, rank == C - 1};
  auto draft_at = [&](int32_t i) -> int64_t {
    const int64_t at = static_cast<int64_t>(b) * a.draft_stride + i;
    return a.drafts64 ? static_cast<const int64_t*>(a.drafts)[at]
                      : static_cast<const int32_t*>(a.drafts)[at];
  };
  auto step = [&](int32_t s, int64_t t) -> int32_t {
    return (s < 0 || s >= a.num_states || t < 0 || t >= V)
               ? -1
               : __ldg(a.tok_next + static_cast<int64_t>(s) * V + t);
  };
  // the states along the drafts, each one position ahead
  if (a.bits) {
    if (a.path) {
      for (int32_t i = tid; i <= len; i += kVerifyThreads)
        sh.state[i] = a.path[static_cast<int64_t>(b) * (K + 1) + i];
    } else if (tid == 0) {
      sh.state[0] = a.pool[slot];
    }
  }
  if (tid == 0) sh.bar = order_key(-INFINITY);
  if (sizeof(typename Dt<T>::Bits) == 2) {
    auto two = [&](uint32_t k) { return (k & 1 ? 0xFFFFu : 0u) | (k & 2 ? 0xFFFF0000u : 0u); };
    for (uint32_t k = tid; k < 256; k += kVerifyThreads)
      sh.lanes[k] = make_uint4(two(k), two(k >> 2), two(k >> 4), two(k >> 6));
  }
  __syncthreads();

  const float* noise = a.noise + static_cast<int64_t>(b) * a.noise_stride;
  auto row_of = [&](int32_t i) {
    return Row<T>(
        static_cast<const typename Dt<T>::Bits*>(a.src) + (first + i) * a.src_stride, V);
  };
  auto allow_of = [&](int32_t i) {
    Allow ok{nullptr, true};
    if (a.bits) {
      const int32_t s = sh.state[i];
      ok.any = false;
      if (s >= 0 && s < a.num_states) ok.row = a.bits + static_cast<int64_t>(s) * a.wstride;
    }
    return ok;
  };
  auto noise_fits = [&](const Row<T>& row) {
    return (reinterpret_cast<uintptr_t>(noise + row.head) & 15u) == 0;
  };
  int32_t best = -1;  // of the last row's race
  int32_t n = 0;      // the first position that is not an accepted draft
  for (int32_t begin = 0;; begin += a.window) {
    const int32_t end = min(begin + a.window, len + 1);
    for (int32_t i = begin; i < end; ++i) {
      const Row<T> row = row_of(i);
      const Allow ok = allow_of(i);
      // what the decision needs comes while the row is scanned
      const int64_t d = i < len ? draft_at(i) : -1;
      const bool inside = d >= 0 && d < V;
      float xd = -INFINITY, qd = 1.0f, uniform = 0.0f;
      int32_t next = -1;
      if (i < len) {
        if (inside && ok.has(static_cast<int32_t>(d))) xd = fmaxf(row.at(d), -INFINITY);
        if (!greedy) uniform = a.uniforms[static_cast<int64_t>(b) * a.uniform_stride + i];
        if (a.probs && inside)
          qd = load_prob(a.probs, a.probs_dtype, (pfirst + i) * a.probs_stride + d);
        if (a.bits && !a.path) next = step(sh.state[i], d);
      }
      const Slice r =
          i == len && !greedy
              ? scan_slice<T, true>(row, ok, share, inv, false, noise,
                                    noise_fits(row), best, ring, sh)
              : scan_slice<T, false>(row, ok, share, inv, greedy, noise, false, best,
                                     ring, sh);
      if (tid == 0) {
        sh.slice[i] = r;
        Position& p = sh.position[i];
        p.xd = xd;
        p.qd = qd;
        p.uniform = uniform;
        p.draft = inside ? static_cast<int32_t>(d) : -1;
        if (i < len && a.bits && !a.path) sh.state[i + 1] = next;
      }
      __syncthreads();
    }
    cluster_barrier<C>();
    // a warp puts a position's slices together and decides on it
    for (int32_t i = begin + (tid >> 5); i < end; i += kVerifyWarps) {
      Position& p = sh.position[i];
      Slice r;
      const uint32_t peer = C > 1 ? peer_shared(&sh.slice[i], lane < C ? lane : 0) : 0;
      if constexpr (C > 1) {
        r.m = __uint_as_float(peer_u32(peer));
        r.idx = lane < C ? static_cast<int32_t>(peer_u32(peer + 4)) : -1;
        r.s = __uint_as_float(peer_u32(peer + 8));
        const uint64_t k = warp_max_u64(r.idx < 0 ? 0 : pack_arg(order_key(r.m), r.idx));
        const float m = k ? key_value(static_cast<uint32_t>(k >> 32)) : -INFINITY;
        r.s = warp_sum(r.idx < 0 ? 0.0f : r.s * weight(r.m, m, inv));
        r.m = m;
        r.idx = k ? unpack_idx(k) : -1;
      } else {
        r = sh.slice[i];
      }
      if (lane == 0) {
        p.m = r.m;
        p.s = r.s;
        p.idx = r.idx;
        p.accept = i < len && r.idx >= 0 &&
                   (greedy ? p.draft == r.idx
                           : p.uniform * p.qd < weight(p.xd, r.m, inv) / r.s);
      }
    }
    __syncthreads();
    for (n = begin; n < end && sh.position[n].accept; ++n) {
      if (rank == 0 && tid == 0) {
        const Position& p = sh.position[n];
        tokens[n] = p.draft;
        logprobs[n] = (p.xd == p.m ? 0.0f : (p.xd - p.m) * inv) - logf(p.s);
      }
    }
    if (n < end) break;
  }
  const Position p = sh.position[n];
  int64_t token = -1;
  float logprob = 0.0f;
  if (p.idx >= 0) {  // else nothing is allowed here
    const Row<T> row = row_of(n);
    if (greedy) {
      token = p.idx;
    } else {
      const Allow ok = allow_of(n);
      uint64_t won = 0;
      if (tid == 0) sh.bar = 0;
      __syncthreads();
      if (n == len && p.m < INFINITY) {
        const float w = best >= 0 ? weight(row.at(best), p.m, inv) : 0.0f;
        won = block_max(w > 0.0f ? race_key(w / noise[best], best) : 0, sh);
      } else {
        Given given{nullptr, a.probs_dtype, false};
        if (n < len && a.probs) {
          const int32_t size = a.probs_dtype == BPD_F32 ? 4 : 2;
          const char* q = static_cast<const char*>(a.probs) + (pfirst + n) * a.probs_stride * size;
          given.p = q;
          given.aligned =
              reinterpret_cast<uintptr_t>(q + row.head * size) % min(16, Row<T>::kEpv * size) == 0;
        }
        won = race_slice<T>(row, ok, share, inv, p.m, 1.0f / p.s, noise,
                            noise_fits(row), given, n < len && !a.probs ? p.draft : -1, ring, sh);
      }
      won = cluster_max<C>(won, sh.race[0]);
      if (!won) {  // nothing left of p - q: the race is over p
        __syncthreads();
        if (tid == 0) sh.bar = 0;
        __syncthreads();
        won = cluster_max<C>(
            race_slice<T>(row, ok, share, inv, p.m, 1.0f / p.s, noise,
                          noise_fits(row), Given{nullptr, 0, false}, -1, ring, sh),
            sh.race[1]);
      }
      if (won) token = unpack_idx(won);
    }
    if (token >= 0) {
      const float xt = row.at(token);
      logprob = (xt == p.m ? 0.0f : (xt - p.m) * inv) - logf(p.s);
    }
  }
  if (rank == 0) {
    for (int32_t i = n + tid; i <= K; i += kVerifyThreads) {
      tokens[i] = i == n ? token : -1;
      logprobs[i] = i == n ? logprob : 0.0f;
    }
    if (tid == 0) {
      a.counts[b] = n + (token >= 0);
      if (a.tok_next) {
        const int32_t next = token < 0 ? -1 : step(sh.state[n], token);
        if (a.next_out) a.next_out[b] = next;
        if (a.write_back) a.pool[slot] = next;
      }
    }
  }
  cluster_barrier<C>();  // nobody leaves while a neighbour may read its shared memory
}

template <typename T, int C>
cudaError_t launch_verify(const VerifyArgs& a, cudaStream_t st) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev].load(std::memory_order_relaxed))) {
    e = cudaFuncSetAttribute(verify_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kRingBytes * kVerifyThreads);
    if (e == cudaSuccess && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch) * C);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.dynamicSmemBytes = kRingBytes * kVerifyThreads;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = BPD_PDL ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, verify_kernel<T, C>, a);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

extern "C" bpd_status bpd_verify_drafts(
    const void* src, int32_t src_dtype, int64_t src_stride, int64_t src_total,
    const int64_t* src_rows, const void* drafts, int32_t drafts_int64, int64_t draft_stride,
    const int32_t* draft_lens, const void* probs, int32_t probs_dtype, int64_t probs_stride,
    int64_t probs_total, const int64_t* prob_rows, const float* uniforms, int64_t uniform_stride,
    const float* noise, int64_t noise_stride, const float* temperature, float temperature_all,
    int32_t batch, int32_t max_drafts, int32_t vocab_size, int32_t* state_pool,
    const int64_t* slots, const int32_t* path, const uint32_t* allow_bits, int32_t words_stride,
    const int32_t* tok_next, int32_t num_states, int64_t* tokens_out, int32_t* counts_out,
    float* logprobs_out, int32_t* next_out, int32_t write_back, void* stream) {
  const char* what = "bpd_verify_drafts";
  BPD_REQUIRE(batch >= 0 && vocab_size > 0 && max_drafts >= 0 && src_total >= 0,
              "%s: bad sizes", what);
  if (max_drafts > BPD_MAX_DRAFTS)
    return fail(BPD_ERR_CAPACITY, "%s: more than %d drafts", what, BPD_MAX_DRAFTS);
  if (batch > INT_MAX / kMaxCluster) return fail(BPD_ERR_CAPACITY, "%s: batch too large", what);
  if (batch == 0) return BPD_OK;
  BPD_REQUIRE(src && tokens_out && counts_out && logprobs_out, "%s: null pointer", what);
  BPD_REQUIRE(src_stride >= vocab_size, "%s: row stride < vocab", what);
  BPD_REQUIRE(max_drafts == 0 || (drafts && draft_stride >= max_drafts),
              "%s: drafts missing, or their row stride < max_drafts", what);
  const bool all_greedy = temperature == nullptr && !(temperature_all > 0.0f);
  BPD_REQUIRE(all_greedy || (noise && noise_stride >= vocab_size),
              "%s: sampling needs a row of noise for each request", what);
  BPD_REQUIRE(all_greedy || max_drafts == 0 || (uniforms && uniform_stride >= max_drafts),
              "%s: sampling needs a uniform number for each draft", what);
  BPD_REQUIRE(!probs || (probs_stride >= vocab_size && probs_total >= 0 && probs_dtype >= BPD_F32 &&
                         probs_dtype <= BPD_F16),
              "%s: bad draft probabilities", what);
  BPD_REQUIRE(!allow_bits || (words_stride >= (vocab_size + 31) / 32 && num_states > 0),
              "%s: words_stride too small, or no states", what);
  BPD_REQUIRE(!allow_bits || path || (state_pool && tok_next),
              "%s: a grammar needs state_pool and tok_next, or path", what);
  BPD_REQUIRE((!next_out && !write_back) || (state_pool && tok_next && allow_bits),
              "%s: next states need state_pool, allow_bits and tok_next", what);
  VerifyArgs a{src, src_stride, src_total, src_rows, drafts, draft_stride, drafts_int64,
               draft_lens, probs, probs_dtype, probs_stride, probs_total, prob_rows, uniforms,
               uniform_stride, noise, noise_stride, temperature, temperature_all, batch,
               max_drafts, vocab_size, state_pool, slots, path, allow_bits, words_stride,
               allow_bits ? tok_next : nullptr, num_states, tokens_out, counts_out, logprobs_out,
               next_out, write_back, 1};
  cudaStream_t st = as_stream(stream);
  return with_dtype(src_dtype, what, [&](auto tag) {
    using T = decltype(tag);
    // Positions are scanned ahead of the decisions where all rows are few
    // enough to be read in less time than the cluster takes to meet.
    const int64_t rows_bytes = static_cast<int64_t>(batch) * (max_drafts + 1) * vocab_size *
                               static_cast<int64_t>(sizeof(typename Dt<T>::Bits));
    a.window = rows_bytes <= (100ll << 20) ? max_drafts + 1 : 1;
    // enough CTAs to fill the SMs four times over, as far as a cluster reaches
    const int64_t room = kCtasPerSm * static_cast<int64_t>(sm_count());
    const cudaError_t e = batch * 8ll <= room   ? launch_verify<T, 8>(a, st)
                          : batch * 4ll <= room ? launch_verify<T, 4>(a, st)
                          : batch * 2ll <= room ? launch_verify<T, 2>(a, st)
                                                : launch_verify<T, 1>(a, st);
    return e == cudaSuccess ? BPD_OK : fail(BPD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  });
}
