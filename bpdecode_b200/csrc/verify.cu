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
// of the row once, with a running maximum and sum; the slices' (m, argmax, s)
// meet through distributed shared memory in a fixed order, so a result does
// not depend on timing. The row that is replaced is scanned a second time
// (from L2) with the noise and the draft's probabilities.
#include <algorithm>
#include <climits>

#include "common.cuh"

namespace bpd {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxCluster = 8;

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
};

// What a slice of a row comes to: its maximum, the first index that has it
// (-1: nothing allowed), and the sum of exp((x - m) / T).
struct Slice {
  float m;
  int32_t idx;
  float s;
};

// The two races over a slice: packed (score, lowest index) of max(p - q, 0) / e
// and of p / e; 0 where nothing takes part.
struct Race {
  uint64_t left;
  uint64_t all;
};

struct Shared {
  uint64_t warp_key[kVerifyWarps];
  uint64_t warp_key2[kVerifyWarps];
  float warp_sum[kVerifyWarps];
  Slice slice[2];  // by the position's parity: a neighbour may still read the other
  Race race;
  Slice row;       // the whole row's
  Race winner;
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

// A row's allow bits: every token (no grammar), a row of bits, or nothing.
struct Allow {
  const uint32_t* row;  // NULL: see `any`
  bool any;
  __device__ __forceinline__ bool has(int32_t t) const {
    return row ? ((__ldg(row + (t >> 5)) >> (t & 31)) & 1u) : any;
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

// Maximum, its first index and the sum over tokens [t0, t1), by the whole CTA.
template <typename T>
__device__ Slice scan_slice(const void* row, const Allow& ok, int32_t t0, int32_t t1, float inv,
                            Shared& sh) {
  float m = -INFINITY, s = 0.0f;
  int32_t idx = -1;
  for (int32_t t = t0 + static_cast<int32_t>(threadIdx.x); t < t1; t += kVerifyThreads) {
    if (!ok.has(t)) continue;
    const float x = load_logit<T>(row, t);
    if (!(x > -INFINITY)) continue;  // NaN counts as -inf
    if (x > m) {
      s = idx < 0 ? 1.0f : fmaf(s, expf((m - x) * inv), 1.0f);
      m = x;
      idx = t;
    } else {
      s += weight(x, m, inv);
    }
  }
  const uint64_t mine = idx < 0 ? 0 : pack_arg(order_key(m), idx);
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t k = warp_max_u64(mine);
  if (lane == 0) sh.warp_key[warp] = k;
  __syncthreads();
  k = sh.warp_key[lane < kVerifyWarps ? lane : 0];
  k = warp_max_u64(k);
  Slice out;
  out.idx = k ? unpack_idx(k) : -1;
  out.m = k ? load_logit<T>(row, out.idx) : -INFINITY;
  s = idx < 0 ? 0.0f : s * weight(m, out.m, inv);
  s = warp_sum(s);
  if (lane == 0) sh.warp_sum[warp] = s;
  __syncthreads();
  out.s = warp_sum(lane < kVerifyWarps ? sh.warp_sum[lane] : 0.0f);
  return out;
}

__device__ __forceinline__ uint64_t race_key(float score, int32_t t) {
  return pack_arg(__float_as_uint(score > 0.0f ? score : 0.0f), t);
}

// The two races over tokens [t0, t1). `given`: the draft's row of
// probabilities, or NULL; `draft`: the token that takes no part (-1: none).
template <typename T>
__device__ Race race_slice(const void* row, const Allow& ok, int32_t t0, int32_t t1, float inv,
                           float m, float rz, const float* noise, const void* given,
                           int32_t given_dtype, int32_t draft, Shared& sh) {
  Race r{0, 0};
  for (int32_t t = t0 + static_cast<int32_t>(threadIdx.x); t < t1; t += kVerifyThreads) {
    if (!ok.has(t)) continue;
    const float w = weight(fmaxf(load_logit<T>(row, t), -INFINITY), m, inv);
    if (!(w > 0.0f)) continue;
    const float p = w * rz, e = noise[t];
    const uint64_t a = race_key(p / e, t);
    r.all = a > r.all ? a : r.all;
    float left = p;
    if (given) left = p - load_prob(given, given_dtype, t);
    if (left > 0.0f && t != draft) {
      const uint64_t l = race_key(left / e, t);
      r.left = l > r.left ? l : r.left;
    }
  }
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  r.left = warp_max_u64(r.left);
  r.all = warp_max_u64(r.all);
  if (lane == 0) {
    sh.warp_key[warp] = r.left;
    sh.warp_key2[warp] = r.all;
  }
  __syncthreads();
  r.left = warp_max_u64(sh.warp_key[lane < kVerifyWarps ? lane : 0]);
  r.all = warp_max_u64(sh.warp_key2[lane < kVerifyWarps ? lane : 0]);
  __syncthreads();
  return r;
}

template <typename T, int C>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
  __shared__ Shared sh;
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
  const int32_t per = ((V + C - 1) / C + 127) / 128 * 128;
  const int32_t t0 = min(V, static_cast<int32_t>(rank) * per), t1 = min(V, t0 + per);
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
  // the states along the drafts
  if (a.bits) {
    if (a.path) {
      for (int32_t i = tid; i <= len; i += kVerifyThreads)
        sh.state[i] = a.path[static_cast<int64_t>(b) * (K + 1) + i];
    } else if (tid == 0) {
      int32_t s = a.pool[slot];
      sh.state[0] = s;
      for (int32_t i = 0; i < len; ++i) sh.state[i + 1] = s = step(s, draft_at(i));
    }
  }
  __syncthreads();

  int32_t n = 0;
  int64_t token = -1;
  float logprob = 0.0f;
  for (;; ++n) {
    const void* row = static_cast<const typename Dt<T>::Bits*>(a.src) + (first + n) * a.src_stride;
    Allow ok{nullptr, true};
    if (a.bits) {
      const int32_t s = sh.state[n];
      ok.any = false;
      if (s >= 0 && s < a.num_states) ok.row = a.bits + static_cast<int64_t>(s) * a.wstride;
    }
    Slice r = scan_slice<T>(row, ok, t0, t1, inv, sh);
    if constexpr (C > 1) {
      Slice& own = sh.slice[n & 1];
      if (tid == 0) own = r;
      cluster_barrier<C>();
      const uint32_t peer = peer_shared(&own, lane < C ? lane : 0);
      r.m = __uint_as_float(peer_u32(peer));
      r.idx = lane < C ? static_cast<int32_t>(peer_u32(peer + 4)) : -1;
      r.s = __uint_as_float(peer_u32(peer + 8));
      const uint64_t k = warp_max_u64(r.idx < 0 ? 0 : pack_arg(order_key(r.m), r.idx));
      const int32_t idx = k ? unpack_idx(k) : -1;
      const float m = k ? load_logit<T>(row, idx) : -INFINITY;
      r.s = warp_sum(r.idx < 0 ? 0.0f : r.s * weight(r.m, m, inv));
      r.m = m;
      r.idx = idx;
    }
    if (r.idx < 0) break;  // nothing is allowed here
    const int64_t d = n < len ? draft_at(n) : -1;
    if (n < len) {
      bool accept;
      float xd = -INFINITY;
      if (d >= 0 && d < V && ok.has(static_cast<int32_t>(d)))
        xd = fmaxf(load_logit<T>(row, d), -INFINITY);
      if (greedy) {
        accept = d == r.idx;
      } else {
        const float p = weight(xd, r.m, inv) / r.s;
        const float q = a.probs && d >= 0 && d < V
                            ? load_prob(a.probs, a.probs_dtype,
                                        (pfirst + n) * a.probs_stride + d)
                            : 1.0f;
        accept = a.uniforms[static_cast<int64_t>(b) * a.uniform_stride + n] * q < p;
      }
      if (accept) {
        if (rank == 0 && tid == 0) {
          tokens[n] = d;
          logprobs[n] = (xd == r.m ? 0.0f : (xd - r.m) * inv) - logf(r.s);
        }
        continue;
      }
    }
    if (greedy) {
      token = r.idx;
    } else {
      const void* given = nullptr;
      if (n < len && a.probs) {
        const int64_t at = (pfirst + n) * a.probs_stride;
        given = static_cast<const char*>(a.probs) + at * (a.probs_dtype == BPD_F32 ? 4 : 2);
      }
      Race w = race_slice<T>(row, ok, t0, t1, inv, r.m, 1.0f / r.s,
                             a.noise + static_cast<int64_t>(b) * a.noise_stride, given,
                             a.probs_dtype,
                             n < len && !a.probs && d >= 0 && d < V ? static_cast<int32_t>(d) : -1,
                             sh);
      if constexpr (C > 1) {
        if (tid == 0) sh.race = w;
        cluster_barrier<C>();
        const uint32_t peer = peer_shared(&sh.race, lane < C ? lane : 0);
        w.left = warp_max_u64(peer_u64(peer));
        w.all = warp_max_u64(peer_u64(peer + 8));
      }
      token = unpack_idx(w.left ? w.left : w.all);
    }
    const float xt = load_logit<T>(row, token);
    logprob = (xt == r.m ? 0.0f : (xt - r.m) * inv) - logf(r.s);
    break;
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch) * C);
  cfg.blockDim = dim3(kVerifyThreads);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, C>, a);
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
               next_out, write_back};
  cudaStream_t st = as_stream(stream);
  return with_dtype(src_dtype, what, [&](auto tag) {
    using T = decltype(tag);
    const cudaError_t e = batch >= 4 * sm_count() ? launch_verify<T, 1>(a, st)
                                                  : launch_verify<T, kMaxCluster>(a, st);
    return e == cudaSuccess ? BPD_OK : fail(BPD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  });
}
