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
// Up to three launches. walk_kernel: the states along the drafts, and what the
// decisions need besides the rows. scan_kernel: the drafts' rows, one CTA for a
// chunk of a row, in one pass with a running maximum and sum. The CTA of a row
// that finishes last puts the chunks together and decides; CTAs are ordered by
// position, and those of a row behind a refused draft leave at once, so in a
// large batch few of these rows are read. last_kernel: the row that decides
// the last token. Behind the last draft it is scanned and raced in one pass, on
// w / e, which needs no Z; a row whose draft was refused is passed over a
// second time, with the noise and the draft's probabilities. No CTA waits for
// another.
//
// All are bound by HBM; few requests by the loads that depend on one another
// (state, allow bits, logits). What a thread finds best in a race is scored
// again with full precision: in the race along with a scan only scores within one
// thread are compared in fast arithmetic, in that of a refused draft none are.
// Nothing depends on the order in which CTAs or warps run: chunks meet in a fixed
// order, a race takes the maximum of (score, lowest index), and what its threads
// share only leaves out tokens that cannot win.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "common.cuh"

namespace bpd {
namespace {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kScanThreads = 256, kScanWarps = kScanThreads / 32;
constexpr int kMaxChunks = 32;  // of a row
constexpr int kScanCtas = 5, kLastCtas = 4;  // on an SM
constexpr int kRaceVecs = 2;    // vectors of a scan's race that a lane reads at once
constexpr float kLog2e = 1.4426950408889634f;

using VerifyArgs = bpd_verify_args;

// What walk_kernel leaves for a position: its state, the draft (-1: none, or
// no token of the vocabulary) with its logit (-inf: rejected) and probability,
// and the uniform number.
struct Position {
  int32_t state, draft;
  float xd, qd, uniform;
  uint32_t arrived;  // chunks of the row that are done
  // the whole row: maximum, its first index (-1: nothing is allowed) and sum
  float m, s;
  int32_t idx;
};

// A chunk of a row: maximum, its first index, the sum of exp((x - m) / T); and
// its best in the race.
struct Part {
  float m, s;
  int32_t idx;
  int32_t best;
  float x, e;
};

struct Request {
  int32_t len;       // -1: idle
  int32_t end;       // the first position that is not an accepted draft
  uint32_t arrived;  // chunks of its row that are done
  uint32_t pad;
  unsigned long long race;  // its winner so far
};

struct Workspace {
  Request* request;    // [batch]
  Position* position;  // [batch, K + 1]
  Part* part;          // [batch, K + 1, kMaxChunks]
};

// The inverse of order_key.
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values, one instruction for both.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair_of(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ void split(const Pair& p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v));
}
__device__ __forceinline__ Pair fma2(const Pair& a, const Pair& b, const Pair& c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair mul2(const Pair& a, const Pair& b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair add2(const Pair& a, const Pair& b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// A row's allow bits: every token (no grammar), a row of bits, or nothing.
struct Allow {
  const uint32_t* row;  // NULL: see `any`
  bool any;
  __device__ __forceinline__ Allow(const VerifyArgs& a, int32_t state)
      : row(nullptr), any(!a.allow_bits) {
    if (a.allow_bits && state >= 0 && state < a.num_states)
      row = a.allow_bits + static_cast<int64_t>(state) * a.words_stride;
  }
  __device__ __forceinline__ bool has(int32_t t) const {
    return row ? ((__ldg(row + (t >> 5)) >> (t & 31)) & 1u) : any;
  }
};

// A row of logits as 16-byte vectors: `head` tokens, `vecs` vectors, a tail;
// in blocks of 128 vectors, four for each lane of a warp.
template <typename T>
struct Row {
  static constexpr int kEpv = Dt<T>::kPerVec;
  using Bits = typename Dt<T>::Bits;
  const Bits* p;
  int32_t head, vecs;
  __device__ Row(const VerifyArgs& a, int64_t row)
      : p(static_cast<const Bits*>(a.src) + row * a.src_stride) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    head = min(a.vocab_size,
               static_cast<int32_t>((16u - off) & 15u) / static_cast<int32_t>(sizeof(Bits)));
    vecs = (a.vocab_size - head) / kEpv;
  }
  __device__ __forceinline__ float at(int64_t t) const { return Dt<T>::to_float(p[t]); }
  __device__ __forceinline__ int32_t token(int32_t vec) const { return head + vec * kEpv; }
  __device__ __forceinline__ uint4 vec(int32_t j) const {
    return __ldg(reinterpret_cast<const uint4*>(p + head) + j);
  }
  // the blocks [first, end) of chunk c of n
  __device__ __forceinline__ void chunk(int32_t c, int32_t n, int32_t& first, int32_t& end) const {
    const int32_t blocks = (vecs + 127) / 128;
    first = static_cast<int32_t>(static_cast<int64_t>(blocks) * c / n);
    end = static_cast<int32_t>(static_cast<int64_t>(blocks) * (c + 1) / n);
  }
  // This lane's 32 (or 16) allow bits of block b: lane l has word l, of 32
  // tokens; 0 behind the vectors.
  __device__ __forceinline__ uint32_t bits(const Allow& ok, int32_t b, int32_t V) const {
    constexpr int kLanes = 32 / kEpv;  // vectors of a word
    const int32_t l = threadIdx.x & (4 * kEpv - 1);
    const int32_t have = vecs - b * 128 - l * kLanes;  // vectors from here on
    if (have <= 0) return 0u;
    uint32_t w = ok.any ? ~0u : 0u;
    if (ok.row) {
      const int32_t at = (head >> 5) + b * (4 * kEpv) + l, shift = head & 31;
      const uint32_t lo = __ldg(ok.row + at);
      const uint32_t hi = shift && at + 1 < (V + 31) / 32 ? __ldg(ok.row + at + 1) : 0u;
      w = __funnelshift_r(lo, hi, shift);
    }
    return have < kLanes ? w & ((1u << have * kEpv) - 1u) : w;
  }
  // From the lanes' words, the bits of this lane's vector q of four.
  __device__ __forceinline__ static uint32_t keep(uint32_t word, int32_t q) {
    constexpr int kLanes = 32 / kEpv;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t w = __shfl_sync(kFull, word, q * kEpv + lane / kLanes);
    return (w >> (lane % kLanes * kEpv)) & ((1u << kEpv) - 1u);
  }
  // Calls f for the tokens around the vectors, by one warp of the first and
  // last chunk.
  template <typename F>
  __device__ __forceinline__ void edges(int32_t c, int32_t n, int32_t V, F&& f) const {
    const int32_t i = threadIdx.x, tail = token(vecs);
    if (c == 0 && i < head) f(i);
    if (c == n - 1 && i >= 32 && i - 32 < V - tail) f(tail + i - 32);
  }
  // Calls f for each token of this thread's share of chunk c, one by one.
  template <typename F>
  __device__ __forceinline__ void each(int32_t c, int32_t n, int32_t V, F&& f) const {
    int32_t first, end;
    chunk(c, n, first, end);
    const int32_t last = min(token(vecs), token(end * 128));
    for (int32_t t = token(first * 128) + static_cast<int32_t>(threadIdx.x); t < last;
         t += kScanThreads)
      f(t);
    edges(c, n, V, f);
  }
};

// exp((x - m) / T) where x is not NaN and m the row's maximum: 1 at the
// maximum itself, which may be +inf, 0 at -inf.
__device__ __forceinline__ float weight(float x, float m, float inv) {
  if (x == m) return 1.0f;
  return x > -INFINITY ? expf((x - m) * inv) : 0.0f;
}

__device__ __forceinline__ float load_prob(const void* row, int32_t dtype, int64_t t) {
  if (dtype == BPD_F32) return static_cast<const float*>(row)[t];
  const uint16_t u = static_cast<const uint16_t*>(row)[t];
  return dtype == BPD_BF16 ? Dt<__nv_bfloat16>::to_float(u) : Dt<__half>::to_float(u);
}

// N consecutive floats from p on.
template <int N>
__device__ __forceinline__ void load_floats(const float* p, bool aligned, float (&out)[N]) {
  if (aligned) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(p + i));
      out[i] = f.x;
      out[i + 1] = f.y;
      out[i + 2] = f.z;
      out[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = __ldg(p + i);
  }
}

// A row of the draft's probabilities (p == NULL: none).
struct Given {
  const uint8_t* p;
  int32_t dtype;
  __device__ __forceinline__ int32_t size() const { return dtype == BPD_F32 ? 4 : 2; }
  // whether N from token t on can be read as whole vectors
  template <int N>
  __device__ __forceinline__ bool fits(int32_t t) const {
    return reinterpret_cast<uintptr_t>(p + t * static_cast<int64_t>(size())) %
               min(16, N * size()) == 0;
  }
  template <int N>
  __device__ __forceinline__ void load(int32_t t, bool aligned, float (&out)[N]) const {
    if (dtype == BPD_F32) {
      load_floats<N>(reinterpret_cast<const float*>(p) + t, aligned, out);
      return;
    }
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + t;
    uint32_t w[N / 2];
    if (aligned) {
      if constexpr (N == 8) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(h));
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
      } else {
        const uint2 v = __ldcs(reinterpret_cast<const uint2*>(h));
        w[0] = v.x;
        w[1] = v.y;
      }
    } else {
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

// For each byte of allow bits, the 16-bit lanes of a vector that it keeps.
struct Lanes {
  uint4 of[256];
  __device__ __forceinline__ void fill() {
    auto two = [](uint32_t k) { return (k & 1 ? 0xFFFFu : 0u) | (k & 2 ? 0xFFFF0000u : 0u); };
    for (uint32_t k = threadIdx.x; k < 256; k += kScanThreads)
      of[k] = make_uint4(two(k), two(k >> 2), two(k >> 4), two(k >> 6));
  }
};

// `v` with -inf in the lanes that `keep` leaves out.
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& v, uint32_t keep, const Lanes& lanes) {
  if constexpr (sizeof(typename Dt<T>::Bits) == 4) {
    return make_uint4(keep & 1 ? v.x : 0xFF800000u, keep & 2 ? v.y : 0xFF800000u,
                      keep & 4 ? v.z : 0xFF800000u, keep & 8 ? v.w : 0xFF800000u);
  } else {
    constexpr uint32_t kNone = std::is_same_v<T, __half> ? 0xFC00FC00u : 0xFF80FF80u;
    const uint4 k = lanes.of[keep];
    return make_uint4((v.x & k.x) | (kNone & ~k.x), (v.y & k.y) | (kNone & ~k.y),
                      (v.z & k.z) | (kNone & ~k.z), (v.w & k.w) | (kNone & ~k.w));
  }
}

// The larger of each of two vectors' elements, and the largest of a vector's;
// NaN only where there is nothing else.
template <typename T>
__device__ __forceinline__ uint4 vec_max2(const uint4& a, const uint4& b) {
  uint4 r;
  if constexpr (sizeof(typename Dt<T>::Bits) == 4) {
    r.x = __float_as_uint(fmaxf(__uint_as_float(a.x), __uint_as_float(b.x)));
    r.y = __float_as_uint(fmaxf(__uint_as_float(a.y), __uint_as_float(b.y)));
    r.z = __float_as_uint(fmaxf(__uint_as_float(a.z), __uint_as_float(b.z)));
    r.w = __float_as_uint(fmaxf(__uint_as_float(a.w), __uint_as_float(b.w)));
  } else {
    using Two = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const Two* p = reinterpret_cast<const Two*>(&a);
    const Two* q = reinterpret_cast<const Two*>(&b);
    Two* o = reinterpret_cast<Two*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __hmax2(p[i], q[i]);
  }
  return r;
}
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
// look at. A score has to be over the bar less this much to be looked at, more
// than all roundings between them, so the winner always is, whatever the order
// in which the bar rises. (Scores whose weights are exp2 of up to 128 in magnitude,
// from arguments, logarithms and differences rounded to 2^-24 of that: 4e-5.)
constexpr float kSlack = 1.0f - 1.0f / 8192;
constexpr float kMostScore = 1.0e30f;  // a bar is no higher: noise near 0 is still compared

// The bar of a race that is run along with the scan: log2 of a score, `over` that of
// a token at the reference `ref` of the thread that found it (see Scan). The two
// are kept apart, since at low temperatures, or with large logits, fp32 has no
// room in ref c for the scores over it: at a logit of 20 and T = 1e-6 its unit is 2.
struct Lead {
  float ref, over;
  __device__ __forceinline__ static Lead of(uint64_t v) {
    return {__uint_as_float(static_cast<uint32_t>(v >> 32)),
            __uint_as_float(static_cast<uint32_t>(v))};
  }
  __device__ __forceinline__ uint64_t bits() const {
    return uint64_t(__float_as_uint(ref)) << 32 | __float_as_uint(over);
  }
  // over another reference
  __device__ __forceinline__ float from(float base, float c) const {
    return fmaf(ref - base, c, over);
  }
};

__device__ __forceinline__ uint64_t race_key(float score, int32_t t) {
  return pack_arg(__float_as_uint(score > 0.0f ? score : 0.0f), t);
}

__device__ __forceinline__ uint64_t block_max(uint64_t k, uint64_t* warps) {
  const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  k = warp_max_u64(k);
  if (lane == 0) warps[warp] = k;
  __syncthreads();
  return warp_max_u64(warps[lane & (kScanWarps - 1)]);
}

__device__ __forceinline__ int32_t step(const VerifyArgs& a, int32_t s, int64_t t) {
  return (s < 0 || s >= a.num_states || t < 0 || t >= a.vocab_size)
             ? -1
             : __ldg(a.tok_next + static_cast<int64_t>(s) * a.vocab_size + t);
}

__device__ __forceinline__ int64_t first_row(const VerifyArgs& a, int32_t b) {
  return a.src_rows ? a.src_rows[b] : static_cast<int64_t>(b) * (a.max_drafts + 1);
}
__device__ __forceinline__ int64_t first_prob(const VerifyArgs& a, int32_t b) {
  return a.prob_rows ? a.prob_rows[b] : static_cast<int64_t>(b) * a.max_drafts;
}
__device__ __forceinline__ float heat_of(const VerifyArgs& a, int32_t b) {
  return a.temperature ? a.temperature[b] : a.temperature_all;
}

// ---------------------------------------------------------------------------
// One warp for a request, a lane for each position.

template <typename T>
__global__ void __launch_bounds__(128) walk_kernel(const VerifyArgs a, const Workspace w) {
  pdl_trigger();
  pdl_wait();
  const int32_t b = static_cast<int32_t>(blockIdx.x * 4 + (threadIdx.x >> 5));
  const int32_t lane = threadIdx.x & 31, K = a.max_drafts;
  if (b >= a.batch) return;
  const int32_t len = a.draft_lens ? a.draft_lens[b] : K;
  const int64_t first = first_row(a, b), pfirst = first_prob(a, b);
  const int64_t slot = a.slots ? a.slots[b] : b;
  const bool idle = len < 0 || len > K || first < 0 || first > a.src_total - 1 - len ||
                    (a.probs && len > 0 && (pfirst < 0 || pfirst > a.probs_total - len));
  if (lane == 0) w.request[b] = Request{idle ? -1 : len, len, 0, 0, 0};
  if (idle) {
    if (lane <= K) {
      a.tokens_out[static_cast<int64_t>(b) * (K + 1) + lane] = -1;
      a.logprobs_out[static_cast<int64_t>(b) * (K + 1) + lane] = 0.0f;
    }
    if (lane == 0) {
      a.counts_out[b] = 0;
      if (a.next_out) a.next_out[b] = a.tok_next ? a.state_pool[slot] : -2;
    }
    return;
  }
  Position p{-1, -1, -INFINITY, 1.0f, 0.0f, 0, -INFINITY, 0.0f, -1};
  if (lane < len) {
    const int64_t at = static_cast<int64_t>(b) * a.draft_stride + lane;
    const int64_t d = a.drafts_int64 ? static_cast<const int64_t*>(a.drafts)[at]
                                 : static_cast<const int32_t*>(a.drafts)[at];
    if (d >= 0 && d < a.vocab_size) p.draft = static_cast<int32_t>(d);
    if (heat_of(a, b) > 0.0f)
      p.uniform = a.uniforms[static_cast<int64_t>(b) * a.uniform_stride + lane];
    if (a.probs && p.draft >= 0)
      p.qd = load_prob(a.probs, a.probs_dtype, (pfirst + lane) * a.probs_stride + p.draft);
  }
  if (a.allow_bits) {
    if (a.path) {
      if (lane <= len) p.state = a.path[static_cast<int64_t>(b) * (K + 1) + lane];
    } else {
      int32_t s = a.state_pool[slot];
      for (int32_t i = 0; i <= len; ++i) {
        if (lane == i) p.state = s;
        s = i < len ? step(a, s, __shfl_sync(kFull, p.draft, i)) : -1;
      }
    }
  }
  if (p.draft >= 0 && Allow(a, p.state).has(p.draft))
    p.xd = fmaxf(Row<T>(a, first + lane).at(p.draft), -INFINITY);
  if (lane <= len) w.position[static_cast<int64_t>(b) * (K + 1) + lane] = p;
}

// ---------------------------------------------------------------------------
// What a thread keeps of a row that it scans: the maximum m and the sum of
// exp2((x - ref) c) with c = log2(e) / T. ref is not the maximum but some logit
// within kReach of it, so that it hardly ever changes. The difference comes first:
// ref c leaves the range of fp32 for logits like its lowest value and for the
// lowest temperatures, and above 2^29 is rounded by more than an exponential can
// take. (As x c - ref c, one multiply-add, 256 x 3 rows in fp32 took 118 us for
// 121 so, rows in 16 bits the same.)
struct Scan {
  static constexpr float kReach = 16.0f;
  float m = -INFINITY, ref = 0.0f, limit = -INFINITY, s = 0.0f;
  int32_t from = -1;         // the block whose vectors have m (-1: see idx)
  int32_t idx = INT_MAX;     // the first token that has m
  float score = -INFINITY;   // the race: log2 of this thread's best, less ref
  float bar = 0.0f;          // what it has to pass, times -1
  int32_t best = -1;
  __device__ __forceinline__ void raise(float top, float c) {
    if (top > limit) {  // the first value, or one far above it
      const float by = (ref - top) * c;
      s *= limit > -INFINITY ? exp2_fast(by) : 0.0f;
      score = limit > -INFINITY ? score + by : score;
      ref = top;
      limit = top + kReach * fminf(1.0f / c, 3.0e38f);
    }
  }
};

struct ScanShared {
  Lanes lanes;
  uint64_t warps[kScanWarps];
  unsigned long long lead;  // of a scan's race: a Lead
  float sums[kScanWarps];
  uint32_t bar;             // of a race by itself: a score
  int32_t last;
  __device__ __forceinline__ float bar_over(float ref, float c) const {
    return exp2_fast(
        Lead::of(*const_cast<const volatile unsigned long long*>(&lead)).from(ref, c));
  }
  // Raises the bar to this thread's best. Where another thread comes first the bar
  // stays as that one left it, which only has more scores looked at (trying again,
  // or a warp's best alone, took as long or up to 4 us more of 118).
  __device__ __forceinline__ void offer(const Scan& k, float c) {
    const Lead mine{k.ref, fminf(k.score, __log2f(kMostScore))};
    unsigned long long seen = *const_cast<volatile unsigned long long*>(&lead);
    if (mine.from(Lead::of(seen).ref, c) > Lead::of(seen).over) atomicCAS(&lead, seen, mine.bits());
  }
};

// Looks at four vectors of each lane, `word` their allow bits. kRace: with the
// noise, two at a time for the registers' sake.
template <typename T, bool RACE>
__device__ __forceinline__ void scan_block(const Row<T>& row, int32_t b, uint32_t word, float c,
                                           const float* noise, bool noise_fits, Scan& k,
                                           ScanShared& sh) {
  constexpr int kEpv = Row<T>::kEpv;
  constexpr int kAtOnce = RACE ? kRaceVecs : 4;
  const int32_t lane0 = b * 128 + static_cast<int32_t>(threadIdx.x & 31);
  auto vec_of = [&](int q) { return lane0 + q * 32; };
#pragma unroll
  for (int q0 = 0; q0 < 4; q0 += kAtOnce) {
    uint32_t keep[kAtOnce];
    uint4 v[kAtOnce];
    float e[RACE ? kAtOnce : 1][kEpv];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      keep[q] = Row<T>::keep(word, q0 + q);
      v[q] = uint4{};
      if (keep[q]) v[q] = row.vec(vec_of(q0 + q));
      if constexpr (RACE) {
        if (keep[q]) {
          load_floats<kEpv>(noise + row.token(vec_of(q0 + q)), noise_fits, e[q]);
        } else {
#pragma unroll
          for (int i = 0; i < kEpv; ++i) e[q][i] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) v[q] = masked<T>(v[q], keep[q], sh.lanes);
    uint4 larger = v[0];
    if constexpr (kAtOnce == 2) larger = vec_max2<T>(v[0], v[1]);
    if constexpr (kAtOnce == 4)
      larger = vec_max2<T>(vec_max2<T>(v[0], v[1]), vec_max2<T>(v[2], v[3]));
    const float top = vec_top<T>(larger);
    if (top > k.m) {
      k.from = b;
      k.idx = INT_MAX;
      k.m = top;
    }
    k.raise(top, c);
    if constexpr (RACE) k.bar = sh.bar_over(k.ref, c) * -kSlack;
    // ref is 0 as long as there is nothing but -inf: weights of 0
    const Pair c2 = pair_of(c, c), low = pair_of(-k.ref, -k.ref);
    const Pair bar2 = pair_of(k.bar, k.bar);
    Pair s = pair_of(0.0f, 0.0f);
    float w[RACE ? kAtOnce : 1][kEpv], over = 0.0f;
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
      for (int i = 0; i < kEpv; i += 2) {
        float lo, hi;
        split(mul2(add2(pair_of(Dt<T>::to_float(vec_get<T>(v[q], i)),
                                Dt<T>::to_float(vec_get<T>(v[q], i + 1))), low), c2), lo, hi);
        lo = exp2_fast(lo);
        hi = exp2_fast(hi);
        const Pair both = pair_of(lo, hi);
        s = add2(s, both);
        if constexpr (RACE) {
          w[q][i] = lo;
          w[q][i + 1] = hi;
          split(fma2(bar2, pair_of(e[q][i], e[q][i + 1]), both), lo, hi);
          over = fmaxf(over, fmaxf(lo, hi));
        }
      }
    float lo, hi;
    split(s, lo, hi);
    k.s += lo + hi;
    if constexpr (RACE) {
      if (over > 0.0f) {
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
          for (int i = 0; i < kEpv; ++i) {
            const float f = __log2f(w[q][i]) - __log2f(e[q][i]);
            if (f > k.score && w[q][i] > 0.0f) {
              k.score = f;
              k.best = row.token(vec_of(q0 + q)) + i;
            }
          }
        sh.offer(k, c);
      }
    }
  }
}

// The same for a block that allows few tokens: each lane goes through the
// tokens of its word, four at a time.
template <typename T, bool RACE>
__device__ __forceinline__ void scan_few(const Row<T>& row, int32_t b, uint32_t word, float c,
                                         const float* noise, Scan& k, ScanShared& sh) {
  const int32_t lane = threadIdx.x & 31, t0 = row.token(b * 128) + lane * 32;
  if (lane >= 4 * Row<T>::kEpv) word = 0;
  while (__any_sync(kFull, word != 0)) {
    int32_t t[4];
    float x[4], e[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      t[u] = t0 + __ffs(word) - 1;
      x[u] = -INFINITY;
      e[u] = 0.0f;
      if (word) {
        x[u] = row.at(t[u]);
        if (RACE) e[u] = __ldg(noise + t[u]);
      }
      word &= word - 1;
    }
    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if (top > k.m) {
      k.m = top;
      k.from = -1;
#pragma unroll
      for (int u = 3; u >= 0; --u)
        if (x[u] == top) k.idx = t[u];
    }
    k.raise(top, c);
    const float bar = RACE ? sh.bar_over(k.ref, c) * kSlack : 0.0f;
    float over = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x[u] = exp2_fast((x[u] - k.ref) * c);
      if (RACE) over = fmaxf(over, fmaf(-bar, e[u], x[u]));
    }
    k.s += (x[0] + x[1]) + (x[2] + x[3]);
    if (RACE && over > 0.0f) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float f = __log2f(x[u]) - __log2f(e[u]);
        if (f > k.score && x[u] > 0.0f) {
          k.score = f;
          k.best = t[u];
        }
      }
      sh.offer(k, c);
    }
  }
}

// Whether a block with this lane's word allows few tokens: an eighth.
template <typename T>
__device__ __forceinline__ bool few(uint32_t word) {
  const uint32_t lane = threadIdx.x & 31;
  return __reduce_add_sync(kFull, lane < 4 * Row<T>::kEpv ? __popc(word) : 0u) <=
         16u * Row<T>::kEpv;
}

// Calls f(block, its allow bits) for this warp's blocks of a chunk that allow
// any token, with the bits of the next two on their way.
template <typename T, typename F>
__device__ __forceinline__ void each_block(const Row<T>& row, const Allow& ok, int32_t chunk,
                                           int32_t chunks, int32_t V, F&& f) {
  int32_t first, end;
  row.chunk(chunk, chunks, first, end);
  int32_t b = first + static_cast<int32_t>(threadIdx.x >> 5);
  auto bits = [&](int32_t at) { return at < end ? row.bits(ok, at, V) : 0u; };
  uint32_t word = bits(b), next = bits(b + kScanWarps);
  for (; b < end; b += kScanWarps) {
    const uint32_t behind = bits(b + 2 * kScanWarps);
    if (__any_sync(kFull, word != 0)) f(b, word);
    word = next;
    next = behind;
  }
}

// A chunk of a row, by the whole CTA; all of it in the thread that the return
// value is true for. RACE: with the race of exp(x / T) / noise.
template <typename T, bool RACE>
__device__ __forceinline__ bool scan_chunk(const Row<T>& row, const Allow& ok, int32_t chunk,
                                           int32_t chunks, int32_t V, float inv, bool greedy,
                                           const float* noise, ScanShared& sh, Part& part) {
  constexpr int kEpv = Row<T>::kEpv;
  const float c = inv * kLog2e;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool noise_fits =
      RACE && (reinterpret_cast<uintptr_t>(noise + row.head) & 15u) == 0;
  Scan k;
  each_block(row, ok, chunk, chunks, V, [&](int32_t b, uint32_t word) {
    if (few<T>(word))
      scan_few<T, RACE>(row, b, word, c, noise, k, sh);
    else
      scan_block<T, RACE>(row, b, word, c, noise, noise_fits, k, sh);
  });
  row.edges(chunk, chunks, V, [&](int32_t t) {
    const float x = ok.has(t) ? fmaxf(row.at(t), -INFINITY) : -INFINITY;
    if (!(x > -INFINITY)) return;
    k.raise(x, c);
    if (x > k.m) {
      k.m = x;
      k.from = -1;
      k.idx = t;
    } else if (x == k.m) {
      k.idx = k.from < 0 ? min(k.idx, t) : t;
    }
    const float f = exp2_fast((x - k.ref) * c);
    k.s += f;
    if (RACE && __log2f(f) - __log2f(noise[t]) > k.score) k.best = t;
  });
  // the chunk's maximum, and where it is first
  float m = warp_max(k.m);
  if (lane == 0) sh.sums[warp] = m;
  __syncthreads();
  m = warp_max(sh.sums[lane & (kScanWarps - 1)]);
  int32_t idx = k.idx;
  uint64_t won = 0;
  part = Part{m, 0.0f, m > -INFINITY ? 0 : -1, -1, 0.0f, 1.0f};
  if (greedy && m > -INFINITY) {
    if (k.m != m) idx = INT_MAX;
    // The vectors of a round in which a lane met m: the warp looks at their
    // tokens together for the first one.
    uint32_t lanes = __ballot_sync(kFull, k.m == m && k.from >= 0);
    for (; lanes; lanes &= lanes - 1) {
      const int32_t l = __ffs(lanes) - 1, from = __shfl_sync(kFull, k.from, l);
#pragma unroll
      for (int q0 = 0; q0 < 4; q0 += 32 / kEpv) {
        const int32_t q = q0 + lane / kEpv;
        const int32_t j = from * 128 + q * 32 + l;
        const int32_t t = row.token(j) + lane % kEpv;
        if (j < row.vecs && ok.has(t) && row.at(t) == m) idx = min(idx, t);
      }
    }
    if (idx != INT_MAX) won = pack_arg(1u, idx);
  }
  // its best in the race, with full precision
  if (RACE && k.best >= 0) {
    part.x = row.at(k.best);
    part.e = noise[k.best];
    const float f = weight(part.x, m, inv);
    if (f > 0.0f) won = race_key(f / part.e, k.best);
  }
  const uint64_t mine = won;
  won = block_max(won, sh.warps);
  float s = warp_sum(k.m > -INFINITY ? k.s * exp2_fast((k.ref - m) * c) : 0.0f);
  if (lane == 0) sh.sums[warp] = s;
  __syncthreads();
  s = warp_sum(lane < kScanWarps ? sh.sums[lane] : 0.0f);
  // an infinite maximum, a NaN, or a temperature at either end of its range
  if (m > -INFINITY && !(s < INFINITY)) {
    s = 0.0f;
    row.each(chunk, chunks, V, [&](int32_t t) {
      if (ok.has(t)) s += weight(fmaxf(row.at(t), -INFINITY), m, inv);
    });
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sh.sums[warp] = s;
    __syncthreads();
    s = warp_sum(lane < kScanWarps ? sh.sums[lane] : 0.0f);
  }
  part.s = s;
  if (greedy && won) part.idx = unpack_idx(won);
  if (RACE && won) part.best = unpack_idx(won);
  // the winner knows its logit and noise
  return RACE && won ? mine == won : tid == 0;
}

// All chunks of a row put together by one warp, a lane for each; `best`: of
// the race (-1: none).
__device__ __forceinline__ Part join(const Part* parts, int32_t chunks, float inv) {
  const int32_t lane = threadIdx.x & 31;
  Part p{-INFINITY, 0.0f, -1, -1, 0.0f, 1.0f};
  if (lane < chunks) {
    const volatile Part* v = parts + lane;
    p.m = v->m;
    p.s = v->s;
    p.idx = v->idx;
    p.best = v->best;
    p.x = v->x;
    p.e = v->e;
  }
  const uint64_t top = warp_max_u64(p.idx < 0 ? 0 : pack_arg(order_key(p.m), p.idx));
  const float m = top ? key_value(static_cast<uint32_t>(top >> 32)) : -INFINITY;
  const float s = warp_sum(p.idx < 0 ? 0.0f : p.s * weight(p.m, m, inv));
  const float f = p.best >= 0 ? weight(p.x, m, inv) : 0.0f;
  const uint64_t best = warp_max_u64(f > 0.0f ? race_key(f / p.e, p.best) : 0);
  return Part{m, s, top ? unpack_idx(top) : -1, best ? unpack_idx(best) : -1, 0.0f, 1.0f};
}

// The drafts' rows.
template <typename T>
__global__ void __launch_bounds__(kScanThreads, kScanCtas)
    scan_kernel(const VerifyArgs a, const Workspace w, const int32_t chunks) {
  __shared__ ScanShared sh;
  const int32_t K = a.max_drafts;
  const int32_t chunk = static_cast<int32_t>(blockIdx.x % chunks);
  const int32_t b = static_cast<int32_t>(blockIdx.x / chunks % a.batch);
  const int32_t i = static_cast<int32_t>(blockIdx.x / chunks / a.batch);  // early ones first
  if (sizeof(typename Dt<T>::Bits) == 2) sh.lanes.fill();
  pdl_trigger();
  pdl_wait();
  Position& pos = w.position[static_cast<int64_t>(b) * (K + 1) + i];
  const int32_t len = w.request[b].len, state = pos.state;
  const float heat = heat_of(a, b);
  // one thread looks, since another CTA may be writing
  if (threadIdx.x == 0) sh.last = *const_cast<volatile int32_t*>(&w.request[b].end) < i;
  __syncthreads();
  if (i >= len || sh.last) return;  // no such row, or one behind a refused draft
  const bool greedy = !(heat > 0.0f);
  const float inv = greedy ? 1.0f : 1.0f / heat;
  Part* parts = w.part + (static_cast<int64_t>(b) * (K + 1) + i) * kMaxChunks;
  Part part;
  if (scan_chunk<T, false>(Row<T>(a, first_row(a, b) + i), Allow(a, state), chunk, chunks,
                           a.vocab_size, inv, greedy, nullptr, sh, part)) {
    parts[chunk] = part;
    __threadfence();
    sh.last = atomicAdd(&pos.arrived, 1u) == static_cast<uint32_t>(chunks) - 1;
  }
  __syncthreads();
  if (!sh.last || threadIdx.x >= 32) return;
  __threadfence();
  const Part all = join(parts, chunks, inv);
  if (threadIdx.x == 0) {
    pos.m = all.m;
    pos.s = all.s;
    pos.idx = all.idx;
    const bool accept = all.idx >= 0 && (greedy ? pos.draft == all.idx
                                                : pos.uniform * pos.qd <
                                                      weight(pos.xd, all.m, inv) / all.s);
    if (!accept) atomicMin(&w.request[b].end, i);
  }
}

// ---------------------------------------------------------------------------

// The best max(p - q, 0) / noise of chunk `chunk` of `chunks` of a row, with
// p = exp((x - m) / T) / s: (score, lowest index), 0 where nothing takes part.
// `without`: a token that takes no part (-1: none). By the whole CTA.
// Fast arithmetic says which tokens to look at, by a bound from above: what is left
// of a p that is hardly over q is all rounding there. p is taken as kOver times
// what fast arithmetic has, which differs from full precision by less (arguments of
// up to 126 rounded three times, 2^-16, and two exponentials). A thread keeps its
// best bound and the next one; its best token is scored in full, and where a next
// one may be better than the winner of all (scores within 2^-14 p / (p - q), in one
// thread) every token is. Scoring all that pass the bar in full took 56 us for 52
// (64 x 4 drafts with probabilities).
constexpr float kOver = 1.0f + 1.0f / 32768;

template <typename T>
__device__ __forceinline__ uint64_t race_chunk(const Row<T>& row, const Allow& ok, int32_t chunk,
                                               int32_t chunks, int32_t V, float inv, float m,
                                               float s, const float* noise, const Given& given,
                                               int32_t without, ScanShared& sh) {
  constexpr int kEpv = Row<T>::kEpv;
  constexpr int kAtOnce = 8 / kEpv;  // vectors: 16 tokens do not fit in the registers (56 us)
  const float c = inv * kLog2e, rz = 1.0f / s;
  auto exact = [&](int32_t t) -> uint64_t {
    if (t == without || !ok.has(t)) return 0;
    float left = weight(fmaxf(row.at(t), -INFINITY), m, inv) * rz;
    if (given.p) left -= load_prob(given.p, given.dtype, t);
    return left > 0.0f ? race_key(left / noise[t], t) : 0;
  };
  uint64_t won = 0;
  auto offer = [&](int32_t t) {
    const uint64_t k = exact(t);
    won = k > won ? k : won;
  };
  __syncthreads();
  if (threadIdx.x == 0) sh.bar = 0;
  __syncthreads();
  if (!(m < INFINITY && c < INFINITY)) {
    row.each(chunk, chunks, V, offer);
    return block_max(won, sh.warps);
  }
  const float most = rz * kOver, gap = rz * (3.0f * (kOver - 1.0f));
  float top = -1.0f, next = -1.0f, low = 0.0f;  // bounds from above, and one from below
  int32_t idx = -1;
  const bool noise_fits = (reinterpret_cast<uintptr_t>(noise + row.head) & 15u) == 0;
  const bool given_fits = given.p && given.template fits<kEpv>(row.head);
  // `up` is the bound of what is left
  auto look = [&](float up, float x, float e, int32_t t) {
    if (!(up > 0.0f)) return;  // nothing left, or no token
    const float by = __fdividef(1.0f, e), f = up * by;
    next = fmaxf(next, fminf(top, f));
    if (f > top) idx = t;
    top = fmaxf(top, f);
    low = fmaxf(low, fmaf(exp2_fast((x - m) * c), -gap, up) * by);
  };
  auto raise = [&] {
    if (low > 0.0f) atomicMax(&sh.bar, __float_as_uint(fminf(low, kMostScore)));
  };
  // a block that allows few tokens: each lane goes through those of its word
  auto few_of = [&](int32_t b, uint32_t word) {
    const int32_t lane = threadIdx.x & 31, t0 = row.token(b * 128) + lane * 32;
    if (lane >= 4 * kEpv) word = 0;
    while (__any_sync(kFull, word != 0)) {
      int32_t t[4];
      float x[4], e[4], up[4], over = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        t[u] = t0 + __ffs(word) - 1;
        const bool in = word != 0 && t[u] != without;
        x[u] = in ? row.at(t[u]) : -INFINITY;
        e[u] = in ? __ldg(noise + t[u]) : 0.0f;
        up[u] = in && given.p ? load_prob(given.p, given.dtype, t[u]) : 0.0f;
        word &= word - 1;
      }
      const float bar = __uint_as_float(*const_cast<volatile uint32_t*>(&sh.bar)) * kSlack;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        up[u] = fmaf(exp2_fast((x[u] - m) * c), most, -up[u]);
        over = fmaxf(over, fmaf(-bar, e[u], up[u]));
      }
      if (over > 0.0f) {
#pragma unroll
        for (int u = 0; u < 4; ++u) look(up[u], x[u], e[u], t[u]);
        raise();
      }
    }
  };
  auto block = [&](int32_t b, uint32_t word) {
    if (few<T>(word)) {
      few_of(b, word);
      return;
    }
    const int32_t j0 = b * 128 + static_cast<int32_t>(threadIdx.x & 31);
#pragma unroll
    for (int q0 = 0; q0 < 4; q0 += kAtOnce) {
      uint32_t keep[kAtOnce];
      uint4 v[kAtOnce];
      float e[kAtOnce][kEpv], left[kAtOnce][kEpv];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        keep[q] = Row<T>::keep(word, q0 + q);
        const int32_t j = j0 + (q0 + q) * 32, t = row.token(j);
#pragma unroll
        for (int i = 0; i < kEpv; ++i) left[q][i] = 0.0f;
        if (keep[q]) {
          v[q] = row.vec(j);
          load_floats<kEpv>(noise + t, noise_fits, e[q]);
          if (given.p) given.load<kEpv>(t, given_fits, left[q]);
          if (static_cast<uint32_t>(without - t) < static_cast<uint32_t>(kEpv))
            keep[q] &= ~(1u << (without - t));
        }
      }
      const float bar = __uint_as_float(*const_cast<volatile uint32_t*>(&sh.bar)) * kSlack;
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        if (!keep[q]) continue;
        const uint4 x = masked<T>(v[q], keep[q], sh.lanes);
        float over = 0.0f;
#pragma unroll
        for (int i = 0; i < kEpv; ++i) {
          const float f = exp2_fast((Dt<T>::to_float(vec_get<T>(x, i)) - m) * c);
          left[q][i] = fmaf(f, most, -left[q][i]);
          over = fmaxf(over, (keep[q] >> i) & 1u ? fmaf(-bar, e[q][i], left[q][i]) : 0.0f);
        }
        if (over > 0.0f) {
#pragma unroll
          for (int i = 0; i < kEpv; ++i)
            if ((keep[q] >> i) & 1u)
              look(left[q][i], Dt<T>::to_float(vec_get<T>(x, i)), e[q][i],
                   row.token(j0 + (q0 + q) * 32) + i);
          raise();
        }
      }
    }
  };
  each_block(row, ok, chunk, chunks, V, block);
  if (idx >= 0) offer(idx);
  row.edges(chunk, chunks, V, offer);
  const uint64_t best = block_max(won, sh.warps);
  const float score = __uint_as_float(static_cast<uint32_t>(best >> 32));
  if (!__syncthreads_or(next > score * kSlack)) return best;
  row.each(chunk, chunks, V, offer);
  return block_max(won, sh.warps);
}

// The row behind a request's accepted drafts, and the results.
template <typename T>
__global__ void __launch_bounds__(kScanThreads, kLastCtas)
    last_kernel(const VerifyArgs a, const Workspace w, const int32_t chunks) {
  __shared__ ScanShared sh;
  const int32_t chunk = static_cast<int32_t>(blockIdx.x % chunks);
  const int32_t b = static_cast<int32_t>(blockIdx.x / chunks);
  const int32_t tid = threadIdx.x, lane = tid & 31, K = a.max_drafts, V = a.vocab_size;
  if (sizeof(typename Dt<T>::Bits) == 2) sh.lanes.fill();
  if (tid == 0) sh.lead = Lead{-FLT_MAX, -INFINITY}.bits();  // below any score
  pdl_trigger();
  pdl_wait();
  Request& request = w.request[b];
  const int32_t len = request.len, n = request.end;
  if (len < 0) return;
  const float heat = heat_of(a, b);
  const bool greedy = !(heat > 0.0f);
  const float inv = greedy ? 1.0f : 1.0f / heat;
  const Position* positions = w.position + static_cast<int64_t>(b) * (K + 1);
  Position p = positions[n];
  const Row<T> row(a, first_row(a, b) + n);
  const Allow ok(a, p.state);
  const float* noise = a.noise + static_cast<int64_t>(b) * a.noise_stride;
  __syncthreads();
  int64_t token = -1;
  bool open = false;  // the race is still to be run, over p
  if (n == len) {
    Part* parts = w.part + (static_cast<int64_t>(b) * (K + 1) + n) * kMaxChunks;
    Part part;
    if (greedy ? scan_chunk<T, false>(row, ok, chunk, chunks, V, inv, true, nullptr, sh, part)
               : scan_chunk<T, true>(row, ok, chunk, chunks, V, inv, false, noise, sh, part)) {
      parts[chunk] = part;
      __threadfence();
      sh.last = atomicAdd(&request.arrived, 1u) == static_cast<uint32_t>(chunks) - 1;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    part = join(parts, chunks, inv);  // by each warp alike
    p.m = part.m;
    p.s = part.s;
    p.idx = part.idx;
    if (p.idx >= 0) token = greedy ? p.idx : part.best;
    open = !greedy && p.idx >= 0 && (part.best < 0 || !(p.m < INFINITY));
  } else if (greedy || p.idx < 0) {
    if (chunk != 0) return;
    token = p.idx;
  } else {
    Given given{nullptr, a.probs_dtype};
    if (a.probs)
      given.p = static_cast<const uint8_t*>(a.probs) +
                (first_prob(a, b) + n) * a.probs_stride * given.size();
    uint64_t won = race_chunk<T>(row, ok, chunk, chunks, V, inv, p.m, p.s, noise, given,
                                 a.probs ? -1 : p.draft, sh);
    if (tid == 0) {
      if (won) atomicMax(&request.race, static_cast<unsigned long long>(won));
      __threadfence();
      sh.last = atomicAdd(&request.arrived, 1u) == static_cast<uint32_t>(chunks) - 1;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    won = *const_cast<volatile unsigned long long*>(&request.race);
    if (won)
      token = unpack_idx(won);
    else
      open = true;  // nothing left of p - q
  }
  if (open) {
    const uint64_t won =
        race_chunk<T>(row, ok, 0, 1, V, inv, p.m, p.s, noise, Given{nullptr, 0}, -1, sh);
    token = won ? unpack_idx(won) : -1;
  }
  if (tid >= 32) return;
  // a lane for each position
  const int64_t out = static_cast<int64_t>(b) * (K + 1) + lane;
  if (lane <= K) {
    int64_t t = -1;
    float logprob = 0.0f;
    if (lane < n) {
      const Position& mine = positions[lane];
      t = mine.draft;
      logprob = (mine.xd == mine.m ? 0.0f : (mine.xd - mine.m) * inv) - logf(mine.s);
    } else if (lane == n && token >= 0) {
      const float x = row.at(token);
      t = token;
      logprob = (x == p.m ? 0.0f : (x - p.m) * inv) - logf(p.s);
    }
    a.tokens_out[out] = t;
    a.logprobs_out[out] = logprob;
  }
  if (lane == 0) {
    a.counts_out[b] = n + (token >= 0);
    if (a.tok_next) {
      const int32_t next = token < 0 ? -1 : step(a, p.state, token);
      if (a.next_out) a.next_out[b] = next;
      if (a.write_back) a.state_pool[a.slots ? a.slots[b] : b] = next;
    } else if (a.next_out) {
      a.next_out[b] = token < 0 ? -1 : p.state;
    }
  }
}

// ---------------------------------------------------------------------------

// Chunks of a row, each a CTA: by what `rows` of them cost on `room` places,
// where a chunk costs its share of the row and a twentieth of a row besides
// (the loads that depend on one another, 3 us), and the last ones leave places
// idle for half their time. No chunk has less than a block of 128 vectors for
// every warp. Measured: 1024 rows of 128,256 in 16 bits with noise 141 us in
// one or two chunks, 146 in four; 128 rows x 2 drafts 58 us in one, 46 in four.
int32_t chunks_of(int64_t rows, int32_t vocab, int32_t vec, int64_t room) {
  const int64_t most =
      std::min<int64_t>(kMaxChunks, (static_cast<int64_t>(vocab) / vec + 1023) / 1024);
  int32_t best = 1;
  double least = 0.0;
  for (int32_t c = 1; c <= most; ++c) {
    const double waves = static_cast<double>(rows * c) / room;
    const double cost = std::max(1.0, waves) * (1.0 / c + 0.05) + (waves > 1.0 ? 0.5 / c : 0.0);
    if (c == 1 || cost < least) {
      least = cost;
      best = c;
    }
  }
  return best;
}

size_t lay_out(int32_t batch, int32_t max_drafts, void* base, Workspace* w) {
  const size_t rows = static_cast<size_t>(batch) * (max_drafts + 1);
  const size_t position = align256(batch * sizeof(Request));
  const size_t part = position + align256(rows * sizeof(Position));
  if (w) {
    uint8_t* p = static_cast<uint8_t*>(base);
    w->request = reinterpret_cast<Request*>(p);
    w->position = reinterpret_cast<Position*>(p + position);
    w->part = reinterpret_cast<Part*>(p + part);
  }
  return part;
}

}  // namespace
}  // namespace bpd

using namespace bpd;

extern "C" size_t bpd_verify_workspace_bytes(int32_t batch, int32_t max_drafts) {
  batch = std::max(batch, 1);
  max_drafts = std::max(max_drafts, 0);
  return lay_out(batch, max_drafts, nullptr, nullptr) +
         align256(static_cast<size_t>(batch) * (max_drafts + 1) * kMaxChunks * sizeof(Part));
}

extern "C" bpd_status bpd_verify_drafts(const bpd_verify_args* args, void* stream) {
  const char* what = "bpd_verify_drafts";
  BPD_REQUIRE(args, "%s: null pointer", what);
  bpd_verify_args a = *args;
  BPD_REQUIRE(a.batch >= 0 && a.vocab_size > 0 && a.max_drafts >= 0 && a.src_total >= 0,
              "%s: bad sizes", what);
  if (a.max_drafts > BPD_MAX_DRAFTS)
    return fail(BPD_ERR_CAPACITY, "%s: more than %d drafts", what, BPD_MAX_DRAFTS);
  if (a.batch == 0) return BPD_OK;
  BPD_REQUIRE(a.src && a.tokens_out && a.counts_out && a.logprobs_out && a.workspace,
              "%s: null pointer", what);
  BPD_REQUIRE(aligned16(a.workspace), "%s: the workspace must be 16-byte aligned", what);
  BPD_REQUIRE(a.src_stride >= a.vocab_size, "%s: row stride < vocab", what);
  BPD_REQUIRE(a.max_drafts == 0 || (a.drafts && a.draft_stride >= a.max_drafts),
              "%s: drafts missing, or their row stride < max_drafts", what);
  const bool all_greedy = a.temperature == nullptr && !(a.temperature_all > 0.0f);
  BPD_REQUIRE(all_greedy || (a.noise && a.noise_stride >= a.vocab_size),
              "%s: sampling needs a row of noise for each request", what);
  BPD_REQUIRE(all_greedy || a.max_drafts == 0 ||
                  (a.uniforms && a.uniform_stride >= a.max_drafts),
              "%s: sampling needs a uniform number for each draft", what);
  BPD_REQUIRE(!a.probs || (a.probs_stride >= a.vocab_size && a.probs_total >= 0 &&
                           a.probs_dtype >= BPD_F32 && a.probs_dtype <= BPD_F16),
              "%s: bad draft probabilities", what);
  BPD_REQUIRE(!a.allow_bits ||
                  (a.words_stride >= (a.vocab_size + 31) / 32 && a.num_states > 0),
              "%s: words_stride too small, or no states", what);
  BPD_REQUIRE(!a.allow_bits || a.path || (a.state_pool && a.tok_next),
              "%s: a grammar needs state_pool and tok_next, or path", what);
  const bool walks = a.state_pool && a.tok_next && a.allow_bits;
  BPD_REQUIRE(!a.write_back || walks, "%s: write_back needs state_pool, allow_bits and tok_next",
              what);
  BPD_REQUIRE(!a.next_out || walks || (a.path && a.allow_bits && !a.tok_next),
              "%s: next_out needs state_pool, allow_bits and tok_next, or path without tok_next",
              what);
  if (!a.allow_bits) a.tok_next = nullptr;
  cudaStream_t st = as_stream(stream);
  return with_dtype(a.src_dtype, what, [&](auto tag) {
    using T = decltype(tag);
    const int64_t rows = static_cast<int64_t>(a.batch) * a.max_drafts, sms = sm_count();
    Workspace w{};
    lay_out(a.batch, a.max_drafts, a.workspace, &w);
    const int32_t chunks =
        chunks_of(rows, a.vocab_size, Dt<T>::kPerVec, kScanCtas * sms);
    const int32_t lasts =
        chunks_of(a.batch, a.vocab_size, Dt<T>::kPerVec, kLastCtas * sms);
    if (std::max(rows * chunks, static_cast<int64_t>(a.batch) * lasts) > INT_MAX)
      return fail(BPD_ERR_CAPACITY, "%s: batch too large", what);
    cudaError_t e = launch_pdl(walk_kernel<T>, dim3((a.batch + 3) / 4), dim3(128), 0, st, a, w);
    if (e == cudaSuccess && a.max_drafts)
      e = launch_pdl(scan_kernel<T>, dim3(static_cast<unsigned>(rows * chunks)),
                     dim3(kScanThreads), 0, st, a, w, chunks);
    if (e == cudaSuccess)
      e = launch_pdl(last_kernel<T>, dim3(static_cast<unsigned>(a.batch) * lasts),
                     dim3(kScanThreads), 0, st, a, w, lasts);
    return e == cudaSuccess ? BPD_OK : fail(BPD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  });
}
