// Beam search's selection: the best continuations of a request's beams over
// the vocabulary.
//
// For beam w of request b with logits x[0, V) and accumulated score c:
//   lse   = log sum_v exp(x[v])                       (rounded to fp32)
//   score = c + (x[v] - lse)                          (ordered in fp64)
// and the K best (beam, token) pairs of a request, best first; equal scores by
// the lowest beam, then, inside a beam, by the larger logit (distinct logits
// can meet in one fp64 score when c is huge or they are tiny) and the lowest
// token. A row's order is so its logits' order: each chunk of a row yields its
// own K best and its share of the sum in one pass over the logits (the only
// large traffic: bound by HBM), and a second launch joins the chunks of a
// request.
//
// Chunk pass: a CTA streams its chunk once, two 16-byte vectors a thread at a
// time with four more on their way; each thread keeps its own maximum and
// the sum relative to it, so nothing waits on another thread until the end.
// Of the 256 threads' maxima each warp's four best are looked at; the K-th of
// those 32 is a threshold that at least K logits reach and few others do. The
// threads whose maximum reaches it (about K of 256) have the steps that hold
// their two largest maxima searched, which every thread keeps in shared memory
// (all their logits are read again if a third step reaches it too), and what
// passes is ranked by counting. (Reading the step again instead of keeping it
// took 3 us of a CTA's 19, now 0.9.) Many threads reach it only when many
// logits are equal to it (masked or constant rows): then the ones above it and,
// in index order, as many equal ones as are missing are taken, from memory
// again. So a vocabulary masked down to fewer than K tokens a chunk, by -inf or
// by a finite mask, is read three times (64 x 8 beams over 128256, bf16: 36.7 us
// unmasked, 37.8 with 1 in 100 tokens left, 81 with 16 of them). If more than
// kBeamCap lie above it (a layout against the threads' order), K rounds of a
// block-wide maximum give the same result.
#pragma once

#include "pa_common.cuh"

namespace pa {

constexpr int kBeamThreads = 256;
constexpr int kBeamCtas = 5;    // per SM, of 40 KB (4 with a deeper ring: 37.5 for 37.2 us)
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamMaxK = 32;   // the threshold looks at 32 maxima
constexpr int kBeamMaxBeams = 256;      // JoinKey's 8 bits
constexpr int kBeamMaxVocab = 1 << 24;  // and 24
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBeamCap = 1024;  // elements ranked by counting
constexpr int kBeamMany = 128;  // threads at the threshold: many logits are equal to it
constexpr int kBeamStep = 2;    // vectors of a thread taken together
constexpr int kBeamRing = 3;    // such steps in flight
constexpr float kBeamSlack = 5.f;
constexpr int kBeamRingBytes = kBeamRing * kBeamStep * kBeamThreads * 16;
constexpr int kBeamSmem = kBeamRingBytes + 2 * kBeamStep * kBeamThreads * 16;  // and two steps kept
static_assert(kBeamRingBytes >= kBeamCap * 8, "the ring holds the candidates at the end");

struct BeamParams {
  const void* logits;
  int64_t stride_b, stride_w;  // elements
  const float* scores;         // [batch, beams]
  int64_t score_stride;
  int32_t batch, beams, vocab, k;
  int32_t chunks, chunk_vectors;  // per row; 16-byte vectors of each thread per chunk
  double* part_off;   // [rows, chunks]: max * log2(e); -inf: nothing finite
  double* part_sum;   // [rows, chunks]: sum of exp(x - max)
  uint64_t* part_key;  // [rows, chunks, k]: best first, 0: none
  float* out_scores;  // [batch, k]
  int32_t* out_parents;
  int32_t* out_tokens;
};

// Order-preserving map of a float (no NaN, no -0) to unsigned, and back.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t order_bits64(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x));
  return b ^ ((b >> 63) ? 0xffffffffffffffffULL : 0x8000000000000000ULL);
}
__device__ __forceinline__ double order_value64(uint64_t k) {
  return __longlong_as_double(
      static_cast<long long>(k ^ ((k >> 63) ? 0x8000000000000000ULL : 0xffffffffffffffffULL)));
}

// (value, index) as one key: larger value first, then the lower index.
__device__ __forceinline__ uint64_t beam_key(float x, int idx) {
  return (static_cast<uint64_t>(order_bits(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(idx));
}

// A candidate of the join, compared as one unsigned number: the score, then
// beam (lower first), logit, token (lower first).
struct JoinKey {
  uint64_t score;
  uint64_t rest;  // 255 - beam : 8, logit's order bits : 32, 2^24 - 1 - token : 24
  __device__ __forceinline__ bool operator>(const JoinKey& o) const {
    return score > o.score || (score == o.score && rest > o.rest);
  }
};
__device__ __forceinline__ uint64_t shfl_xor_key(uint64_t k, int m) {
  return __shfl_xor_sync(0xffffffffu, k, m);
}
__device__ __forceinline__ JoinKey shfl_xor_key(const JoinKey& k, int m) {
  return JoinKey{__shfl_xor_sync(0xffffffffu, k.score, m),
                 __shfl_xor_sync(0xffffffffu, k.rest, m)};
}
// Threshold that at least k <= 32 of the threads' keys reach, or 0 if fewer
// than k threads have one (0: none); *top receives the largest key. One
// barrier. s_four: four keys per warp.
__device__ __forceinline__ uint32_t block_threshold(uint32_t key, int k, uint32_t* s_four, int lane,
                                                    int wid, uint32_t* top) {
  uint32_t left = key;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, left);
    if (lane == 0) s_four[wid * 4 + i] = m;
    const uint32_t who = __ballot_sync(0xffffffffu, left == m);
    if (lane == __ffs(who) - 1) left = 0;
  }
  __syncthreads();
  const uint32_t mine = s_four[lane];
  int reach = 0;  // how many of the 32 are at least mine
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 o = reinterpret_cast<const uint4*>(s_four)[i];
    reach += (o.x >= mine) + (o.y >= mine) + (o.z >= mine) + (o.w >= mine);
  }
  *top = __reduce_max_sync(0xffffffffu, mine);
  return __reduce_max_sync(0xffffffffu, reach >= k ? mine : 0u);
}

template <typename K>
__device__ __forceinline__ K block_max(K best, K* s_key, int lane, int wid) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const K o = shfl_xor_key(best, off);
    if (o > best) best = o;
  }
  __syncthreads();  // s_key may still be read
  if (lane == 0) s_key[wid] = best;
  __syncthreads();
  K t = s_key[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w)
    if (s_key[w] > t) t = s_key[w];
  return t;
}

// Logits as they lie in memory, one 32-bit word at a time: one fp32 or two
// 16-bit values, whose maxima and comparisons work on both at once.
template <typename T>
struct BeamWord;

template <>
struct BeamWord<float> {
  static constexpr int N = 1;
  static constexpr uint32_t kNone = 0xff800000u;  // -inf
  static constexpr float kMost = 3.402823466e38f;
  // NaN becomes -inf, +inf the largest finite value
  static __device__ __forceinline__ uint32_t clean(uint32_t w) {
    return __float_as_uint(fminf(fmaxf(__uint_as_float(w), -INFINITY), 3.402823466e38f));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float at(uint32_t w, int) { return __uint_as_float(w); }
  // the word's first n values, -inf for the others
  static __device__ __forceinline__ uint32_t first(uint32_t w, int n) { return n > 0 ? w : kNone; }
};

template <typename T, typename T2>
struct BeamWord16 {
  static constexpr int N = 2;
  static __device__ __forceinline__ T2 val(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  static __device__ __forceinline__ uint32_t raw(T2 v) {
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return raw(__hmax2(val(a), val(b)));
  }
};
template <>
struct BeamWord<__nv_bfloat16> : BeamWord16<__nv_bfloat16, __nv_bfloat162> {
  static constexpr uint32_t kNone = 0xff80ff80u;
  static constexpr float kMost = 3.3895313892515355e38f;
  static __device__ __forceinline__ uint32_t first(uint32_t w, int n) {
    return n >= 2 ? w : n == 1 ? (w & 0xffffu) | (kNone << 16) : kNone;
  }
  static __device__ __forceinline__ uint32_t clean(uint32_t w) {
    return raw(__hmin2(__hmax2(val(w), val(kNone)), val(0x7f7f7f7fu)));
  }
  static __device__ __forceinline__ float at(uint32_t w, int i) {
    return __uint_as_float(i ? w & 0xffff0000u : w << 16);
  }
};
template <>
struct BeamWord<__half> : BeamWord16<__half, __half2> {
  static constexpr uint32_t kNone = 0xfc00fc00u;
  static constexpr float kMost = 65504.f;
  static __device__ __forceinline__ uint32_t first(uint32_t w, int n) {
    return n >= 2 ? w : n == 1 ? (w & 0xffffu) | (kNone << 16) : kNone;
  }
  static __device__ __forceinline__ uint32_t clean(uint32_t w) {
    return raw(__hmin2(__hmax2(val(w), val(kNone)), val(0x7bff7bffu)));
  }
  static __device__ __forceinline__ float at(uint32_t w, int i) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(i ? w >> 16 : w)));
  }
};

// 16 bytes at `p` (any alignment that is a multiple of the element's), of
// which the first `bytes` > 0 exist: the aligned 16-byte blocks that hold at
// least one of them are read and shifted together. What lies behind `bytes`
// is not to be used.
__device__ __forceinline__ uint4 load16_any(const uint8_t* p, int bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint4* block = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
  const int off = static_cast<int>(a & 15);
  uint4 v = __ldg(block);
  if (off == 0) return v;
  uint4 n = off + bytes > 16 ? __ldg(block + 1) : make_uint4(0, 0, 0, 0);
  if (off & 8) v = make_uint4(v.z, v.w, n.x, n.y), n = make_uint4(n.z, n.w, 0, 0);
  if (off & 4) v = make_uint4(v.y, v.z, v.w, n.x), n = make_uint4(n.y, n.z, n.w, 0);
  if (off & 2)
    v = make_uint4(__funnelshift_r(v.x, v.y, 16), __funnelshift_r(v.y, v.z, 16),
                   __funnelshift_r(v.z, v.w, 16), __funnelshift_r(v.w, n.x, 16));
  return v;
}

// One chunk of one row. Vector i of thread t holds logits base + (i * 256 + t)
// * N and the N - 1 after it whatever the row's alignment, so equal rows give
// equal sums; places past the row hold -inf.
//
// Per logit: half an instruction of packed maxima and 3.5 for the sum (unpack,
// ex2, and subtract, multiply and add for two at a time: 36.9 us where one at
// a time takes 37.7. x log2(e) - ref log2(e) in one fma took 37.4; its rounding
// overflows ex2 for huge logits and costs a certain token its log probability
// of 0). ex2 is the narrowest pipe (16 per
// SM and cycle: 128256 logits of 512 rows take 14.4 us of it, and 20.1 us of
// HBM). NaN needs no instruction of its own: maxima and comparisons pass over
// it, and a thread whose sum is not finite adds its logits up again, cleaned.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, kBeamCtas) beam_chunk_kernel(const BeamParams p) {
  using W = BeamWord<T>;
  constexpr int N = 16 / sizeof(T);
  constexpr int kRow = kBeamThreads * N;  // logits per vector of all threads
  __shared__ alignas(16) uint32_t s_four[32];
  __shared__ uint64_t s_key[kBeamWarps];
  __shared__ double s_sum[kBeamWarps];
  __shared__ int s_warp[kBeamWarps];
  extern __shared__ uint4 ring[];  // kBeamRing steps
  uint64_t* const s_cand = reinterpret_cast<uint64_t*>(ring);  // [kBeamCap], once they are taken
  uint4* const keep = ring + kBeamRing * kBeamStep * kBeamThreads;  // two steps of each thread
  __shared__ int s_who[2 * kBeamMany];
  __shared__ int s_n, s_one, s_all;
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  // rows first: the rows' last chunks, which may be shorter, start last
  const int b = blockIdx.x / p.beams, w = blockIdx.x - b * p.beams, chunk = blockIdx.y;
  const int64_t part = static_cast<int64_t>(blockIdx.x) * p.chunks + chunk;
  const T* x = static_cast<const T*>(p.logits) + b * p.stride_b + w * p.stride_w;
  const int base = chunk * p.chunk_vectors * kRow, K = p.k;
  const int vectors = min(p.chunk_vectors, (p.vocab - base + kRow - 1) / kRow);  // > 0
  if (tid == 0) s_n = s_one = s_all = 0;
  // a beam without a score continues nothing: all its logits count as -inf
  const float c0 = __ldg(p.scores + b * p.score_stride + w);
  const bool dead = !(c0 > -INFINITY);

  // vector i of this thread, whatever its alignment; places past the row: -inf
  auto load = [&](int i) {
    uint4 r = make_uint4(W::kNone, W::kNone, W::kNone, W::kNone);
    const int at = base + (i * kBeamThreads + tid) * N;
    const int left = dead ? 0 : p.vocab - at;
    if (left <= 0) return r;
    r = load16_any(reinterpret_cast<const uint8_t*>(x + at),
                   min(left, N) * static_cast<int>(sizeof(T)));
    if (left < N) {
      r.x = W::first(r.x, left);
      r.y = W::first(r.y, left - W::N);
      r.z = W::first(r.z, left - 2 * W::N);
      r.w = W::first(r.w, left - 3 * W::N);
    }
    return r;
  };
  // vectors whose logits of every thread are inside the row and aligned
  const bool aligned = (reinterpret_cast<uintptr_t>(x + base) & 15) == 0;
  const int whole = aligned && !dead ? min(vectors, (p.vocab - base) / kRow) : 0;
  const uint4* src = reinterpret_cast<const uint4*>(x + base) + tid;
  float best = -INFINITY;
  // the sum of exp(x - ref); ref follows the maximum only when it has grown by
  // kBeamSlack (each time costs the sum one rounding of ex2), and is 0 before
  // the first finite logit
  float ref = 0.f, move = -INFINITY;  // move: where ref follows
  double my_sum = 0.0;
  // The two steps with the largest maxima are kept, slot of `best` and the
  // other one, and the largest logit of all others: nearly every logit that
  // the threshold lets through is then at hand.
  float second = -INFINITY, third = -INFINITY;
  int best_step = 0, second_step = 0, slot = 0;
  auto save = [&](const uint4 (&in)[kBeamStep], int to) {
#pragma unroll
    for (int u = 0; u < kBeamStep; ++u) keep[(to * kBeamStep + u) * kBeamThreads + tid] = in[u];
  };
  auto take = [&](const uint4 (&in)[kBeamStep], int step) {
    uint32_t v[kBeamStep][4];
#pragma unroll
    for (int u = 0; u < kBeamStep; ++u) {
      v[u][0] = in[u].x;
      v[u][1] = in[u].y;
      v[u][2] = in[u].z;
      v[u][3] = in[u].w;
    }
    uint32_t m2 = W::kNone;
#pragma unroll
    for (int u = 0; u < kBeamStep; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) m2 = W::max2(m2, v[u][q]);
    const float m = W::N == 2 ? fmaxf(W::at(m2, 0), W::at(m2, 1)) : W::at(m2, 0);
    if (m > best) {
      third = second;
      second = best;
      best = m;
      second_step = best_step;
      best_step = step;
      slot ^= 1;
      save(in, slot);
      if (m > move) {
        if (move != -INFINITY) my_sum *= ex2((ref - m) * kLog2e);  // (before that it is 0 or NaN)
        ref = m;
        move = m + kBeamSlack;
      }
    } else if (m > second) {
      third = second;
      second = m;
      second_step = step;
      save(in, slot ^ 1);
    } else {
      third = fmaxf(third, m);
    }
    // (two at a time: one word of 16-bit logits, two of fp32)
    const F32x2 minus_ref(-ref, -ref), scale(kLog2e, kLog2e);
    F32x2 part[2] = {F32x2(0.f, 0.f), F32x2(0.f, 0.f)};
    constexpr int kPair = 3 - W::N;  // words of a pair
#pragma unroll
    for (int u = 0; u < kBeamStep; ++u)
#pragma unroll
      for (int q = 0; q < 4; q += kPair) {
        const F32x2 x(W::at(v[u][q], 0),
                      W::N == 2 ? W::at(v[u][q], 1) : W::at(v[u][(q + 1) & 3], 0));
        const F32x2 t = (x + minus_ref) * scale;
        F32x2& p2 = part[q / kPair & 1];
        p2 = p2 + F32x2(ex2(t.lo()), ex2(t.hi()));
      }
    const F32x2 both = part[0] + part[1];
    my_sum += both.lo() + both.hi();
  };
  // Steps of whole vectors first, through a ring of shared memory in which
  // every thread copies and reads its own slots (no barrier), kBeamRing steps
  // in flight. (Loads into registers, each behind its own bounds check, took
  // 47 us where the ring took 38: 512 rows of 128256 bf16.)
  const int steps = whole / kBeamStep;
  auto copy = [&](int step) {
    if (step < steps) {
#pragma unroll
      for (int u = 0; u < kBeamStep; ++u)
        copy_async16(ring + ((step % kBeamRing) * kBeamStep + u) * kBeamThreads + tid,
                     src + (step * kBeamStep + u) * kBeamThreads);
    }
    copy_async_commit();  // (an empty group keeps the count)
  };
  uint4 now[kBeamStep];
  for (int i = 0; i < kBeamRing; ++i) copy(i);
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    copy_async_wait<kBeamRing - 1>();
#pragma unroll
    for (int u = 0; u < kBeamStep; ++u)
      now[u] = ring[((i % kBeamRing) * kBeamStep + u) * kBeamThreads + tid];
    take(now, i);
    copy(i + kBeamRing);
  }
  copy_async_wait<0>();
#pragma unroll 1
  for (int i = steps * kBeamStep; i < vectors; i += kBeamStep) {
#pragma unroll
    for (int u = 0; u < kBeamStep; ++u)
      now[u] = i + u < vectors ? load(i + u)
                               : make_uint4(W::kNone, W::kNone, W::kNone, W::kNone);
    take(now, i / kBeamStep);
  }
  // 0: no logit here. (+ 0.f: -0 and +0 are one value)
  const uint32_t mine =
      base + tid * N < p.vocab ? order_bits(fminf(best, W::kMost) + 0.f) : 0u;
  uint32_t top;
  const uint32_t least = block_threshold(mine, K, s_four, lane, wid, &top);
  const float m = order_value(top);  // the chunk is not empty
  // Threads at the threshold: their kept steps that reach it are listed, or,
  // should a third one reach it too, the thread. (Both counters were set
  // before the barrier above.)
  if (mine >= least && mine != 0) {
    if (order_bits(fminf(third, W::kMost) + 0.f) >= least) {
      const int at = atomicAdd(&s_all, 1);
      if (at < kBeamMany) s_who[kBeamMany + at] = tid;
    } else {
      const bool two = order_bits(fminf(second, W::kMost) + 0.f) >= least;
      const int at = atomicAdd(&s_one, two ? 2 : 1);
      if (at < kBeamMany) s_who[at] = best_step << 9 | slot << 8 | tid;
      if (two && at + 1 < kBeamMany) s_who[at + 1] = second_step << 9 | (slot ^ 1) << 8 | tid;
    }
  }

  // This chunk's sum of exp(x - m). A logit far above all others counts as 1
  // exactly, so that its log probability is 0.
  if (m == -INFINITY || best == -INFINITY) {
    my_sum = 0.0;
  } else if (!(my_sum < 1e30)) {
    // rare (NaN or infinite logits): from memory again, cleaned
    my_sum = 0.0;
#pragma unroll 1
    for (int i = 0; i < vectors; ++i) {
      const uint4 r = load(i);
      const uint32_t word[4] = {W::clean(r.x), W::clean(r.y), W::clean(r.z), W::clean(r.w)};
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < W::N; ++e) my_sum += ex2((W::at(word[q], e) - m) * kLog2e);
    }
  } else {
    my_sum *= ex2((ref - m) * kLog2e);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) my_sum += __shfl_xor_sync(0xffffffffu, my_sum, o);
  if (lane == 0) s_sum[wid] = my_sum;
  __syncthreads();

  // the logits that reach the threshold, in any order: the lanes read a
  // thread's words
  auto index = [&](int i, int q, int e) {
    return base + (i * kBeamThreads + tid) * N + q * W::N + e;
  };
  const int ones = s_one, alls = s_all;
  const bool many = ones > kBeamMany || alls > kBeamMany || least <= order_bits(-INFINITY);
  // one logit: a candidate if it reaches the threshold (NaN does not)
  auto look = [&](float raw, int at) {
    const float f = fminf(raw, W::kMost) + 0.f;
    if (raw == raw && at < p.vocab && order_bits(f) >= least) {
      const int n = atomicAdd(&s_n, 1);
      if (n < kBeamCap) s_cand[n] = beam_key(f, at);
    }
  };
  if (!many) {
    constexpr int kWords = kBeamStep * 4;  // a step's
    for (int k = tid / kWords; k < ones; k += kBeamThreads / kWords) {
      const int who = s_who[k], thread = who & 255, u = tid % kWords / 4, q = tid % 4;
      const uint32_t word = reinterpret_cast<const uint32_t*>(
          keep)[(((who >> 8 & 1) * kBeamStep + u) * kBeamThreads + thread) * 4 + q];
      const int at =
          base + (((who >> 9) * kBeamStep + u) * kBeamThreads + thread) * N + q * W::N;
#pragma unroll
      for (int e = 0; e < W::N; ++e) look(W::at(word, e), at + e);
    }
    // (rare: from memory again)
    for (int k = wid; k < alls; k += kBeamWarps)
      for (int i = lane; i < vectors * N; i += 32) {
        const int at = base + (i / N * kBeamThreads + s_who[kBeamMany + k]) * N + i % N;
        if (at < p.vocab) look(static_cast<float>(__ldg(x + at)), at);
      }
  }
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < kBeamWarps; ++k) total += s_sum[k];
    p.part_off[part] = m * 1.4426950408889634;
    p.part_sum[part] = total;
  }
  uint64_t* out = p.part_key + part * K;
  int n = s_n;
  if (many || n > kBeamCap) {
    // many equal the threshold (or NaN counts as -inf, which nothing above
    // has seen): from memory again, first those above it
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
    const uint32_t equal = max(least, order_bits(-INFINITY));
#pragma unroll 1
    for (int i = 0; i < vectors; ++i) {
      const uint4 r = load(i);
      const uint32_t word[4] = {W::clean(r.x), W::clean(r.y), W::clean(r.z), W::clean(r.w)};
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < W::N; ++e) {
          const float f = W::at(word[q], e) + 0.f;
          if (order_bits(f) > equal && index(i, q, e) < p.vocab) {
            const int at = atomicAdd(&s_n, 1);
            if (at < kBeamCap) s_cand[at] = beam_key(f, index(i, q, e));
          }
        }
    }
    __syncthreads();
    n = s_n;
    // then the first equal ones: vector i of all threads comes before i + 1
#pragma unroll 1
    for (int i = 0; i < vectors && n < K; ++i) {  // n: the same for every thread
      const uint4 r = load(i);
      const uint32_t word[4] = {W::clean(r.x), W::clean(r.y), W::clean(r.z), W::clean(r.w)};
      uint32_t mask = 0;  // which of the vector's logits are equal
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < W::N; ++e)
          if (order_bits(W::at(word[q], e) + 0.f) == equal && index(i, q, e) < p.vocab)
            mask |= 1u << (q * W::N + e);
      int incl = __popc(mask);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (lane == 31) s_warp[wid] = incl;
      __syncthreads();
      int at = n + incl - __popc(mask), total = 0;
#pragma unroll
      for (int k = 0; k < kBeamWarps; ++k) {
        at += k < wid ? s_warp[k] : 0;
        total += s_warp[k];
      }
      const uint64_t value = static_cast<uint64_t>(equal) << 32;
      for (; mask != 0 && at < K; mask &= mask - 1, ++at)
        s_cand[at] = value | (0xffffffffu - static_cast<uint32_t>(index(i, 0, __ffs(mask) - 1)));
      n = min(n + total, K);
      __syncthreads();  // s_warp may be written again; s_cand is complete
    }
  }
  if (n <= kBeamCap) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const uint64_t key = s_cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_cand[j] > key;
      if (rank < K) out[rank] = key;
    }
    for (int i = n + tid; i < K; i += kBeamThreads) out[i] = 0;  // fewer logits than K
    return;
  }
  uint64_t last = ~0ULL;
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    uint64_t best_key = 0;
#pragma unroll 1
    for (int i = 0; i < vectors; ++i) {
      const uint4 r = load(i);
      const uint32_t word[4] = {W::clean(r.x), W::clean(r.y), W::clean(r.z), W::clean(r.w)};
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < W::N; ++e) {
          const uint64_t key = beam_key(W::at(word[q], e) + 0.f, index(i, q, e));
          if (index(i, q, e) < p.vocab && key < last && key > best_key) best_key = key;
        }
    }
    last = block_max<uint64_t>(best_key, s_key, lane, wid);
    if (tid == 0) out[k] = last;
  }
}

// One request: the rows' sums, then the K best of its chunks' candidates.
// Latency: a handful of dependent L2 reads and two barriers.
constexpr int kBeamHeld = 4;  // candidates a thread keeps between the passes

__global__ void __launch_bounds__(kBeamThreads) beam_join_kernel(const BeamParams p) {
  extern __shared__ uint8_t beam_smem[];
  double* s_base = reinterpret_cast<double*>(beam_smem);  // [beams]: score, -inf: no continuation
  double* s_lse = s_base + p.beams;                       // [beams]
  __shared__ alignas(16) uint32_t s_four[32];
  __shared__ JoinKey s_key[kBeamWarps];
  __shared__ JoinKey s_cand[kBeamCap];
  __shared__ int s_n;
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int b = blockIdx.x, K = p.k, C = p.chunks;
  const int lists = p.beams * C, total = lists * K;
  const uint64_t* keys = p.part_key + static_cast<int64_t>(b) * total;
  // candidate i of the request: entry i / lists of list i % lists; list l is
  // chunk l / beams of beam l % beams, so that every warp starts on all beams
  // (the best ones hold most of the winners) and on their lists' best entries
  const int e_step = kBeamThreads / lists, l_step = kBeamThreads - e_step * lists;
  const int e0 = tid / lists, l0 = tid - e0 * lists;
  const float inv = 1.f / p.beams;
  auto beam_of = [&](int l) {  // l % beams, l < 2^22
    return l - __float2int_rd((l + 0.5f) * inv) * p.beams;
  };
  auto read = [&](int e, int l) {
    const int c = __float2int_rd((l + 0.5f) * inv), w = l - c * p.beams;
    return __ldcg(keys + (static_cast<int64_t>(w) * C + c) * K + e);
  };
  // the first ones' keys are read while the sums are joined
  uint64_t held[kBeamHeld];
  {
    int e = e0, l = l0;
#pragma unroll
    for (int i = 0; i < kBeamHeld; ++i) {
      held[i] = tid + i * kBeamThreads < total ? read(e, l) : 0;
      e += e_step;
      l += l_step;
      if (l >= lists) l -= lists, ++e;
    }
  }
  if (tid == 0) s_n = 0;
  for (int w = wid; w < p.beams; w += kBeamWarps) {
    const int64_t at = (static_cast<int64_t>(b) * p.beams + w) * C;
    const float c = p.scores[b * p.score_stride + w];
    double m = -INFINITY, sum = 0.0;
    for (int c0 = 0; c0 < C; c0 += 32) {  // (one round up to 32 chunks)
      const bool in = c0 + lane < C;
      const double mc = in ? __ldcg(p.part_off + at + c0 + lane) : -INFINITY;
      const double sc = in ? __ldcg(p.part_sum + at + c0 + lane) : 0.0;
      double top = mc;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmax(top, m);
      if (top == -INFINITY) continue;
      // (a weight's fp32 exponential is as exact as the summands are)
      double add = mc == -INFINITY ? 0.0 : ex2(static_cast<float>(mc - top)) * sc;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
      sum = (m == -INFINITY ? 0.0 : sum * ex2(static_cast<float>(m - top))) + add;
      m = top;
    }
    if (lane == 0) {
      const bool dead = m == -INFINITY || !(c > -INFINITY);  // continues nothing
      // log2(sum): the exponent, and fp32's logarithm of the mantissa in [1, 2)
      int ex = 0;
      const float mant = 2.f * static_cast<float>(frexp(sum, &ex));
      const double lse2 = m + (ex - 1) + static_cast<double>(log2f(mant));
      s_lse[w] = dead ? 0.0 : static_cast<float>(lse2 * 0.6931471805599453);
      s_base[w] = dead ? -INFINITY : static_cast<double>(fminf(c, 3.402823466e38f));
    }
  }
  __syncthreads();
  auto candidate = [&](uint64_t key, int l) {
    if (key == 0) return JoinKey{0, 0};
    const int w = beam_of(l);
    const float x = order_value(static_cast<uint32_t>(key >> 32));
    const double s = x == -INFINITY ? -INFINITY : s_base[w] + (x - s_lse[w]);
    const uint32_t token = 0xffffffffu - static_cast<uint32_t>(key);
    return JoinKey{order_bits64(s), (static_cast<uint64_t>(255 - w) << 56) |
                                        ((key >> 32) << 24) | (0xffffffu - token)};
  };
  // f(candidate) for every candidate of this thread
  auto each = [&](auto f) {
    int e = e0, l = l0;
#pragma unroll
    for (int i = 0; i < kBeamHeld; ++i) {
      f(candidate(held[i], l));
      e += e_step;
      l += l_step;
      if (l >= lists) l -= lists, ++e;
    }
    for (int i = tid + kBeamHeld * kBeamThreads; i < total; i += kBeamThreads) {
      f(candidate(read(e, l), l));
      e += e_step;
      l += l_step;
      if (l >= lists) l -= lists, ++e;
    }
  };
  uint64_t best = 0;
  each([&](const JoinKey& c) { best = max(best, c.score); });
  // (the upper half of the score's bits is threshold enough)
  uint32_t top;
  const uint32_t least = block_threshold(static_cast<uint32_t>(best >> 32), K, s_four, lane, wid,
                                         &top);
  if (best != 0 && best >> 32 >= least)
    each([&](const JoinKey& c) {
      if (c.score != 0 && c.score >> 32 >= least) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kBeamCap) s_cand[at] = c;
      }
    });
  __syncthreads();
  auto put = [&](int k, const JoinKey& c) {
    const int64_t at = static_cast<int64_t>(b) * K + k;
    p.out_scores[at] = static_cast<float>(order_value64(c.score));
    p.out_parents[at] = b * p.beams + 255 - static_cast<int>(c.rest >> 56);
    p.out_tokens[at] = 0xffffff - static_cast<int>(c.rest & 0xffffff);
  };
  const int n = s_n;
  if (n <= kBeamCap) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const JoinKey c = s_cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_cand[j] > c;
      if (rank < K) put(rank, c);
    }
    return;
  }
  JoinKey last{~0ULL, ~0ULL};
  for (int k = 0; k < K; ++k) {
    JoinKey next{0, 0};
    each([&](const JoinKey& c) {
      if (last > c && c > next) next = c;
    });
    last = block_max<JoinKey>(next, s_key, lane, wid);
    if (tid == 0) put(k, last);
  }
}

}  // namespace pa
