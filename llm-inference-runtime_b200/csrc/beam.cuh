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
// Chunk pass: a CTA holds a chunk in registers (all its loads in flight at
// once), takes the chunk's maximum and sum from them, and finds a threshold
// that K of its elements reach: in each warp the K-th largest of the threads'
// maxima, the largest of those over the warps. Few elements pass it; they are
// ranked by counting. Keys are (value, lowest index first) in 64 bits, unique,
// so equal logits cost nothing extra; more than kBeamCap elements pass only
// for inputs laid out against the threads' order, and then K rounds of a
// block-wide maximum give the same result.
#pragma once

#include "pa_common.cuh"

namespace pa {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamMaxK = 32;   // the K-th of a warp's 32 maxima
constexpr int kBeamMaxBeams = 256;      // JoinKey's 8 bits
constexpr int kBeamMaxVocab = 1 << 24;  // and 24
constexpr int kBeamCap = 1024;  // elements ranked by counting

struct BeamParams {
  const void* logits;
  int64_t stride_b, stride_w;  // elements
  const float* scores;         // [batch, beams]
  int64_t score_stride;
  int32_t batch, beams, vocab, k, chunks;
  float* part_max;    // [rows, chunks]
  double* part_sum;   // [rows, chunks]: sum of exp(x - part_max)
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

// NaN counts as -inf, +inf as the largest finite value; -0 becomes +0.
__device__ __forceinline__ float clean(float x) {
  x = x != x ? -INFINITY : x;
  return fminf(x, 3.402823466e38f) + 0.f;
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
__device__ __forceinline__ uint64_t shfl_key(uint64_t k, int l) {
  return __shfl_sync(0xffffffffu, k, l);
}
__device__ __forceinline__ JoinKey shfl_key(const JoinKey& k, int l) {
  return JoinKey{__shfl_sync(0xffffffffu, k.score, l), __shfl_sync(0xffffffffu, k.rest, l)};
}

// The warp's 32 keys in descending order over the lanes (bitonic network).
template <typename K>
__device__ __forceinline__ K warp_sort_desc(K key, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const K other = shfl_xor_key(key, step);
      const bool desc = (lane & size) == 0;  // size 32: all descending
      const bool low = (lane & step) == 0;
      const bool take_max = low == desc;
      if (take_max ? other > key : key > other) key = other;
    }
  return key;
}

// Threshold that at least k of the block's elements reach, from each thread's
// best key (zero: none): see the header. s_key: one key per warp.
template <typename K>
__device__ __forceinline__ K block_threshold(K best, int k, K* s_key, int lane, int wid) {
  const K sorted = warp_sort_desc(best, lane);
  const K kth = shfl_key(sorted, k - 1);
  if (lane == 0) s_key[wid] = kth;
  __syncthreads();
  K t = s_key[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w)
    if (s_key[w] > t) t = s_key[w];
  return t;
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

// Eight 16-bit or four 32-bit logits of a thread, as they lie in memory.
template <typename T>
struct BeamVec {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float at(int i) const;
};
template <>
__device__ __forceinline__ float BeamVec<float>::at(int i) const {
  return __uint_as_float(reinterpret_cast<const uint32_t*>(&raw)[i]);
}
template <>
__device__ __forceinline__ float BeamVec<__nv_bfloat16>::at(int i) const {
  const uint32_t w = reinterpret_cast<const uint32_t*>(&raw)[i >> 1];
  return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}
template <>
__device__ __forceinline__ float BeamVec<__half>::at(int i) const {
  const uint32_t w = reinterpret_cast<const uint32_t*>(&raw)[i >> 1];
  return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w >> 16 : w)));
}

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

// One chunk of one row. Element e of vector i of thread t is logit
// chunk * CH + (i * 256 + t) * N + e whatever the row's alignment, so equal
// rows give equal sums.
template <typename T, int VPT>
__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(const BeamParams p) {
  using V = BeamVec<T>;
  constexpr int N = V::N;
  constexpr int CH = kBeamThreads * N * VPT;
  __shared__ uint64_t s_key[kBeamWarps];
  __shared__ double s_sum[kBeamWarps];
  __shared__ uint64_t s_cand[kBeamCap];
  __shared__ int s_n;
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  const int b = row / p.beams, w = row - b * p.beams;
  const T* x = static_cast<const T*>(p.logits) + b * p.stride_b + w * p.stride_w;
  const int base = chunk * CH, K = p.k;
  if (tid == 0) s_n = 0;
  // a beam without a score continues nothing: all its logits count as -inf
  const float c0 = __ldg(p.scores + b * p.score_stride + w);
  const bool dead = !(c0 > -INFINITY);

  V v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int at = base + (i * kBeamThreads + tid) * N;
    const int left = p.vocab - at;
    v[i].raw = make_uint4(0, 0, 0, 0);
    if (left > 0)
      v[i].raw = load16_any(reinterpret_cast<const uint8_t*>(x + at),
                            min(left, N) * static_cast<int>(sizeof(T)));
  }
  auto value = [&](int i, int e) { return dead ? -INFINITY : clean(v[i].at(e)); };
  // elements of vector i inside the row, and their place in it
  auto count = [&](int i) { return p.vocab - base - (i * kBeamThreads + tid) * N; };
  auto index = [&](int i, int e) { return base + (i * kBeamThreads + tid) * N + e; };

  // the thread's best element, the lowest index among equal ones
  float best = -INFINITY;
  int best_at = -1;
#pragma unroll
  for (int i = VPT - 1; i >= 0; --i) {
    const int n = count(i);
#pragma unroll
    for (int e = N - 1; e >= 0; --e) {
      const float f = value(i, e);
      if (e < n && f >= best) {
        best = f;
        best_at = index(i, e);
      }
    }
  }
  const uint64_t mine = best_at >= 0 ? beam_key(best, best_at) : 0;
  const uint64_t least = block_threshold<uint64_t>(mine, K, s_key, lane, wid);
  const uint64_t top = block_max<uint64_t>(mine, s_key, lane, wid);
  const float m = order_value(static_cast<uint32_t>(top >> 32));  // the chunk is not empty

  // this chunk's sum of exp(x - m)
  double sum = 0.0;
  {
    float part[4] = {0.f, 0.f, 0.f, 0.f};
    if (m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int n = count(i);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          // x - m first: exact near the maximum, where the sum's weight is
          const float t = ex2((value(i, e) - m) * 1.4426950408889634f);
          part[e & 3] += e < n ? t : 0.f;
        }
      }
    }
    sum = (static_cast<double>(part[0]) + part[1]) + (static_cast<double>(part[2]) + part[3]);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) s_sum[wid] = sum;

  // the elements that reach the threshold
  if (mine >= least && mine != 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int n = count(i);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint64_t key = beam_key(value(i, e), index(i, e));
        if (e < n && key >= least) {
          const int at = atomicAdd(&s_n, 1);
          if (at < kBeamCap) s_cand[at] = key;
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < kBeamWarps; ++k) total += s_sum[k];
    p.part_max[blockIdx.x] = m;
    p.part_sum[blockIdx.x] = total;
  }
  uint64_t* out = p.part_key + static_cast<int64_t>(blockIdx.x) * K;
  const int n = s_n;
  if (n <= kBeamCap) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const uint64_t key = s_cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_cand[j] > key;
      if (rank < K) out[rank] = key;
    }
    for (int i = n + tid; i < K; i += kBeamThreads) out[i] = 0;  // fewer elements than K
    return;
  }
  uint64_t last = ~0ULL;
  for (int k = 0; k < K; ++k) {
    uint64_t next = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int left = count(i);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint64_t key = beam_key(value(i, e), index(i, e));
        if (e < left && key < last && key > next) next = key;
      }
    }
    last = block_max<uint64_t>(next, s_key, lane, wid);
    if (tid == 0) out[k] = last;
  }
}

// One request: the rows' sums, then the K best of its chunks' candidates.
__global__ void __launch_bounds__(kBeamThreads) beam_join_kernel(const BeamParams p) {
  extern __shared__ uint8_t beam_smem[];
  float* s_lse = reinterpret_cast<float*>(beam_smem);  // [beams]
  double* s_base = reinterpret_cast<double*>(beam_smem + ((p.beams * 4 + 7) & ~7));  // [beams]
  __shared__ JoinKey s_key[kBeamWarps];
  __shared__ JoinKey s_cand[kBeamCap];
  __shared__ int s_n;
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int b = blockIdx.x, K = p.k, C = p.chunks;
  if (tid == 0) s_n = 0;
  for (int w = wid; w < p.beams; w += kBeamWarps) {
    const int64_t at = (static_cast<int64_t>(b) * p.beams + w) * C;
    float m = -INFINITY;
    for (int c = lane; c < C; c += 32) m = fmaxf(m, __ldcg(p.part_max + at + c));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    double sum = 0.0;
    for (int c = lane; c < C; c += 32) {
      const float mc = __ldcg(p.part_max + at + c);
      if (mc != -INFINITY)
        sum += exp(static_cast<double>(mc) - m) * __ldcg(p.part_sum + at + c);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      const float c = p.scores[b * p.score_stride + w];
      const bool dead = m == -INFINITY || !(c > -INFINITY);  // continues nothing
      s_lse[w] = dead ? 0.f : static_cast<float>(m + log(sum));
      s_base[w] = dead ? -INFINITY : static_cast<double>(fminf(c, 3.402823466e38f));
    }
  }
  __syncthreads();
  // candidate i of the request: entry i / lists of list i % lists (a list is
  // a row's chunk), so that a warp's threads start on different lists
  const int lists = p.beams * C, total = lists * K;
  const uint64_t* keys = p.part_key + static_cast<int64_t>(b) * total;
  auto candidate = [&](int i) {
    const int e = i / lists, l = i - e * lists;
    const uint64_t key = __ldcg(keys + static_cast<int64_t>(l) * K + e);
    if (key == 0) return JoinKey{0, 0};
    const int w = l / C;
    const float x = order_value(static_cast<uint32_t>(key >> 32));
    const double s = x == -INFINITY ? -INFINITY
                                    : s_base[w] + (static_cast<double>(x) - s_lse[w]);
    const uint32_t token = 0xffffffffu - static_cast<uint32_t>(key);
    return JoinKey{order_bits64(s), (static_cast<uint64_t>(255 - w) << 56) |
                                        ((key >> 32) << 24) | (0xffffffu - token)};
  };
  JoinKey best{0, 0};
  for (int i = tid; i < total; i += kBeamThreads) {
    const JoinKey c = candidate(i);
    if (c > best) best = c;
  }
  const JoinKey least = block_threshold<JoinKey>(best, K, s_key, lane, wid);
  if (!(least > best) && best.score != 0) {
    for (int i = tid; i < total; i += kBeamThreads) {
      const JoinKey c = candidate(i);
      if (c.score != 0 && !(least > c)) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kBeamCap) s_cand[at] = c;
      }
    }
  }
  __syncthreads();
  auto put = [&](int k, const JoinKey& c) {
    p.out_scores[b * K + k] = static_cast<float>(order_value64(c.score));
    p.out_parents[b * K + k] = b * p.beams + 255 - static_cast<int>(c.rest >> 56);
    p.out_tokens[b * K + k] = 0xffffff - static_cast<int>(c.rest & 0xffffff);
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
    for (int i = tid; i < total; i += kBeamThreads) {
      const JoinKey c = candidate(i);
      if (last > c && c > next) next = c;
    }
    last = block_max<JoinKey>(next, s_key, lane, wid);
    if (tid == 0) put(k, last);
  }
}

}  // namespace pa
