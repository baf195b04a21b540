// Sliding-window attention with sinks: what a request's queries can see, and
// the decode plan over it.
//
// A query at position p of a request sees the keys j <= p with
//   j >= p - window_left   (the window, window_left + 1 keys with its own)
//   or j < num_sink_tokens (the first tokens, which stay visible).
// The reference serves full contexts only (src/models/llama.py:221, 239);
// this is FlashInfer's window_left plus sinks.
//
// Pages that hold no visible key are never read, and neither are their page
// ids: a serving loop gives them back to the pool and leaves anything (-1) in
// the table. So the request's keys become a stream of its visible pages,
// first the sinks' pages, then the window's: stream page v is table page v
// for v < sink_pages and v + shift otherwise, and inside the stream the keys
// [hole_lo, hole_hi) are hidden (the rest of the last sink page, and the keys
// of the window's first page before the window).
//
// Decode writes that stream out as a CSR table of its own in the workspace
// and runs the decode kernel over it unchanged but for the hole: the plan's
// equal runs, its flat page-id reads and its merges then see visible pages
// only. One layer's launch reads (window + sinks) keys per request whatever
// the context's length.
#pragma once

#include "decode.cuh"

namespace pa {

struct WindowSpan {
  int hole_lo, hole_hi;  // keys of the stream that are hidden (empty: both 0)
  int sink_pages;        // stream pages before the gap
  int shift;             // table pages left out after them
};

// The stream of the queries at positions >= first_query (their window starts
// at first_query - window). Exact for the first one; later queries hide more.
__host__ __device__ inline WindowSpan window_span(int64_t first_query, int window, int sinks,
                                                  int page_size) {
  int64_t start = first_query - window;
  if (start < 0) start = 0;
  WindowSpan w;
  const int64_t first = start / page_size;
  const int64_t sp = (static_cast<int64_t>(sinks) + page_size - 1) / page_size;
  w.shift = first > sp ? static_cast<int>(first - sp) : 0;
  w.sink_pages = static_cast<int>(sp < first ? sp : first);
  const int64_t hi = start - static_cast<int64_t>(w.shift) * page_size;
  const bool hole = hi > sinks;
  w.hole_lo = hole ? sinks : 0;
  w.hole_hi = hole ? static_cast<int>(hi) : 0;
  return w;
}

// Workspace of a window decode: the decode plan's, with the compacted table
// between its header and the rest. The header is at offset 0 as every plan's
// is, so a plan of any other kind over the same workspace replaces it, whatever
// else it leaves standing. (Behind the plan's partial states, megabytes away,
// the table cost each launch 0.4 us.)
struct WindowDecodeWsLayout {
  size_t indptr, window, indices, table_bytes, total;
  int64_t capacity;  // page ids the compacted table holds
};

// What the header says of a window plan beside the batch and the heads: a run
// for another window or another table's size is refused.
__host__ __device__ inline int4 window_plan_key(int window, int sinks, int64_t capacity,
                                                int64_t num_indices) {
  constexpr int64_t kMost = 0x7fffffff;
  return make_int4(window, sinks, static_cast<int>(capacity < kMost ? capacity : kMost),
                   static_cast<int>(num_indices < kMost ? num_indices : kMost));
}

// Pages of one request's stream at most: the sinks', and the window's
// window + 1 keys over one page more than they fill.
__host__ __device__ inline int64_t window_pages_max(int window, int sinks, int page_size) {
  return (static_cast<int64_t>(sinks) + page_size - 1) / page_size +
         static_cast<int64_t>(window) / page_size + 2;
}

__host__ __device__ inline WindowDecodeWsLayout window_decode_ws_layout(
    int batch, int64_t num_indices, int window, int sinks, int page_size, size_t decode_bytes) {
  WindowDecodeWsLayout L;
  const int64_t most = window_pages_max(window, sinks, page_size) * batch;
  L.capacity = most < num_indices ? most : num_indices;
  constexpr size_t kHeader = 256;
  static_assert(sizeof(DecodePlanHeader) <= kHeader, "the table starts at the next 256 bytes");
  size_t o = kHeader;
  L.indptr = o;
  o = align256(o + 4 * (static_cast<size_t>(batch) + 1));
  L.window = o;  // int4 {hole_lo, hole_hi, sink_pages, shift} per request
  o = align256(o + sizeof(int4) * static_cast<size_t>(batch));
  L.indices = o;
  o = align256(o + 4 * static_cast<size_t>(L.capacity));
  L.table_bytes = o - kHeader;
  L.total = decode_bytes + L.table_bytes;
  return L;
}

// What a table row says about a request: its stream, 0 pages when the row is
// malformed (the caller reports that).
struct WindowRow {
  int base, pages, visible;
  WindowSpan span;
  bool bad;
};

__device__ __forceinline__ WindowRow window_row(const int32_t* indptr, const int32_t* last_len,
                                                int b, int64_t num_indices, int page_size,
                                                int window, int sinks) {
  WindowRow r;
  const int s = __ldg(indptr + b), e = __ldg(indptr + b + 1);
  r.base = s;
  r.pages = e - s;
  r.visible = 0;
  r.span = WindowSpan{0, 0, 0, 0};
  r.bad = s < 0 || e < s || e > num_indices;
  if (r.bad || e == s) return r;
  const int lp = __ldg(last_len + b);
  r.bad = lp < 1 || lp > page_size;
  if (r.bad) return r;
  const int64_t len = static_cast<int64_t>(r.pages - 1) * page_size + lp;
  r.span = window_span(len - 1, window, sinks, page_size);
  r.visible = r.pages - r.span.shift;
  return r;
}

// The indptr that this CTA has just made: its first kWindowHeld entries in
// shared memory, the others read past the read-only path (which may hold
// older bytes).
constexpr int kWindowHeld = 2048;

struct FreshIndptr {
  const int32_t* held;
  const int32_t* all;
  __device__ __forceinline__ int operator[](int i) const {
    return i < kWindowHeld ? held[i] : __ldcg(all + i);
  }
};

constexpr int kWindowPlanThreads = 1024;
constexpr int kWindowRows = 64;

// CTA 0 scans the requests' visible pages into the compacted indptr, records
// each request's hole and cuts the stream into runs (decode_plan_block).
// The other CTAs copy the visible page ids, each for a range of requests
// whose offset it adds up by itself, so one launch does both.
__global__ void __launch_bounds__(kWindowPlanThreads)
    window_decode_plan_kernel(const int32_t* __restrict__ kv_indptr,
                              const int32_t* __restrict__ last_len,
                              const int32_t* __restrict__ kv_indices, int64_t num_indices,
                              int batch, int hkv, int hq, int head_dim, int page_size, int window,
                              int sinks, int num_groups, int hb, int min_per_group, int max_pieces,
                              uint8_t* __restrict__ ws, WindowDecodeWsLayout L) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int s_warp[32];
  __shared__ int s_carry;
  __shared__ int s_bad;
  __shared__ int32_t s_held[kWindowHeld];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  if (blockIdx.x == 0) {
    int32_t* out_indptr = reinterpret_cast<int32_t*>(ws + L.indptr);
    int4* out_window = reinterpret_cast<int4*>(ws + L.window);
    if (tid == 0) {
      s_carry = 0;
      s_bad = __ldg(kv_indptr) != 0;
      out_indptr[0] = s_held[0] = 0;
    }
    __syncthreads();
    for (int b0 = 0; b0 < batch; b0 += kWindowPlanThreads) {
      const int b = b0 + tid;
      WindowRow r{0, 0, 0, {0, 0, 0, 0}, false};
      if (b < batch) r = window_row(kv_indptr, last_len, b, num_indices, page_size, window, sinks);
      if (r.bad) s_bad = 1;
      int incl = r.visible;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (lane == 31) s_warp[wid] = incl;
      __syncthreads();
      if (wid == 0) {
        int w = s_warp[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, w, off);
          if (lane >= off) w += v;
        }
        s_warp[lane] = w;
      }
      __syncthreads();
      const int carry = s_carry;
      if (b < batch) {
        const int end = carry + (wid > 0 ? s_warp[wid - 1] : 0) + incl;
        out_indptr[b + 1] = end;
        if (b + 1 < kWindowHeld) s_held[b + 1] = end;
        out_window[b] = make_int4(r.span.hole_lo, r.span.hole_hi, r.span.sink_pages, r.span.shift);
      }
      __syncthreads();
      if (tid == 0) s_carry = carry + s_warp[31];
      __syncthreads();
    }
    decode_plan_block(FreshIndptr{s_held, out_indptr}, last_len, batch, hkv, hq, head_dim, page_size,
                      L.capacity, num_groups, hb, min_per_group, ws, kWindowDecodeMagic, s_bad != 0,
                      max_pieces, window_plan_key(window, sinks, L.capacity, num_indices),
                      L.table_bytes);
    return;
  }
  int32_t* out_indices = reinterpret_cast<int32_t*>(ws + L.indices);
  const int ctas = gridDim.x - 1, c = blockIdx.x - 1;
  const int b0 = static_cast<int>(static_cast<int64_t>(batch) * c / ctas);
  const int b1 = static_cast<int>(static_cast<int64_t>(batch) * (c + 1) / ctas);
  // (64 bits: the rows of a malformed table may claim the same entries again
  // and again)
  __shared__ int64_t s_sum[32];
  int64_t at = 0;
  for (int b = tid; b < b0; b += kWindowPlanThreads)
    at += window_row(kv_indptr, last_len, b, num_indices, page_size, window, sinks).visible;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) at += __shfl_xor_sync(0xffffffffu, at, off);
  if (lane == 0) s_sum[wid] = at;
  __syncthreads();
  at = 0;
#pragma unroll
  for (int w = 0; w < 32; ++w) at += s_sum[w];
  // the range's rows, kWindowRows at a time, read by a thread each
  __shared__ int4 s_row[kWindowRows];  // {first table entry, visible pages, sink pages, shift}
  for (int g = b0; g < b1; g += kWindowRows) {
    const int n = min(kWindowRows, b1 - g);
    if (tid < n) {
      const WindowRow r =
          window_row(kv_indptr, last_len, g + tid, num_indices, page_size, window, sinks);
      s_row[tid] = make_int4(r.base, r.visible, r.span.sink_pages, r.span.shift);
    }
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      const int4 r = s_row[i];
      for (int v = tid; v < r.y; v += kWindowPlanThreads)
        // a malformed table (which CTA 0 reports) may claim more than there is
        if (at + v < L.capacity)
          out_indices[at + v] = __ldg(kv_indices + r.x + v + (v < r.z ? 0 : r.w));
      at += r.y;
    }
    __syncthreads();  // s_row may be written again
  }
}

}  // namespace pa
