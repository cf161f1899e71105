// Page tables and slot maps of a step, built on the device for MI355X (gfx950),
// C-ABI in pda.h (pda_extend_tables).
//
// Reference step replaced: the host loops that give a step's tokens their rows
// (KVCache.rows, python/instinct/paged_kv.py:259-265; DecodeBatch.__init__,
// batches.py:148-179) and draw the pages that the requests' lengths ask for
// (PagePool.allocate, paged_kv.py:79-153). Here the host reserves pages ahead (the
// feed) and the step draws on them by itself, so that it can be replayed from a
// graph: with n_b new tokens behind l_b held rows, P rows a page and h_b pages held,
//   starts = prefix sums of n,  fresh_b = max(0, ceil((l_b + n_b) / P) - h_b),
// page h_b + j of sequence b is the feed's (drawn + fresh_0 + .. + fresh_{b-1} + j)-th,
// and token i of sequence b goes to row table[(l_b + i) / P] P + (l_b + i) % P.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "pda.h"
#include "pda_internal.h"

namespace {

using pda_internal::fail;
using pda_internal::ok;
using pda_internal::overlap;
using pda_internal::Span;

constexpr int kThreads = 256;
constexpr int kNodes = 64;             // of a tree at most
constexpr int kTreeTokens = kThreads - kNodes;
constexpr int kChainTokens = 4 * kThreads;
constexpr int kMaxBatch = 4096;        // prefix sums in LDS
constexpr int kMaxGroups = 1024;

struct ExtendParams {
  int32_t* tables;         // [batch, stride], in place
  const int32_t* lengths;  // [batch] rows held
  const int32_t* counts;   // [batch] new tokens
  const int32_t* pages;    // [batch] pages held
  const int32_t* feed;     // [feed_len]
  int32_t* drawn;          // [2]: pages drawn so far, workgroups arrived
  const int32_t* parents;  // [tokens], or null: every sequence's tokens are a chain
  int32_t* starts;         // [batch + 1]
  int32_t* out_lengths;    // [batch]
  int32_t* out_pages;      // [batch]
  int32_t* out_drawn;      // [2]
  int32_t* rows;           // [tokens]
  int32_t* positions;      // [tokens]
  uint64_t* masks;         // [tokens] with parents
  int64_t tokens;
  int32_t stride;
  int32_t feed_len;
  int32_t batch;
  int32_t page_size;
};

// Sum over the workgroup of the values of the threads before this one; `all`: of
// every thread's.
__device__ __forceinline__ int64_t before_me(int64_t mine, int64_t& all) {
  __shared__ int64_t s_sum[kThreads / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  __syncthreads();
  if (lane == 63) s_sum[w] = upto;
  __syncthreads();
  int64_t before = upto - mine;
  all = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < w) before += s_sum[i];
    all += s_sum[i];
  }
  return before;
}

// Last entry of an ascending list of n + 1 that is at most x (the list's first is).
__device__ __forceinline__ int find(const int32_t* list, int n, int64_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

struct Held {
  int32_t rows, have, need;
};
// Rows and pages a sequence holds and, with its n new tokens, needs.
__device__ __forceinline__ Held held_of(const ExtendParams& p, int b, int n) {
  Held x;
  x.rows = max(0, p.lengths[b]);
  x.have = min(max(0, p.pages[b]), p.stride);
  const int64_t end = (int64_t)x.rows + n;
  const int64_t need = (end + p.page_size - 1) / p.page_size;
  x.need = n > 0 ? (int)max((int64_t)x.have, min(need, (int64_t)p.stride)) : x.have;
  return x;
}

__device__ __forceinline__ int saturated(int64_t x) { return (int)min(x, (int64_t)INT32_MAX); }

// Every workgroup forms the prefix sums over the sequences (the arrays are a few
// KiB, and a second launch costs more), then takes its share of the tokens and of
// the fresh pages. What may be written in place (lengths, pages, drawn) is written
// by the last workgroup to have read it. Nothing else is ordered between them. What it
// takes is the launch and its chain of dependent reads: a tree of 16 nodes 4.6 us, 256
// sequences of 1 to 1024 new tokens each 10.6.
__global__ __launch_bounds__(kThreads) void extend_tables_kernel(const ExtendParams p) {
  __shared__ int32_t s_start[kMaxBatch + 1], s_fresh[kMaxBatch + 1];
  __shared__ uint64_t s_mask[kThreads];
  __shared__ int s_up[kThreads];
  __shared__ int s_last;
  const int tid = threadIdx.x;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  int64_t mine = 0, all;
  for (int b = b0; b < b1; ++b) mine += max(0, p.counts[b]);
  int64_t at = before_me(mine, all);
  for (int b = b0; b < b1; ++b) {
    s_start[b] = (int)min(at, p.tokens);
    at += max(0, p.counts[b]);
  }
  const int total = (int)min(all, p.tokens);
  if (tid == 0) s_start[p.batch] = total;
  __syncthreads();
  const int drawn = p.drawn[0];
  mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Held x = held_of(p, b, s_start[b + 1] - s_start[b]);
    s_fresh[b] = x.need - x.have;
    mine += s_fresh[b];
  }
  at = before_me(mine, all);
  for (int b = b0; b < b1; ++b) {
    const int n = s_fresh[b];
    s_fresh[b] = saturated(at);
    at += n;
  }
  const int fresh = saturated(all);
  if (tid == 0) s_fresh[p.batch] = fresh;
  __syncthreads();
  auto fed = [&](int64_t j) -> int {  // the feed's page of the call's j-th fresh one
    const int64_t i = (int64_t)drawn + j;
    return i >= 0 && i < p.feed_len ? p.feed[i] : -1;
  };

  const int groups = gridDim.x;
  for (int64_t j = (int64_t)blockIdx.x * kThreads + tid; j < fresh;
       j += (int64_t)groups * kThreads) {
    const int b = find(s_fresh, p.batch - 1, j);
    const int have = min(max(0, p.pages[b]), p.stride);
    p.tables[(int64_t)b * p.stride + have + (j - s_fresh[b])] = fed(j);
  }

  const bool tree = p.parents != nullptr;
  const int64_t step = tree ? kTreeTokens : kThreads;
  for (int64_t t0 = (int64_t)blockIdx.x * step; t0 < p.tokens; t0 += (int64_t)groups * step) {
    // With parents a workgroup also takes the 64 tokens before its own, among
    // which are the ancestors of its first ones.
    const int64_t t = tree ? t0 - kNodes + tid : t0 + tid;
    const bool real = t >= 0 && t < total;
    const int b = real ? find(s_start, p.batch - 1, t) : 0;
    const int i = real ? (int)(t - s_start[b]) : 0;
    uint64_t mask = 0;
    int depth = i;
    if (tree) {
      int up = -1;
      if (real && i < kNodes) {
        const int parent = p.parents[t];
        mask = 1ull << i;
        if (parent >= 0 && parent < i) up = tid - (i - parent);
      }
      // Every turn doubles the ancestors known. (Those of the 64 tokens in front
      // may lie before the workgroup's tokens; theirs are not written.)
      if (up < 0) up = -1;
#pragma unroll
      for (int turn = 0; turn < 6; ++turn) {
        s_mask[tid] = mask;
        s_up[tid] = up;
        __syncthreads();
        if (up >= 0) {
          mask |= s_mask[up];
          up = s_up[up];
        }
        __syncthreads();
      }
      depth = max(0, (int)__popcll(mask) - 1);
    }
    if (t < p.tokens && (!tree || tid >= kNodes)) {
      int row = -1, position = 0;
      if (real) {
        const Held x = held_of(p, b, s_start[b + 1] - s_start[b]);
        const int64_t pos = (int64_t)x.rows + i;
        const int64_t j = pos / p.page_size;
        int page = -1;
        if (j < x.have)
          page = p.tables[(int64_t)b * p.stride + j];
        else if (j < x.need)
          page = fed((int64_t)s_fresh[b] + (j - x.have));
        const int64_t r = (int64_t)page * p.page_size + pos % p.page_size;
        if (page >= 0 && r <= INT32_MAX) row = (int)r;
        position = saturated((int64_t)x.rows + depth);
      }
      p.rows[t] = row;
      p.positions[t] = position;
      if (tree) p.masks[t] = mask;
    }
  }

  if (blockIdx.x == 0)
    for (int b = tid; b <= p.batch; b += kThreads) p.starts[b] = s_start[b];
  __syncthreads();  // (every thread's reads have returned: their values were used)
  if (groups > 1) {
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(&p.drawn[1], 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
    __syncthreads();
    if (!s_last) return;
  }
  for (int b = tid; b < p.batch; b += kThreads) {
    const Held x = held_of(p, b, s_start[b + 1] - s_start[b]);
    p.out_lengths[b] = saturated((int64_t)x.rows + s_start[b + 1] - s_start[b]);
    p.out_pages[b] = x.need;
  }
  if (tid == 0) {
    p.out_drawn[0] = saturated((int64_t)drawn + fresh);
    p.out_drawn[1] = 0;
    p.drawn[1] = 0;
  }
}

}  // namespace

extern "C" {

int pda_extend_tables(int32_t* tables, int32_t table_stride, const int32_t* lengths,
                      const int32_t* counts, const int32_t* pages, const int32_t* feed,
                      int32_t feed_len, int32_t* drawn, const int32_t* parents, int32_t batch,
                      int32_t page_size, int32_t tokens, int32_t* starts, int32_t* out_lengths,
                      int32_t* out_pages, int32_t* out_drawn, int32_t* rows, int32_t* positions,
                      uint64_t* masks, void* stream) {
  if (batch < 0 || table_stride <= 0 || feed_len < 0 || page_size <= 0 || tokens < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "batch=%d table_stride=%d feed_len=%d page_size=%d tokens=%d", batch, table_stride,
                feed_len, page_size, tokens);
  if (batch > kMaxBatch)
    return fail(PDA_ERR_TOO_LONG, "a step of %d sequences: at most %d are taken", batch, kMaxBatch);
  const bool none = batch == 0;
  if (!starts || !drawn || !out_drawn || (tokens > 0 && (!rows || !positions)) ||
      (!none && (!tables || !lengths || !counts || !pages || !out_lengths || !out_pages)) ||
      (feed_len > 0 && !feed) || (parents && tokens > 0 && !masks))
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  const uintptr_t mis = (uintptr_t)tables | (uintptr_t)lengths | (uintptr_t)counts |
                        (uintptr_t)pages | (uintptr_t)feed | (uintptr_t)drawn |
                        (uintptr_t)parents | (uintptr_t)starts | (uintptr_t)out_lengths |
                        (uintptr_t)out_pages | (uintptr_t)out_drawn | (uintptr_t)rows |
                        (uintptr_t)positions;
  if ((mis & 3) || ((uintptr_t)masks & 7))
    return fail(PDA_ERR_ALIGNMENT, "int32 buffers must be 4-byte aligned, masks 8-byte aligned");
  // (Workgroups read the inputs, and the pages that the tables hold, while others write; what
  // may be in place is written by the last one, entry by entry.)
  const int64_t n = 4 * (int64_t)batch, t = 4 * (int64_t)tokens;
  const Span in[] = {{"lengths", lengths, n}, {"counts", counts, n},
                     {"pages", pages, n},     {"feed", feed, 4 * (int64_t)feed_len},
                     {"drawn", drawn, 8},     {"parents", parents, parents ? t : 0}};
  const struct {
    Span of;
    const void* in_place;
  } results[] = {{{"tables", tables, n * table_stride}, nullptr},
                 {{"starts", starts, n + 4}, nullptr},
                 {{"out_lengths", out_lengths, n}, lengths},
                 {{"out_pages", out_pages, n}, pages},
                 {{"out_drawn", out_drawn, 8}, drawn},
                 {{"rows", rows, t}, nullptr},
                 {{"positions", positions, t}, nullptr},
                 {{"masks", masks, parents ? 2 * t : 0}, nullptr}};
  for (const auto& r : results) {
    for (const Span& x : in)
      if (overlap(r.of, x) && !(r.of.at == x.at && x.at == r.in_place))
        return fail(PDA_ERR_INVALID_ARGUMENT, "%s overlaps %s", r.of.name, x.name);
    for (const auto& x : results)
      if (&x != &r && overlap(r.of, x.of))
        return fail(PDA_ERR_INVALID_ARGUMENT, "%s overlaps %s", r.of.name, x.of.name);
  }
  ExtendParams prm{tables,    lengths,     counts,    pages,     feed,   drawn,
                   parents,   starts,      out_lengths, out_pages, out_drawn, rows,
                   positions, masks,       tokens,    table_stride, feed_len, batch,
                   page_size};
  const int per = parents ? kTreeTokens : kChainTokens;
  const int groups =
      std::min(kMaxGroups, std::max(1, (int)(((int64_t)tokens + per - 1) / per)));
  void* args[] = {&prm};
  const hipError_t err =
      hipLaunchKernel(reinterpret_cast<const void*>(extend_tables_kernel), dim3(groups),
                      dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

}  // extern "C"
