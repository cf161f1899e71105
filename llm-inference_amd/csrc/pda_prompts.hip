// Attention of whole prompts packed one behind the other for MI355X (gfx950),
// C-ABI in pda.h (pda_packed_prompt_attention). No counterpart in the reference,
// which prefills one sequence a call from its paged cache (PrefillBatch.attend,
// python/instinct/batches.py:84-132).
//
// Token i of a prompt attends to tokens max(0, i - window + 1) .. i of the same
// prompt, whose keys and values lie beside the queries (slices of one projection's
// output, read where they are): flops 4 D per (query head, query, key), every
// operand read once.
//
// Bound by the matrix cores from a few hundred tokens on, as far as the exponentials
// beside them let it: 16384 tokens, 28/4 heads of 128, bf16, 1.79 to 1.86 ms by
// the card, 1.04 to 1.07 PFLOP/s (a large bf16 matrix product: 1.38), matrix cores 55%
// busy, VALU 46%, 5.7 VALU instructions a product. Short prompts pay for their ends: an item of one tile of keys
// takes as long as five tiles more (16 prompts of 128-2048: 236 us, 728 TFLOP/s), which
// is why workgroups stay and load the next item's first keys and queries beside the end
// of the one at hand (a workgroup an item: 285 us; heads of 256, window 1024, one
// workgroup a CU: 280 and 248).

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "pda.h"
#include "pda_internal.h"
#include "pda_rows.h"

namespace {

using namespace pda_rows;
using pda_internal::fail;
using pda_internal::ok;

constexpr int kThreads = 256;
constexpr int kTile = 128;  // queries of a workgroup
constexpr int kXcds = 8;
constexpr int kCus = 256;

struct PromptParams {
  const f16* q;
  const f16* k;
  const f16* v;
  f16* out;  // [tokens, hq, dim]
  const int32_t* starts;  // [batch + 1]
  int64_t q_token, k_token, v_token;  // elements between tokens,
  int64_t q_head, k_head, v_head;     //   between heads
  int32_t tokens;
  int32_t batch;
  int32_t tiles;  // query tiles there are at most
  int32_t hq;
  int32_t hkv;
  int32_t dim;
  int32_t window;
  Shape shape;
};

// Sequence b's tokens [a, z).
__device__ __forceinline__ void bounds(const PromptParams& p, int b, int& a, int& z) {
  a = max(0, min(p.starts[b], p.tokens));
  z = max(a, min(p.starts[b + 1], p.tokens));
}
__device__ __forceinline__ int tiles_of(const PromptParams& p, int b) {
  int a, z;
  bounds(p, b, a, z);
  return (z - a + kTile - 1) / kTile;
}

// What a workgroup works on: 128 queries of a head.
struct Item {
  int a, len;  // the prompt's tokens [a, a + len) (len 0: there is no item)
  int q0;      // its first query there
  int h, kvh;  // the query head, and its kv head
};

// The items in the order in which workgroups take them: tiles of 128 queries, each with
// its query heads. Sorted, those that see the most keys come first (tile i of any prompt
// before tile i - 1 of any), so that what is left for the end is short: with F(i) = sum of
// max(0, tiles - i) tiles at i or above, and the prompts by their tiles, tile x is at the
// i with F(i) > x >= F(i + 1), of the prompt that comes x - F(i + 1)-th. Else (as many
// workgroups as items, or more prompts or tiles than there is room for here) prompt after
// prompt, each from its last tile.
struct Order {
  static constexpr int kPrompts = 256;  // sorted at most,
  static constexpr int kLevels = 1024;  //   and tiles of each
  static constexpr int kList = 64;
  int32_t tiles[kPrompts], by_tiles[kPrompts];
  int32_t from[kLevels + 1];  // F, or the sum before each thread's prompts
  int32_t sum[kThreads / 64];
  int32_t all, sorted;
  Item list[kList];  // this workgroup's next items
};

// Sum over the workgroup of the values of the threads before this one, and of all.
__device__ __forceinline__ int before_me(Order& o, int mine, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 63) o.sum[w] = upto;
  __syncthreads();
  int before = upto - mine;
  all = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < w) before += o.sum[i];
    all += o.sum[i];
  }
  return before;
}

__device__ __forceinline__ void make_order(const PromptParams& p, Order& o) {
  const int tid = threadIdx.x;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of(p, b);
  if (per <= 1) o.tiles[tid] = mine;
  if (tid == 0) o.sorted = per <= 1 && p.tiles * (int64_t)p.hq > gridDim.x;
  int all;
  const int before = before_me(o, mine, all);
  if (tid == 0) o.all = all;
  if (o.sorted) {  // (written before the barrier in before_me)
    int most = 0, rank = 0;
    for (int b = 0; b < p.batch; ++b) {
      const int n = o.tiles[b];
      most = max(most, n);
      rank += n > mine || (n == mine && b < tid) ? 1 : 0;
    }
    if (tid < p.batch) o.by_tiles[rank] = tid;
    if (most > Order::kLevels) {
      __syncthreads();
      if (tid == 0) o.sorted = 0;
    } else {
      for (int i = tid; i <= most; i += kThreads) {
        int n = 0;
        for (int b = 0; b < p.batch; ++b) n += max(0, o.tiles[b] - i);
        o.from[i] = n;
      }
    }
  }
  __syncthreads();
  if (!o.sorted) o.from[tid] = before;
  __syncthreads();
}

// The workgroup's items from its i-th on, a lane of the first wave each.
__device__ __forceinline__ void fill_list(const PromptParams& p, Order& o, int i) {
  __syncthreads();
  if (threadIdx.x < Order::kList) {
    const int G = p.hq / p.hkv;
    const int all = o.all;
    Item found = {0, 0, 0, 0, 0};
    int64_t y = blockIdx.x + (int64_t)(i + threadIdx.x) * gridDim.x;
    if (y < (int64_t)all * p.hq) {
      // The G query heads of a kv head follow each other on one XCD (workgroups go
      // round robin over the XCDs): its L2 serves their keys and values.
      const int64_t runs = (int64_t)all * p.hkv;
      if (y < runs / kXcds * kXcds * G) {
        const int64_t j = y / kXcds;
        y = ((j / G) * kXcds + y % kXcds) * G + j % G;
      }
      const int64_t run = y / G;
      const int x = (int)(run / p.hkv);
      found.kvh = (int)(run % p.hkv);
      found.h = found.kvh * G + (int)(y % G);
      int seq, tile;
      if (o.sorted) {
        int lo = 0, hi = Order::kLevels;  // from[lo] > x; from[hi] <= x, were it there
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (mid <= o.tiles[o.by_tiles[0]] && o.from[mid] > x)
            lo = mid;
          else
            hi = mid;
        }
        tile = lo;
        seq = o.by_tiles[x - (lo < o.tiles[o.by_tiles[0]] ? o.from[lo + 1] : 0)];
      } else {
        int lo = 0, hi = kThreads;  // the last thread whose prompts begin at x or before
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (o.from[mid] <= x)
            lo = mid;
          else
            hi = mid;
        }
        const int per = (p.batch + kThreads - 1) / kThreads;
        int left = x - o.from[lo];
        seq = lo * per;
        for (int n = tiles_of(p, seq); left >= n; n = tiles_of(p, seq)) {
          left -= n;
          ++seq;
        }
        tile = tiles_of(p, seq) - 1 - left;
      }
      int z;
      bounds(p, seq, found.a, z);
      found.len = z - found.a;
      found.q0 = tile * kTile;
    }
    o.list[threadIdx.x] = found;
  }
  __syncthreads();
}

// A query tile's keys and values on their way through LDS, and their masks. EXACT: the
// head dim is D. (Tested in the loop, the steps fall apart around their copies.)
template <int D, bool BF, bool EXACT>
struct PromptTiles {
  static constexpr int kPlanes = D / 32;
  static constexpr int kHalves = kPlanes * kPlane;  // of a tile
  static constexpr int kCopies = 2 * kPlanes;
  static constexpr bool kSpread = true;  // (the copies are there long before they are needed)

  const PromptParams& p;
  f16* s_k;          // [2][kHalves]
  f16* s_v;
  int* s_left;       // [3] by item: whether values that are not finite were taken as zeros
  bool special;      // a softcap, or a scale that is no positive factor
  int lane, w, gk, kchunk, vchunk;
  uint32_t k_dst, v_dst;

  // The item's.
  const f16* kb;     // the prompt's first key and value of the kv head
  const f16* vb;
  int q0, last;      // first query and last key of the workgroup
  int wq0, wlast;    // first and last query of the wave
  int at;            // this lane's query
  int t1;            // the end of its tiles
  int odd;           // added to a tile's number for its place in LDS
  int number;        // of the item
  // The next one: its first K tile (this thread's row of it) is copied where the item's
  // own are all there, its queries (this lane's row) are loaded when the item's are done
  // with.
  const f16* next_k;
  const f16* next_q;
  const f16* src_k;  // this thread's rows that are copied now
  const f16* src_v;

  __device__ __forceinline__ void init() {
    const int tid = threadIdx.x;
    lane = tid & 63;
    w = uniform(tid >> 6);
    // Copies: thread tid moves key tid / 4 of a tile, one 16-byte chunk a plane.
    gk = tid >> 2;
    kchunk = 8 * ((lane & 3) ^ ((lane >> 4) & 3));
    vchunk = 8 * (lane & 3);
    k_dst = uniform(lds_address(s_k) + 1024 * w);
    v_dst = uniform(lds_address(s_v) + 1024 * w);
    special = p.shape.cap_out > 0.0f || !(p.shape.scale_log2 > 0.0f);
    if (tid < 3) s_left[tid] = 0;
    if constexpr (!EXACT) {  // what no copy writes
      for (int i = 8 * tid; i < 2 * kHalves; i += 8 * kThreads) {
        *reinterpret_cast<f16x8*>(s_k + i) = f16x8{};
        *reinterpret_cast<f16x8*>(s_v + i) = f16x8{};
      }
    }
    __syncthreads();
    number = -1;
  }
  __device__ __forceinline__ int last_of(const Item& x) const { return min(x.q0 + kTile, x.len) - 1; }
  __device__ __forceinline__ int begin_of(const Item& x) const {
    return p.window > 0 ? max(0, x.q0 - p.window + 1) / kKeys : 0;
  }
  // (Rows past the prompt's last see what that one sees, and are not stored.)
  __device__ __forceinline__ int query_of(const Item& x) const {
    return min(x.q0 + 32 * w + (lane & 31), x.len - 1);
  }
  __device__ __forceinline__ const f16* keys_of(const Item& x) const {
    return p.k + (int64_t)x.a * p.k_token + (int64_t)x.kvh * p.k_head;
  }
  __device__ __forceinline__ const f16* queries_of(const Item& x) const {
    return p.q + (int64_t)(x.a + query_of(x)) * p.q_token + (int64_t)x.h * p.q_head;
  }
  // Takes up an item, and the one after it.
  __device__ __forceinline__ void take(const Item& x, const Item& after) {
    kb = keys_of(x);
    vb = p.v + (int64_t)x.a * p.v_token + (int64_t)x.kvh * p.v_head;
    q0 = x.q0;
    last = last_of(x);
    wq0 = x.q0 + 32 * w;
    wlast = min(wq0 + 31, x.len - 1);
    at = query_of(x);
    // (The first K of an item lies where the last item's next one would.)
    odd = number < 0 ? 0 : (t1 + odd + begin_of(x)) & 1;
    t1 = last / kKeys + 1;
    ++number;
    next_q = after.len > 0 ? queries_of(after) : queries_of(x);
    next_k = (after.len > 0 ? keys_of(after) + (int64_t)min(begin_of(after) * kKeys + gk, last_of(after)) * p.k_token
                            : kb) + kchunk;
  }
  __device__ __forceinline__ int slot(int t) const { return (t + odd) & 1; }
  __device__ __forceinline__ const f16* keys(int t) const { return s_k + slot(t) * kHalves; }
  __device__ __forceinline__ const f16* values(int t) const { return s_v + slot(t) * kHalves; }

  // Where this thread's rows of V of tile t and of K of tile t + 1 (past the last one the
  // next item's first) are.
  __device__ __forceinline__ void aim(int t) {
    src_v = vb + (int64_t)min(t * kKeys + gk, last) * p.v_token + vchunk;
    aim_k(t + 1);
  }
  __device__ __forceinline__ void aim_k(int t) {
    const f16* own = kb + (int64_t)min(t * kKeys + gk, last) * p.k_token + kchunk;
    const uint64_t on = (uint64_t)(t < t1 ? -1 : 0);  // (a select: no branch in the loop)
    src_k = reinterpret_cast<const f16*>((reinterpret_cast<uint64_t>(own) & on) |
                                         (reinterpret_cast<uint64_t>(next_k) & ~on));
  }
  template <int i>
  __device__ __forceinline__ void copy_k(int t) const {
    if (!EXACT && 32 * i + kchunk >= p.dim) return;
    copy_plane_to_lds<i>(src_k, k_dst + slot(t) * (2 * kHalves));
  }
  template <int j>
  __device__ __forceinline__ void copy(int t) const {
    if constexpr (j >= kPlanes)
      copy_k<j - kPlanes>(t + 1);
    else if (EXACT || 32 * j + vchunk < p.dim)
      copy_plane_to_lds<j>(src_v, v_dst + slot(t) * (2 * kHalves));
  }
  __device__ __forceinline__ void first(int t) {
    if (number == 0) {
      aim_k(t);
      auto of_k = [&](auto i) { copy_k<i.value>(t); };
      each(of_k, std::make_integer_sequence<int, kPlanes>{});
    }
    aim(t);
    auto one = [&](auto j) { copy<j.value>(t); };
    each(one, std::make_integer_sequence<int, kCopies>{});
    if (number == 0) {
      if constexpr (EXACT)
        wait_vmem<kCopies>();  // the first K alone
      else
        wait_vmem<0>();  // (planes that no lane copies are not counted)
      __syncthreads();
    }
    // (The flag of the item after this one: every wave is past the item before.)
    if (threadIdx.x == 0) s_left[(number + 1) % 3] = 0;
  }
  __device__ __forceinline__ void ahead(Rows<D, BF>& r) const {
    r.load(next_q, p.dim, true);
  }

  // Tiles that a row of the workgroup does not see whole.
  __device__ __forceinline__ bool edge(int t) const {
    return t * kKeys + kKeys - 1 > q0 || (p.window > 0 && t * kKeys <= last - p.window);
  }
  // There, values that are not finite become zeros (a weight of 0 would make them NaN
  // in rows that do not see them).
  __device__ __forceinline__ void close(int t) {
    wait_vmem<0>();
    if (edge(t)) {
      f16* mine = s_v + slot(t) * kHalves + 32 * gk + 8 * (lane & 3);
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) {
        const f16x8 x = *reinterpret_cast<const f16x8*>(mine + kPlane * i);
        if (not_finite<BF>(x)) {
          s_left[number % 3] = 1;
          *reinterpret_cast<f16x8*>(mine + kPlane * i) = finite_only<BF>(x);
        }
      }
    }
    __syncthreads();
  }

  // What the lane's row sees of the 32 keys from k0 on; whether a row of the wave does
  // not see them all.
  __device__ __forceinline__ uint32_t visible(int k0) const {
    uint32_t see = below(at - k0 + 1);
    if (p.window > 0) see &= ~below(at - k0 - p.window + 1);
    return see;
  }
  __device__ __forceinline__ bool partly(int k0) const {
    return k0 + 31 > wq0 || (p.window > 0 && k0 <= wlast - p.window);
  }
  __device__ __forceinline__ bool rough(int t) const {
    return special || partly(t * kKeys) || partly(t * kKeys - 32);
  }
  __device__ __forceinline__ void shape(f32x16& x, int k0) const {
    if (special) Rows<D, BF>::shape(x, p.shape);
    if (partly(k0)) Rows<D, BF>::mask(x, visible(k0));
  }
  // After the last tile: the values that were taken as zeros, to the rows that see
  // them.
  __device__ __forceinline__ void add_left_out(Rows<D, BF>& r, int t0) const {
    if (uniform(s_left[number % 3]) == 0) return;  // (written before the last barrier)
    for (int t = t0; t < t1; ++t) {
      if (!edge(t)) continue;
      for (int k = t * kKeys; k <= min(t * kKeys + kKeys - 1, last); ++k)
        r.add_not_finite(k <= at && (p.window == 0 || k > at - p.window), p.dim, [&](int d) {
          return widen4<BF>(vb + (int64_t)k * p.v_token + d);
        });
    }
  }
};

// Workgroups of four waves that take item after item, as many as a CU holds: at D = 64
// three (4 prompts of 3000 tokens, 14/2 heads: 105 us with two, 100 with three).
template <int D>
constexpr int groups_a_cu() { return D == 64 ? 3 : D <= 128 ? 2 : 1; }

template <int D, bool BF, bool EXACT>
__global__ __launch_bounds__(kThreads, groups_a_cu<D>()) void packed_prompt_kernel(
    const PromptParams p) {
  using Tiles = PromptTiles<D, BF, EXACT>;
  __shared__ __align__(1024) f16 s_k[2 * Tiles::kHalves];
  __shared__ __align__(1024) f16 s_v[2 * Tiles::kHalves];
  __shared__ Order s_order;
  __shared__ int s_left[3];

  // Rows behind the last prompt: zeros.
  {
    const int real = max(0, min(p.starts[p.batch], p.tokens));
    const int64_t from = (int64_t)real * p.hq * p.dim / 8, to = (int64_t)p.tokens * p.hq * p.dim / 8;
    for (int64_t i = from + blockIdx.x * kThreads + threadIdx.x; i < to;
         i += (int64_t)gridDim.x * kThreads)
      reinterpret_cast<f16x8*>(p.out)[i] = f16x8{};
  }
  make_order(p, s_order);
  fill_list(p, s_order, 0);
  auto item = [&](int i) {
    const Item& x = s_order.list[i % Order::kList];
    return Item{uniform(x.a), uniform(x.len), uniform(x.q0), uniform(x.h), uniform(x.kvh)};
  };
  Item now = item(0);
  if (now.len == 0) return;
  Rows<D, BF> r;
  r.init(p.shape);
  Tiles x{p, s_k, s_v, s_left};
  x.init();
  r.load(x.queries_of(now), p.dim, true);
  for (int i = 0;; ++i) {
    r.settle_queries();
    if ((i + 1) % Order::kList == 0) fill_list(p, s_order, i + 1);
    const Item next = item(i + 1);
    x.take(now, next);
    // Tiles that this wave's rows see.
    const int t0 = x.begin_of(now);
    const int wa = p.window > 0 ? max(0, x.wq0 - p.window + 1) / kKeys : 0;
    const int wb = x.wq0 < now.len ? x.wlast / kKeys + 1 : 0;
    attend(r, x, t0, x.t1, wa, wb, x.wlast >= (wb - 1) * kKeys + 32);
    x.add_left_out(r, t0);
    const float inv = r.inverse();
    const int row = x.wq0 + (x.lane & 31);
    if (row < now.len) r.store(p.out + ((int64_t)(now.a + row) * p.hq + now.h) * p.dim, p.dim, inv);
    if (next.len == 0) break;
    r.clear();
    now = next;
  }
}

template <bool BF, bool EXACT>
const void* kernel_for(int width) {
  return width == 64    ? reinterpret_cast<const void*>(packed_prompt_kernel<64, BF, EXACT>)
         : width == 96  ? reinterpret_cast<const void*>(packed_prompt_kernel<96, BF, EXACT>)
         : width == 128 ? reinterpret_cast<const void*>(packed_prompt_kernel<128, BF, EXACT>)
                        : reinterpret_cast<const void*>(packed_prompt_kernel<256, BF, EXACT>);
}
template <bool BF>
const void* kernel_for(int width, bool exact) {
  return exact ? kernel_for<BF, true>(width) : kernel_for<BF, false>(width);
}

int packed_prompt(const void* queries, int64_t q_token, int64_t q_head, const void* keys,
                  int64_t k_token, int64_t k_head, const void* values, int64_t v_token,
                  int64_t v_head, const int32_t* starts, void* out, int32_t tokens, int32_t batch,
                  int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale,
                  int32_t window, float softcap, bool bf16_elems, void* stream) {
  if (tokens < 0 || batch < 0 || q_heads <= 0 || kv_heads <= 0 || window < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "tokens=%d batch=%d q_heads=%d kv_heads=%d window=%d",
                tokens, batch, q_heads, kv_heads, window);
  if (q_heads % kv_heads)
    return fail(PDA_ERR_HEAD_RATIO, "query heads must be a multiple of kv heads");
  const int width = width_for(head_dim);
  if (width == 0)
    return fail(PDA_ERR_HEAD_DIM, "head_dim %d: packed prompts serve multiples of 8 up to 256",
                head_dim);
  if (!(scale == scale) || isinf(scale) || !(softcap >= 0.0f) || isinf(softcap))
    return fail(PDA_ERR_INVALID_ARGUMENT, "scale must be finite and softcap >= 0");
  if (tokens == 0) return ok();
  if (!queries || !keys || !values || !starts || !out)
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  const int64_t strides[] = {q_token, q_head, k_token, k_head, v_token, v_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8)
      return fail(PDA_ERR_ALIGNMENT, "strides must be multiples of 8 elements, got %lld",
                  (long long)s);
  if (((uintptr_t)queries | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)out) & 15)
    return fail(PDA_ERR_ALIGNMENT, "query, K/V and output buffers must be 16-byte aligned");
  if ((uintptr_t)starts & 3)
    return fail(PDA_ERR_ALIGNMENT, "the starts must be 4-byte aligned");
  if (tokens > INT32_MAX - 1024)  // (positions past a prompt's last tile are formed)
    return fail(PDA_ERR_TOO_LONG, "%d tokens: below 2^31 - 1024 are taken", tokens);
  // As many query tiles as the prompts can have.
  const int64_t tiles = ((int64_t)tokens + (int64_t)(kTile - 1) * batch) / kTile;
  if (tiles * q_heads > INT32_MAX)
    return fail(PDA_ERR_TOO_LONG, "%lld query tiles of %d heads are more than 2^31",
                (long long)tiles, q_heads);
  PromptParams prm;
  prm.q = static_cast<const f16*>(queries);
  prm.k = static_cast<const f16*>(keys);
  prm.v = static_cast<const f16*>(values);
  prm.out = static_cast<f16*>(out);
  prm.starts = starts;
  prm.q_token = q_token;
  prm.k_token = k_token;
  prm.v_token = v_token;
  prm.q_head = q_head;
  prm.k_head = k_head;
  prm.v_head = v_head;
  prm.tokens = tokens;
  prm.batch = batch;
  prm.tiles = (int32_t)tiles;
  prm.hq = q_heads;
  prm.hkv = kv_heads;
  prm.dim = head_dim;
  prm.window = window;
  prm.shape = shape_of(scale, softcap);
  // As many workgroups as the GPU holds at once. (All items, and rows to clear, are
  // theirs: one at least.)
  const int a_cu = width == 64 ? groups_a_cu<64>() : width <= 128 ? groups_a_cu<128>() : groups_a_cu<256>();
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>(tiles * q_heads, kCus * a_cu));
  void* args[] = {&prm};
  const hipError_t err =
      hipLaunchKernel(bf16_elems ? kernel_for<true>(width, width == head_dim)
                                 : kernel_for<false>(width, width == head_dim),
                      dim3((unsigned)groups), dim3(kThreads), args, 0,
                      static_cast<hipStream_t>(stream));
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

}  // namespace

extern "C" {

int pda_packed_prompt_attention(const void* queries, int64_t q_token, int64_t q_head,
                                const void* keys, int64_t k_token, int64_t k_head,
                                const void* values, int64_t v_token, int64_t v_head,
                                const int32_t* starts, void* out, int32_t tokens, int32_t batch,
                                int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale,
                                int32_t window, float softcap, void* stream) {
  return packed_prompt(queries, q_token, q_head, keys, k_token, k_head, values, v_token, v_head,
                       starts, out, tokens, batch, q_heads, kv_heads, head_dim, scale, window,
                       softcap, false, stream);
}

int pda_packed_prompt_attention_bf16(const void* queries, int64_t q_token, int64_t q_head,
                                     const void* keys, int64_t k_token, int64_t k_head,
                                     const void* values, int64_t v_token, int64_t v_head,
                                     const int32_t* starts, void* out, int32_t tokens,
                                     int32_t batch, int32_t q_heads, int32_t kv_heads,
                                     int32_t head_dim, float scale, int32_t window,
                                     float softcap, void* stream) {
  return packed_prompt(queries, q_token, q_head, keys, k_token, k_head, values, v_token, v_head,
                       starts, out, tokens, batch, q_heads, kv_heads, head_dim, scale, window,
                       softcap, true, stream);
}

}  // extern "C"
