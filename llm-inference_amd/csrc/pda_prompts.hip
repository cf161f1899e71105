// Attention of whole prompts packed one behind the other for MI355X (gfx950),
// C-ABI in pda.h (pda_packed_prompt_attention). No counterpart in the reference,
// which prefills one sequence a call from its paged cache (PrefillBatch.attend,
// python/instinct/batches.py:84-132).
//
// Token i of a prompt attends to tokens max(0, i - window + 1) .. i of the same
// prompt, whose keys and values lie beside the queries (slices of one projection's
// output, read where they are): flops 4 D per (query head, query, key), every
// operand read once.

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
  int32_t tiles;  // query tiles of the grid
  int32_t hq;
  int32_t hkv;
  int32_t dim;
  int32_t window;
  Shape shape;
};

// Sequence b's tokens [a, z); b = batch: those behind the last sequence.
__device__ __forceinline__ void bounds(const PromptParams& p, int b, int& a, int& z) {
  a = max(0, min(p.starts[b], p.tokens));
  z = b < p.batch ? max(a, min(p.starts[b + 1], p.tokens)) : p.tokens;
}

__device__ __forceinline__ int sum64(int x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
  return x;
}

struct Place {
  int seq, tile, a, z;  // the sequence (-1: none), the tile of its tokens [a, z)
};

// The x-th query tile of all sequences, those that see the most keys first: tile i of
// any sequence before tile i - 1 of any. Every wave finds it by itself, a lane for a
// sequence: count(i) = sum of max(0, tiles - i) is how many lie at i or above.
__device__ __forceinline__ Place locate_few(const PromptParams& p, int x) {
  const int lane = threadIdx.x & 63;
  int a = 0, z = 0;
  if (lane <= p.batch) bounds(p, lane, a, z);
  const int mine = lane <= p.batch ? (z - a + kTile - 1) / kTile : 0;
  int lo = 0, hi = p.tiles, above = 0;  // count(lo) > x >= count(hi) = above
  const int all = sum64(mine);
  if (x >= all) return {-1, 0, 0, 0};
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    const int n = sum64(max(0, mine - mid));
    if (n > x)
      lo = mid;
    else
      hi = mid, above = n;
  }
  const uint64_t here = __ballot(mine > lo);
  const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(here >> 32),
                                             __builtin_amdgcn_mbcnt_lo((uint32_t)here, 0));
  const int seq = __builtin_ctzll(__ballot(mine > lo && rank == x - above));
  return {seq, lo, __shfl(a, seq), __shfl(z, seq)};
}

// For more sequences than lanes: sequence after sequence, each from its last tile.
__device__ __forceinline__ Place locate_many(const PromptParams& p, int x) {
  __shared__ int s_sum[kThreads / 64];
  __shared__ Place s_found;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int per = (p.batch + kThreads) / kThreads;  // of batch + 1
  const int b0 = tid * per, b1 = min(b0 + per, p.batch + 1);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    int a, z;
    bounds(p, b, a, z);
    mine += (z - a + kTile - 1) / kTile;
  }
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 63) s_sum[w] = upto;
  if (tid == 0) s_found.seq = -1;
  __syncthreads();
  int before = upto - mine;
  for (int i = 0; i < w; ++i) before += s_sum[i];
  if (x >= before && x < before + mine) {
    int left = x - before;
    for (int b = b0; b < b1; ++b) {
      int a, z;
      bounds(p, b, a, z);
      const int n = (z - a + kTile - 1) / kTile;
      if (left < n) {
        s_found = {b, n - 1 - left, a, z};
        break;
      }
      left -= n;
    }
  }
  __syncthreads();
  return s_found;
}

// A query tile's keys and values on their way through LDS, and their masks.
template <int D, bool BF>
struct PromptTiles {
  static constexpr int kPlanes = D / 32;
  static constexpr int kHalves = kPlanes * kPlane;  // of a tile
  static constexpr int kCopies = 2 * kPlanes;

  const PromptParams& p;
  f16* s_k;          // [2][kHalves]
  f16* s_v;
  int* s_left;       // whether values that are not finite were taken as zeros
  const f16* kb;     // the prompt's first key and value of the kv head
  const f16* vb;
  int q0, last;      // first query and last key of the workgroup
  int wq0, wlast;    // first and last query of the wave
  int at;            // this lane's query
  bool special;      // a softcap, or a scale that is no positive factor
  int lane, w, gk, kchunk, vchunk;
  uint32_t k_dst, v_dst;

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
    if (tid == 0) *s_left = 0;
    if (p.dim != D) {  // what no copy writes
      for (int i = 8 * tid; i < 2 * kHalves; i += 8 * kThreads) {
        *reinterpret_cast<f16x8*>(s_k + i) = f16x8{};
        *reinterpret_cast<f16x8*>(s_v + i) = f16x8{};
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ const f16* keys(int t) const { return s_k + (t & 1) * kHalves; }
  __device__ __forceinline__ const f16* values(int t) const { return s_v + (t & 1) * kHalves; }

  template <int i>
  __device__ __forceinline__ void copy_k(int t) const {
    if (D == p.dim || 32 * i + kchunk < p.dim)
      copy_plane_to_lds<i>(kb + (int64_t)min(t * kKeys + gk, last) * p.k_token + kchunk,
                           k_dst + (t & 1) * (2 * kHalves));
  }
  template <int j>
  __device__ __forceinline__ void copy(int t) const {
    if constexpr (j >= kPlanes)
      copy_k<j - kPlanes>(t + 1);
    else if (D == p.dim || 32 * j + vchunk < p.dim)
      copy_plane_to_lds<j>(vb + (int64_t)min(t * kKeys + gk, last) * p.v_token + vchunk,
                           v_dst + (t & 1) * (2 * kHalves));
  }
  __device__ __forceinline__ void first(int t) {
    auto of_k = [&](auto i) { copy_k<i.value>(t); };
    each(of_k, std::make_integer_sequence<int, kPlanes>{});
    auto one = [&](auto j) { copy<j.value>(t); };
    each(one, std::make_integer_sequence<int, kCopies>{});
    if (D == p.dim)
      wait_vmem<kCopies>();  // the first K alone
    else
      wait_vmem<0>();  // (planes that no lane copies are not counted)
    __syncthreads();
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
      f16* mine = s_v + (t & 1) * kHalves + 32 * gk + 8 * (lane & 3);
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) {
        const f16x8 x = *reinterpret_cast<const f16x8*>(mine + kPlane * i);
        if (not_finite<BF>(x)) {
          *s_left = 1;
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
  __device__ __forceinline__ void add_left_out(Rows<D, BF>& r, int t0, int t1) const {
    __syncthreads();
    if (uniform(*s_left) == 0) return;
    for (int t = t0; t < t1; ++t) {
      if (!edge(t)) continue;
      for (int k = t * kKeys; k <= min(t * kKeys + kKeys - 1, last); ++k)
        r.add_not_finite(k <= at && (p.window == 0 || k > at - p.window), p.dim, [&](int d) {
          return widen4<BF>(vb + (int64_t)k * p.v_token + d);
        });
    }
  }
};

template <int D, bool BF>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void packed_prompt_kernel(
    const PromptParams p) {
  using Tiles = PromptTiles<D, BF>;
  __shared__ __align__(1024) f16 s_k[2 * Tiles::kHalves];
  __shared__ __align__(1024) f16 s_v[2 * Tiles::kHalves];
  __shared__ int s_left;

  const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6);
  const int G = p.hq / p.hkv;
  // The G query heads of a kv head follow each other on one XCD (workgroups go
  // round robin over the XCDs): its L2 serves their keys and values.
  int item = blockIdx.x;
  const int runs = p.tiles * p.hkv;
  if (item < runs / kXcds * kXcds * G) {
    const int j = item / kXcds;
    item = ((j / G) * kXcds + item % kXcds) * G + j % G;
  }
  const int run = item / G;
  const int kvh = run % p.hkv, h = kvh * G + item % G;
  const Place place = p.batch < 64 ? locate_few(p, run / p.hkv) : locate_many(p, run / p.hkv);
  const int seq = uniform(place.seq);
  if (seq < 0) return;
  const int a = uniform(place.a), len = uniform(place.z) - a;
  const int q0 = uniform(place.tile) * kTile, wq0 = q0 + 32 * w, row = wq0 + (lane & 31);
  f16* out = p.out + ((int64_t)(a + row) * p.hq + h) * p.dim;
  Rows<D, BF> r;
  r.init(p.shape);
  if (seq == p.batch) {  // behind the last sequence: zeros
    if (row < len) r.store(out, p.dim, 0.0f);
    return;
  }
  // (Rows past the prompt's last see what that one sees, and are not stored.)
  const int at = min(row, len - 1);
  r.load(p.q + (int64_t)(a + at) * p.q_token + (int64_t)h * p.q_head, p.dim, true);

  const int last = min(q0 + kTile, len) - 1;
  const int t0 = p.window > 0 ? max(0, q0 - p.window + 1) / kKeys : 0, t1 = last / kKeys + 1;
  const int wlast = min(wq0 + 31, len - 1);
  Tiles x{p, s_k, s_v, &s_left, p.k + (int64_t)a * p.k_token + (int64_t)kvh * p.k_head,
          p.v + (int64_t)a * p.v_token + (int64_t)kvh * p.v_head, q0, last, wq0, wlast, at};
  x.init();
  // Tiles that this wave's rows see.
  const int wa = p.window > 0 ? max(0, wq0 - p.window + 1) / kKeys : 0;
  const int wb = wq0 < len ? wlast / kKeys + 1 : 0;
  attend(r, x, t0, t1, wa, wb, wlast >= (wb - 1) * kKeys + 32);
  x.add_left_out(r, t0, t1);
  const float inv = r.inverse();
  if (row < len) r.store(out, p.dim, inv);
}

template <bool BF>
const void* kernel_for(int width) {
  return width == 64    ? reinterpret_cast<const void*>(packed_prompt_kernel<64, BF>)
         : width == 96  ? reinterpret_cast<const void*>(packed_prompt_kernel<96, BF>)
         : width == 128 ? reinterpret_cast<const void*>(packed_prompt_kernel<128, BF>)
                        : reinterpret_cast<const void*>(packed_prompt_kernel<256, BF>);
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
  // As many query tiles as the prompts and the rows behind them can have.
  const int64_t tiles = ((int64_t)tokens + (int64_t)(kTile - 1) * (batch + 1)) / kTile;
  if (tiles * q_heads >= (int64_t)1 << 24)  // 2^32 threads a launch
    return fail(PDA_ERR_TOO_LONG, "%lld query tiles of %d heads exceed one launch",
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
  void* args[] = {&prm};
  const hipError_t err =
      hipLaunchKernel(bf16_elems ? kernel_for<true>(width) : kernel_for<false>(width),
                      dim3((unsigned)(tiles * q_heads)), dim3(kThreads), args, 0,
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
