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

// The sequence and the tile of the packed tiles' x-th; sequence -1: there is none.
__device__ __forceinline__ void locate(const PromptParams& p, int x, int& seq, int& tile) {
  __shared__ int s_sum[kThreads / 64];
  __shared__ int s_found[2];
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
  if (tid == 0) s_found[0] = -1;
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
        s_found[0] = b;
        s_found[1] = left;
        break;
      }
      left -= n;
    }
  }
  __syncthreads();
  seq = uniform(s_found[0]);
  tile = uniform(s_found[1]);
}

template <int D, bool BF>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void packed_prompt_kernel(
    const PromptParams p) {
  constexpr int kPlanes = D / 32;
  constexpr int kTileHalves = kPlanes * kPlane;
  __shared__ __align__(1024) f16 s_k[2][kTileHalves];
  __shared__ __align__(1024) f16 s_v[2][kTileHalves];
  __shared__ uint16_t s_bad[2][4];  // keys whose values are not finite, by wave

  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
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
  int seq, tile;
  locate(p, run / p.hkv, seq, tile);
  if (seq < 0) return;
  int a, z;
  bounds(p, seq, a, z);
  a = uniform(a);
  z = uniform(z);
  const int q0 = tile * kTile, len = z - a;
  const int wq0 = q0 + 32 * w, row = wq0 + (lane & 31);
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
  const int first = p.window > 0 ? max(0, q0 - p.window + 1) : 0;
  const int t0 = first / kKeys, t1 = last / kKeys + 1;
  // Tiles that this wave's rows see.
  const bool wave_live = wq0 < len;
  const int wlast = min(wq0 + 31, len - 1);
  const int wa = p.window > 0 ? max(t0, max(0, wq0 - p.window + 1) / kKeys) : t0;
  const int wb = wave_live ? wlast / kKeys + 1 : 0;

  // Copies: thread tid moves key tid / 4 of a tile, one 16-byte chunk a plane.
  const int gk = tid >> 2;
  const int kchunk = 8 * ((lane & 3) ^ ((lane >> 4) & 3)), vchunk = 8 * (lane & 3);
  const f16* kb = p.k + (int64_t)a * p.k_token + (int64_t)kvh * p.k_head;
  const f16* vb = p.v + (int64_t)a * p.v_token + (int64_t)kvh * p.v_head;
  const uint32_t k_dst = uniform(lds_address(&s_k[0][0]) + 1024 * w);
  const uint32_t v_dst = uniform(lds_address(&s_v[0][0]) + 1024 * w);
  if (p.dim != D) {  // what no copy writes
    f16* flat_k = &s_k[0][0];
    f16* flat_v = &s_v[0][0];
    for (int i = 8 * tid; i < 2 * kTileHalves; i += 8 * kThreads) {
      *reinterpret_cast<f16x8*>(flat_k + i) = f16x8{};
      *reinterpret_cast<f16x8*>(flat_v + i) = f16x8{};
    }
    __syncthreads();
  }
  auto copies = [&](int t) {
    const int key = min(t * kKeys + gk, last);
    const f16* src_k = kb + (int64_t)key * p.k_token + kchunk;
    const f16* src_v = vb + (int64_t)key * p.v_token + vchunk;
    const uint32_t off = ((t - t0) & 1) * (2 * kTileHalves);
#pragma unroll
    for (int i = 0; i < kPlanes; ++i) {
      if (D == p.dim || 32 * i + kchunk < p.dim)
        copy_to_lds(src_k + 32 * i, k_dst + off + 2 * kPlane * i);
      if (D == p.dim || 32 * i + vchunk < p.dim)
        copy_to_lds(src_v + 32 * i, v_dst + off + 2 * kPlane * i);
    }
  };
  // Tiles that a row of the workgroup does not see whole.
  auto edge = [&](int t) {
    return t * kKeys + kKeys - 1 > q0 || (p.window > 0 && t * kKeys <= last - p.window);
  };
  // There, values that are not finite become zeros (a weight of 0 would make them
  // NaN in rows that do not see them) and their keys are remembered.
  auto clean = [&](int t) {
    if (!edge(t)) return;
    const int buf = (t - t0) & 1;
    bool bad = false;
    f16* mine = &s_v[buf][32 * gk + 8 * (lane & 3)];
#pragma unroll
    for (int i = 0; i < kPlanes; ++i) {
      const f16x8 x = *reinterpret_cast<const f16x8*>(mine + kPlane * i);
      if (not_finite<BF>(x)) {
        bad = true;
        *reinterpret_cast<f16x8*>(mine + kPlane * i) = finite_only<BF>(x);
      }
    }
    const uint32_t keys = keys_of(__ballot(bad));
    if (lane == 0) s_bad[buf][w] = (uint16_t)keys;
  };

  const bool special = p.shape.cap_out > 0.0f || !(p.shape.scale_log2 > 0.0f);
  copies(t0);
  wait_vmem<0>();
  clean(t0);
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    if (t + 1 < t1) copies(t + 1);
    if (t >= wa && t < wb) {
      const int buf = (t - t0) & 1;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k0 = t * kKeys + 32 * j;
        f32x16 x;
        f16x8 weights[2];
        r.scores(x, s_k[buf] + 1024 * j);
        if (special) r.shape(x, p.shape);
        const bool masks = k0 + 31 > wq0 || (p.window > 0 && k0 <= wlast - p.window);
        uint32_t see = 0xFFFFFFFFu;
        if (masks) {
          see = below(at - k0 + 1);
          if (p.window > 0) see &= ~below(at - k0 - p.window + 1);
          r.mask(x, see);
        }
        r.weigh(x, weights);
        r.accumulate(weights, s_v[buf] + 1024 * j);
        if (edge(t)) {
          const uint32_t bad = uniform((int)(s_bad[buf][2 * j] | s_bad[buf][2 * j + 1] << 16));
          if (bad)
            r.add_not_finite(weights, bad, see, p.dim, [&](int k, int d) {
              return widen4<BF>(vb + (int64_t)min(k0 + k, last) * p.v_token + d);
            });
        }
      }
    }
    wait_vmem<0>();
    if (t + 1 < t1) clean(t + 1);
    __syncthreads();
  }
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
