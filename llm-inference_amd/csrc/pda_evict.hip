// Eviction from the paged K/V cache by accumulated attention weight for MI355X
// (gfx950), C-ABI in pda.h (pda_attention_weights, pda_evict_select,
// pda_evict_move). No reference counterpart: the reference bounds a cache by
// sliding windows alone.
//
// After a step's attention every key of a sequence is credited with the
// weights it was given, w[t] += sum over the query heads of a kv head of
// softmax(score)[t]; when a sequence passes its bound the keys with the least
// credit go and the rows of the others are packed, per kv head (a page tile's
// rows of different heads need not hold the same positions). Credits are kept
// per sequence and logical position, so sequences that share a prefix's pages
// do not share them.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "pda.h"
#include "pda_internal.h"

namespace {

using pda_internal::fail;
using pda_internal::ok;

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

// Until the wave's loads have returned: before a barrier past which others
// overwrite what was loaded.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---------------------------------------------------------------------------
// Weights.

constexpr int kWaves = 4;        // waves of a score workgroup
constexpr int kSlots = 16;       // query heads per workgroup
constexpr int kAddKeys = 1024;   // keys an adding workgroup takes
constexpr int kMaxChunksX = 4096;
constexpr int kScoreGroups = 1024;  // score workgroups to fill an MI355X

// 32-dim planes of a head that the score kernels hold, and the blocks of 16 keys
// a wave takes at once: 64 registers of K.
constexpr int planes_for(int dim) {
  return dim <= 64 ? 2 : dim <= 96 ? 3 : dim <= 128 ? 4 : dim <= 256 ? 8 : 16;
}
constexpr int blocks_for(int planes) { return planes <= 4 ? 4 : 16 / planes; }
constexpr int chunk_for(int planes) { return 16 * kWaves * blocks_for(planes); }

struct WeightParams {
  const f16* q;        // [batch, hq, D]
  const void* k;       // arena: 16-bit, or int8 with scales
  const f16* kscale;
  const int32_t* tables;
  const int32_t* lengths;
  const float* weights;  // [batch, hkv, capacity]
  float* out;
  float* scores;       // [batch, hq, pitch] times log2 e
  float2* stats;       // [batch, hq, chunks] (max, sum) of each chunk
  int64_t arena_pages;
  int64_t page_elems, scale_page;  // elements between pages,
  int32_t head_elems, scale_head;  //   kv heads of a page,
  int32_t row_elems, scale_row;    //   rows of a page and head
  int32_t table_stride;
  int32_t page_size;
  int32_t hq;
  int32_t hkv;
  int32_t head_dim;
  int32_t capacity;
  int32_t pitch;       // capacity, up to a multiple of 4
  int32_t chunk;       // keys per chunk
  int32_t chunks;      // ceil(capacity / chunk)
  int32_t window;
  int32_t fresh;
  float scale_log2;
  float cap_in;        // 2 log2(e) scale / softcap
  float cap_out;       // softcap log2(e); 0: no softcap
};

__device__ __forceinline__ int keys_of(const WeightParams& p, int b) {
  const int64_t cap = min((int64_t)p.table_stride * p.page_size, (int64_t)p.capacity);
  return (int)max((int64_t)0, min((int64_t)p.lengths[b], cap));
}

// 8 elements of a row from dim d on, as they are stored. VEC: head dims that are
// multiples of 8; past the head dim the row's last elements again (the queries
// are zeros there). Else element by element, zeros past the head dim.
template <class E, class V, bool VEC>
__device__ __forceinline__ V load8(const void* base, int64_t at, int d, int dim) {
  const E* src = static_cast<const E*>(base) + at;
  if constexpr (VEC) return *reinterpret_cast<const V*>(src + min(d, dim - 8));
  V x = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (d + i >= dim) break;
    if constexpr (sizeof(E) == 1)
      x[i / 4] |= (uint32_t)(uint8_t)src[d + i] << (8 * (i % 4));
    else
      x[i] = src[d + i];
  }
  return x;
}

// Them as operands: integers of 8 bits are exact in either type. (They are held
// as two dwords: a vector of bytes would take a register each.)
template <bool BF>
__device__ __forceinline__ f16x8 operand(const f16x8& x) { return x; }
template <bool BF>
__device__ __forceinline__ f16x8 operand(const u32x2& y) {
  f16x8 x;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = (float)(int)__builtin_amdgcn_sbfe((int)y[i / 4], 8 * (i % 4), 8);
    if constexpr (BF)
      x[i] = __builtin_bit_cast(f16, (bf16)f);
    else
      x[i] = (f16)f;
  }
  return x;
}

template <bool BF>
__device__ __forceinline__ f32x4 mfma(const f16x8& a, const f16x8& b, const f32x4& c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// (largest, sum relative to it) of two sets of scores together.
__device__ __forceinline__ float2 join(const float2& a, const float2& b) {
  const float m = fmaxf(a.x, b.x), mu = m == -INFINITY ? 0.0f : m;
  return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - mu) +
                            b.y * __builtin_amdgcn_exp2f(b.x - mu));
}

// Scores (times log2 e) of a sequence's keys against up to 16 heads of one kv
// head, with each head's largest and sum of exp2(score - largest) per chunk of
// keys. K is read once, straight into the matrix cores' operands (lane: key
// lane % 16, 8 dims), 64 bytes of a row per instruction; a lane ends with 4
// consecutive keys of one head per block. The scores are stored as they are, so
// the waves of a chunk meet only for its statistics. A workgroup goes over its
// chunks with the next one's rows, and the page numbers of the one after that,
// under way. Reads K and writes 4 bytes a head and key: the K bytes bound it
// (at the shape below 316 MB in 75 us, 4.2 TB/s).
template <int NC, bool Q8, bool BF, bool VEC>
__global__ __launch_bounds__(64 * kWaves, NC == 16 && !Q8 ? 1 : 2) void attention_scores_kernel(const WeightParams p) {
  typedef std::conditional_t<Q8, signed char, f16> Elem;
  typedef std::conditional_t<Q8, u32x2, f16x8> Elem8;
  constexpr int kBlocks = blocks_for(NC);
  constexpr int kChunk = chunk_for(NC);
  __shared__ float2 s_stats[2][kWaves][kSlots];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int n16 = lane & 15, g4 = lane >> 4;
  const int group = p.hq / p.hkv, tiles = (group + kSlots - 1) / kSlots;
  const int kvh = blockIdx.y / tiles, first = (blockIdx.y % tiles) * kSlots;
  const int b = blockIdx.z;
  const int slot = first + n16;
  const bool live = slot < group;
  const int h = kvh * group + slot;
  const int keys = keys_of(p, b);
  const int lo = p.window > 0 ? max(0, keys - p.window) : 0;
  const uint32_t pages = (uint32_t)min(p.arena_pages, (int64_t)INT32_MAX);
  const int32_t* table = p.tables + (int64_t)b * p.table_stride;
  const int stride = gridDim.x;
  const int c_end = (keys + kChunk - 1) / kChunk;
  const int c_first = lo / kChunk + blockIdx.x;
  if (c_first >= c_end) return;

  f16x8 qf[NC];
  const int64_t qat = ((int64_t)b * p.hq + (live ? h : 0)) * p.head_dim;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = 32 * c + 8 * g4;
    qf[c] = load8<f16, f16x8, VEC>(p.q, qat, d, p.head_dim);
    if (!live || d >= p.head_dim) qf[c] = f16x8{};
  }
  // The keys of a chunk that this lane looks up: 16 i + n16 of the wave's.
  struct Rows {
    uint32_t page[kBlocks];
  };
  struct Keys {
    Elem8 k[kBlocks][NC];
    f16 scale[kBlocks];
    uint32_t seen;  // bit i: this lane's key of block i has a row
  };
  auto key_at = [&](int chunk, int i) {
    return chunk * (int64_t)kChunk + w * (16 * kBlocks) + 16 * i + n16;
  };
  auto look_up = [&](int chunk, Rows& r) {
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
      r.page[i] = (uint32_t)table[(uint32_t)min(key_at(chunk, i), (int64_t)keys - 1) /
                                  (uint32_t)p.page_size];
  };
  auto fetch = [&](int chunk, const Rows& r, Keys& x) {
    x.seen = 0;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int64_t key = key_at(chunk, i);
      const bool have = key >= lo && key < keys && r.page[i] < pages;
      x.seen |= have ? 1u << i : 0u;
      const uint32_t row = (uint32_t)min(key, (int64_t)keys - 1) % (uint32_t)p.page_size;
      const uint32_t page = have ? r.page[i] : 0u;
      const int64_t at =
          page * p.page_elems + (int64_t)kvh * p.head_elems + (int64_t)row * p.row_elems;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        x.k[i][c] = load8<Elem, Elem8, VEC>(p.k, at, 32 * c + 8 * g4, p.head_dim);
      x.scale[i] = (f16)1.0f;
      if constexpr (Q8)
        x.scale[i] = p.kscale[page * p.scale_page + (int64_t)kvh * p.scale_head +
                                     (int64_t)row * p.scale_row];
    }
  };
  float* dst = p.scores + ((int64_t)b * p.hq + h) * p.pitch;
  auto weigh = [&](int chunk, const Keys& x, int buf) {
    f32x4 s[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) s[i] = f32x4{};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) s[i] = mfma<BF>(operand<BF>(x.k[i][c]), qf[c], s[i]);
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[i][v] *= __shfl((float)x.scale[i], 4 * g4 + v);
    }
    if (p.cap_out > 0.0f) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float e = __builtin_amdgcn_exp2f(s[i][v] * p.cap_in);
          s[i][v] = (1.0f - 2.0f / (e + 1.0f)) * p.cap_out;
        }
    } else {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[i][v] *= p.scale_log2;
    }
    // Key 4 g4 + v of a block was looked up by lane 4 g4 + v.
    float2 all = make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const uint32_t have = (uint32_t)__ballot(x.seen >> i & 1) >> (4 * g4);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        if (!(have >> v & 1)) s[i][v] = -INFINITY;
        all.x = fmaxf(all.x, s[i][v]);
      }
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int64_t key = key_at(chunk, i) - n16 + 4 * g4;
        if (key < keys) *reinterpret_cast<f32x4*>(dst + key) = s[i];
      }
    }
    const float mu = all.x == -INFINITY ? 0.0f : all.x;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) all.y += __builtin_amdgcn_exp2f(s[i][v] - mu);
    // The lanes', then the waves' statistics of a head. (Two buffers: a chunk's are
    // read before the next one's barrier.)
    all = join(all, make_float2(__shfl_xor(all.x, 16), __shfl_xor(all.y, 16)));
    all = join(all, make_float2(__shfl_xor(all.x, 32), __shfl_xor(all.y, 32)));
    if (g4 == 0) s_stats[buf][w][n16] = all;
    __syncthreads();
    if (live && w == 0 && g4 == 0) {
#pragma unroll
      for (int i = 1; i < kWaves; ++i) all = join(all, s_stats[buf][i][n16]);
      p.stats[((int64_t)b * p.hq + h) * p.chunks + chunk] = all;
    }
  };
  Rows rows;
  Keys even, odd;
  look_up(c_first, rows);
  fetch(c_first, rows, even);
  if (c_first + stride < c_end) look_up(c_first + stride, rows);
  for (int c = c_first;; c += 2 * stride) {
    Rows next;
    if (c + 2 * stride < c_end) look_up(c + 2 * stride, next);
    if (c + stride < c_end) fetch(c + stride, rows, odd);
    weigh(c, even, 0);
    if (c + stride >= c_end) break;
    if (c + 3 * (int64_t)stride < c_end) look_up(c + 3 * stride, rows);
    if (c + 2 * stride < c_end) fetch(c + 2 * stride, next, even);
    weigh(c + stride, odd, 1);
    if (c + 2 * stride >= c_end) break;
  }
}

// out[t] = weights[t] (0 for the `fresh` newest) + the sum over the kv head's
// query heads, in their order, of exp2(score - the head's largest) / its sum, the
// two joined from the chunks' once a workgroup, while the scores themselves
// are already under way. Reads 4 bytes a head and key, from the caches that the
// launch before left them in.
__global__ __launch_bounds__(256) void attention_weights_kernel(const WeightParams p) {
  constexpr int kHeads = 8;  // heads at once: two a wave for the statistics
  constexpr int kEach = kAddKeys / 256;
  __shared__ float2 s_stats[kHeads];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int group = p.hq / p.hkv, kvh = blockIdx.y, b = blockIdx.z;
  const int keys = keys_of(p, b);
  const int lo = p.window > 0 ? max(0, keys - p.window) : 0;
  const int c_lo = lo / p.chunk, c_hi = (keys + p.chunk - 1) / p.chunk;
  const int64_t base = ((int64_t)b * p.hkv + kvh) * p.capacity;
  for (int64_t k0 = (int64_t)blockIdx.x * kAddKeys; k0 < keys; k0 += (int64_t)gridDim.x * kAddKeys) {
    float acc[kEach] = {}, old[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t t = k0 + 256 * i + tid;
      old[i] = t < (int64_t)keys - p.fresh ? p.weights[base + t] : 0.0f;
    }
    for (int h0 = 0; h0 < group; h0 += kHeads) {
      const int heads = min(kHeads, group - h0);
      const int64_t row = (int64_t)b * p.hq + kvh * group + h0;
      float x[kHeads][kEach];
#pragma unroll
      for (int j = 0; j < kHeads; ++j)
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int64_t t = k0 + 256 * i + tid;
          x[j][i] = -INFINITY;
          if (j < heads && t >= lo && t < keys) x[j][i] = p.scores[(row + j) * p.pitch + t];
        }
      __syncthreads();
      for (int i = w; i < heads; i += 4) {
        const float2* st = p.stats + (row + i) * p.chunks;
        float2 all = make_float2(-INFINITY, 0.0f);
        for (int c = c_lo + lane; c < c_hi; c += 64) all = join(all, st[c]);
#pragma unroll
        for (int d = 32; d; d >>= 1)
          all = join(all, make_float2(__shfl_xor(all.x, d), __shfl_xor(all.y, d)));
        // (A head that sees no key gives nothing.)
        if (lane == 0)
          s_stats[i] = make_float2(all.x == -INFINITY ? 0.0f : all.x,
                                   all.y == 0.0f ? 0.0f : 1.0f / all.y);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kHeads; ++j) {
        if (j >= heads) break;
        const float2 st = s_stats[j];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          // (A hidden key gets nothing, also beside a visible one that is NaN.)
          acc[i] = x[j][i] == -INFINITY
                       ? acc[i]
                       : fmaf(__builtin_amdgcn_exp2f(x[j][i] - st.x), st.y, acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t t = k0 + 256 * i + tid;
      if (t < keys) p.out[base + t] = old[i] + acc[i];
    }
  }
}

template <bool Q8, bool BF>
const void* scores_kernel(int dim) {
  const int nc = planes_for(dim);
  if (dim % 8 == 0) {
    switch (nc) {
      case 2: return (const void*)attention_scores_kernel<2, Q8, BF, true>;
      case 3: return (const void*)attention_scores_kernel<3, Q8, BF, true>;
      case 4: return (const void*)attention_scores_kernel<4, Q8, BF, true>;
      case 8: return (const void*)attention_scores_kernel<8, Q8, BF, true>;
      default: return (const void*)attention_scores_kernel<16, Q8, BF, true>;
    }
  }
  return nc <= 4 ? (const void*)attention_scores_kernel<4, Q8, BF, false>
                 : (const void*)attention_scores_kernel<16, Q8, BF, false>;
}

// Planes of the kernel that scores_kernel picks.
int planes_run(int dim) {
  const int nc = planes_for(dim);
  return dim % 8 == 0 ? nc : nc <= 4 ? 4 : 16;
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// (The chunks of the widest heads, the smallest, whatever the head dim.)
size_t stats_bytes(int batch, int q_heads, int capacity) {
  const int chunk = chunk_for(16);
  return up256((size_t)batch * q_heads * (((size_t)capacity + chunk - 1) / chunk) * 8);
}

size_t weights_workspace(int batch, int q_heads, int capacity) {
  return stats_bytes(batch, q_heads, capacity) +
         up256((size_t)batch * q_heads * (((size_t)capacity + 3) & ~(size_t)3) * 4);
}

int attention_weights(const void* queries, const void* keys, const void* key_scales, bool q8,
                      const int32_t* tables, const int32_t* lengths, const float* weights,
                      float* out, int32_t batch, int32_t q_heads, int32_t kv_heads,
                      int32_t head_dim, int32_t page_size, int32_t table_stride,
                      int64_t arena_rows, int32_t layout, int32_t capacity, int32_t longest,
                      float scale, int32_t window, float softcap, int32_t fresh, bool bf,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 0 || batch > 65535 || q_heads <= 0 || kv_heads <= 0 || page_size <= 0 ||
      table_stride <= 0 || window < 0 || capacity <= 0 || fresh < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "batch=%d q_heads=%d kv_heads=%d page_size=%d table_stride=%d window=%d "
                "capacity=%d fresh=%d",
                batch, q_heads, kv_heads, page_size, table_stride, window, capacity, fresh);
  if (q_heads % kv_heads)
    return fail(PDA_ERR_HEAD_RATIO, "query heads must be a multiple of kv heads");
  if (head_dim <= 0 || head_dim > 512)
    return fail(PDA_ERR_HEAD_DIM, "head_dim %d: 1..512", head_dim);
  if (batch == 0) return ok();
  if (!queries || !keys || !tables || !lengths || !weights || !out || (q8 && !key_scales))
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (layout != PDA_LAYOUT_ROWS && layout != PDA_LAYOUT_PAGES)
    return fail(PDA_ERR_INVALID_ARGUMENT, "unknown K/V layout %d", layout);
  if ((int64_t)page_size * kv_heads * head_dim > INT32_MAX)
    return fail(PDA_ERR_INVALID_ARGUMENT, "a page of one layer holds more than 2^31 elements");
  if (arena_rows < page_size)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld holds no whole page",
                (long long)arena_rows);
  if (!(scale == scale) || isinf(scale) || !(softcap >= 0.0f) || isinf(softcap))
    return fail(PDA_ERR_INVALID_ARGUMENT, "scale must be finite and softcap >= 0");
  if (capacity > INT32_MAX - 2 * kAddKeys)
    return fail(PDA_ERR_TOO_LONG, "capacity %d next to 2^31", capacity);
  if (((uintptr_t)queries | (uintptr_t)keys) & 15)
    return fail(PDA_ERR_ALIGNMENT, "query and key buffers must be 16-byte aligned");
  if (((uintptr_t)tables | (uintptr_t)lengths | (uintptr_t)weights | (uintptr_t)out) & 3)
    return fail(PDA_ERR_ALIGNMENT, "tables, lengths and weights must be 4-byte aligned");
  if (q8 && ((uintptr_t)key_scales & 1))
    return fail(PDA_ERR_ALIGNMENT, "fp16 scale arenas must be 2-byte aligned");
  const int group = q_heads / kv_heads;
  const int64_t grid_y = (int64_t)kv_heads * ((group + kSlots - 1) / kSlots);
  if (grid_y > 65535)
    return fail(PDA_ERR_INVALID_ARGUMENT, "%d kv heads of %d query heads", kv_heads, group);
  const size_t need = weights_workspace(batch, q_heads, capacity);
  if (!workspace || workspace_bytes < need)
    return fail(PDA_ERR_WORKSPACE, "a workspace of %zu bytes is needed (got %zu)", need,
                workspace ? workspace_bytes : (size_t)0);
  if ((uintptr_t)workspace & 255)
    return fail(PDA_ERR_ALIGNMENT, "the workspace must be 256-byte aligned");
  WeightParams prm;
  prm.q = static_cast<const f16*>(queries);
  prm.k = keys;
  prm.kscale = static_cast<const f16*>(key_scales);
  prm.tables = tables;
  prm.lengths = lengths;
  prm.weights = weights;
  prm.out = out;
  prm.pitch = (capacity + 3) & ~3;
  prm.chunk = chunk_for(planes_run(head_dim));
  prm.chunks = (capacity + prm.chunk - 1) / prm.chunk;
  prm.stats = static_cast<float2*>(workspace);
  prm.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                       stats_bytes(batch, q_heads, capacity));
  prm.arena_pages = arena_rows / page_size;
  const bool rows = layout == PDA_LAYOUT_ROWS;
  prm.page_elems = (int64_t)page_size * kv_heads * head_dim;
  prm.head_elems = rows ? head_dim : page_size * head_dim;
  prm.row_elems = rows ? kv_heads * head_dim : head_dim;
  prm.scale_page = (int64_t)page_size * kv_heads;
  prm.scale_head = rows ? 1 : page_size;
  prm.scale_row = rows ? kv_heads : 1;
  prm.table_stride = table_stride;
  prm.page_size = page_size;
  prm.hq = q_heads;
  prm.hkv = kv_heads;
  prm.head_dim = head_dim;
  prm.capacity = capacity;
  prm.window = window;
  prm.fresh = fresh;
  prm.scale_log2 = scale * kLog2e;
  prm.cap_in = softcap > 0.0f ? 2.0f * kLog2e * scale / softcap : 0.0f;
  prm.cap_out = softcap * kLog2e;
  // The grid covers `longest` keys (workgroups go on to later ones if there
  // are): a workgroup a chunk while the GPU holds them all at once, else up to
  // four chunks each, whose loads then overlap. An odd number per sequence:
  // workgroups go to the 8 XCDs in turn, and with 8 a sequence the first XCD has
  // a share of every sequence and the last only of the longest (64 sequences of
  // 512 to 8192 keys, 28 over 4 heads of 128 dims: scores 81 us with 8 and 82
  // with 16, 75 with 9 and 73 with 17).
  const int64_t span = std::max<int64_t>(1, std::min<int64_t>(longest, capacity));
  const int64_t seen =
      window > 0 ? std::min<int64_t>(span, (int64_t)window + prm.chunk) : span;
  const int64_t chunks = (seen + prm.chunk - 1) / prm.chunk;
  const int64_t one = std::max<int64_t>(1, kScoreGroups / (grid_y * batch));
  const unsigned gx = (unsigned)std::min<int64_t>(
      std::max(std::min(chunks, one), (chunks + 3) / 4), kMaxChunksX) | 1;
  const unsigned ax =
      (unsigned)std::min<int64_t>((span + kAddKeys - 1) / kAddKeys, kMaxChunksX) | 1;
  void* args[] = {&prm};
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  const void* fn = q8 ? (bf ? scores_kernel<true, true>(head_dim)
                            : scores_kernel<true, false>(head_dim))
                      : (bf ? scores_kernel<false, true>(head_dim)
                            : scores_kernel<false, false>(head_dim));
  hipError_t err = hipLaunchKernel(fn, dim3(gx, (unsigned)grid_y, batch), dim3(64 * kWaves), args,
                                   0, hs);
  if (err == hipSuccess)
    err = hipLaunchKernel((const void*)attention_weights_kernel, dim3(ax, kv_heads, batch),
                          dim3(256), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

// ---------------------------------------------------------------------------
// Selection.

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kSelectEach = 8;  // positions a thread holds
constexpr int kSelectBlock = kSelectEach * kSelectThreads;
// Positions and kept rows of a sequence: the loops go on by a block at most past
// the last, in 32 bits.
constexpr int kMaxPositions = INT32_MAX - kSelectBlock;
constexpr int kBins = 2048;

struct SelectParams {
  const float* weights;  // [batch, hkv, capacity]
  float* out_weights;    // [batch, hkv, out_capacity]
  const int32_t* tables;
  const int32_t* lengths;
  int32_t* kept;         // [batch, hkv, keep]
  int32_t* new_lengths;  // [batch]
  int64_t arena_pages;
  int32_t table_stride;
  int32_t page_size;
  int32_t hkv;
  int32_t capacity;
  int32_t out_capacity;
  int32_t keep;
  int32_t recent;
  int32_t sinks;
};

// Weights as unsigned integers of the same order; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums over the lanes up to each, by moves within rows of 16 lanes and of a row's
// last lane to the rows after it.
__device__ __forceinline__ int scan64(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // 1, 2, 4, 8 lanes on
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // rows 2 and 3
  return x;
}

// One workgroup a (sequence, kv head), a block of 8192 positions at a time, 8 a
// thread in registers (one block is read once). The rank of the least kept
// weight is found digit by digit from the top (11, 11 and 10 bits): a histogram
// of the candidates that share the digits found so far, in LDS, and the bin in
// which the count from above passes what is to be kept. Then each 64 positions
// (a wave's ballot) are counted, the counts are summed over those before, and
// the kept positions written in order; of those at the last rank the lowest
// positions are kept. Counts are integers, so their order does not matter. Bound
// by its chain of reads and meetings: 1100 positions 12 us, 128 times up to 8079
// 16 us.
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const SelectParams p) {
  constexpr int kEach = kSelectEach, kBlock = kSelectBlock;
  constexpr int kGroups = kEach * kSelectWaves;  // ballots of a block
  // (Two of each, so that a digit's need no meeting before the next one's.)
  __shared__ int s_hist[2][kBins];
  __shared__ int s_part[2][kSelectWaves];
  __shared__ int s_found[2][2];  // the digit's bin, what it has to give
  __shared__ int s_count[2];     // guarded positions, candidates
  __shared__ int s_over[kGroups], s_equal[kGroups];
  __shared__ int s_total[2];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int64_t cap = min((int64_t)p.table_stride * p.page_size, (int64_t)p.capacity);
  const int n = (int)max((int64_t)0, min((int64_t)p.lengths[b], cap));
  const float* weights = p.weights + ((int64_t)b * p.hkv + kvh) * p.capacity;
  const int32_t* table = p.tables + (int64_t)b * p.table_stride;
  const uint32_t pages = (uint32_t)min(p.arena_pages, (int64_t)INT32_MAX);
  auto count = [](uint64_t lanes) { return (int)__popcll(lanes); };
  for (int i = tid; i < kBins; i += kSelectThreads) s_hist[0][i] = 0;
  if (tid < 2) s_count[tid] = 0;
  __syncthreads();
  // This thread's positions t0 + 1024 i + tid of a block: ranks, and bits of
  // those that are guarded and of those that stand for selection.
  float x[kEach];
  uint32_t rank[kEach], guarded = 0, open = 0;
  const int blocks = (n + kBlock - 1) / kBlock;
  auto load = [&](int block) {
    guarded = open = 0;
    uint32_t page[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = min(block * kBlock + i * kSelectThreads + tid, n - 1);
      page[i] = (uint32_t)table[(uint32_t)t / (uint32_t)p.page_size];
      x[i] = weights[t];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = block * kBlock + i * kSelectThreads + tid;
      rank[i] = rank_of(x[i]);
      if (t < n && page[i] < pages) {
        if (t < p.sinks || t >= n - p.recent)
          guarded |= 1u << i;
        else
          open |= 1u << i;
      }
    }
  };
  int guards = 0, rest = 0;
  for (int block = 0; block < blocks; ++block) {
    load(block);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      guards += count(__ballot(guarded >> i & 1));
      rest += count(__ballot(open >> i & 1));
    }
  }
  if (lane == 0) {
    atomicAdd(&s_count[0], guards);
    atomicAdd(&s_count[1], rest);
  }
  __syncthreads();
  guards = s_count[0];
  rest = s_count[1];
  const int total = min(p.keep, guards + rest);
  int want = max(0, p.keep - guards);  // candidates to keep
  uint32_t least = 0;                  // rank of the least kept one
  if (want == 0) {
    least = 0xFFFFFFFFu;
  } else if (want < rest) {
    uint32_t mask = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const int bins = pass == 2 ? 1024 : 2048;
      int* hist = s_hist[pass & 1];
      int* part = s_part[pass & 1];
      int* found = s_found[pass & 1];
      for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load(block);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if ((open >> i & 1) && (rank[i] & mask) == least)
            atomicAdd(&hist[rank[i] >> shift & (bins - 1)], 1);
      }
      for (int i = tid; pass < 2 && i < kBins; i += kSelectThreads) s_hist[~pass & 1][i] = 0;
      __syncthreads();
      // Thread i takes the bins i * per .. from the top; the one in whose bins
      // the running count passes `want` names the bin.
      const int per = bins / kSelectThreads;
      int mine = 0;
      for (int i = 0; i < per; ++i) mine += hist[bins - 1 - (tid * per + i)];
      int upto = scan64(mine);
      if (lane == 63) part[w] = upto;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kSelectWaves; ++i) upto += i < w ? part[i] : 0;
      int above = upto - mine;
      if (above < want && want <= upto) {
        for (int i = 0; i < per; ++i) {
          const int bin = bins - 1 - (tid * per + i);
          if (above + hist[bin] >= want) {
            found[0] = bin;
            found[1] = want - above;
            break;
          }
          above += hist[bin];
        }
      }
      __syncthreads();
      least |= (uint32_t)found[0] << shift;
      want = found[1];
      mask |= (uint32_t)(bins - 1) << shift;
    }
  }
  // (All candidates kept: least 0, and want of them at rank 0 is enough for
  // the NaN, which alone have it.)
  int32_t* kept = p.kept + ((int64_t)b * p.hkv + kvh) * p.keep;
  float* dst = p.out_weights + ((int64_t)b * p.hkv + kvh) * p.out_capacity;
  // (One block's weights have all been read: they may be overwritten at once.)
  const bool at_once = p.out_weights && (p.out_weights != p.weights || blocks == 1);
  const uint64_t lower = (1ull << lane) - 1;
  int done = 0, equals = 0;  // kept, and met at the last rank, in the blocks before
  for (int block = 0; block < blocks; ++block) {
    if (blocks > 1) load(block);
    uint32_t over = guarded, equal = 0;
    int overs = 0, equals_here = 0;  // lane i's: of ballot i
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if ((open >> i & 1) && rank[i] > least) over |= 1u << i;
      if ((open >> i & 1) && rank[i] == least) equal |= 1u << i;
      const uint64_t o = __ballot(over >> i & 1), e = __ballot(equal >> i & 1);
      overs = lane == i ? count(o) : overs;
      equals_here = lane == i ? count(e) : equals_here;
    }
    if (lane < kEach) {
      s_over[lane * kSelectWaves + w] = overs;
      s_equal[lane * kSelectWaves + w] = equals_here;
    }
    __syncthreads();
    if (w < 2) {  // exclusive sums: one wave each, two groups a lane
      int* c = w ? s_equal : s_over;
      const int a = c[2 * lane], z = c[2 * lane + 1];
      const int upto = scan64(a + z);
      c[2 * lane] = upto - a - z;
      c[2 * lane + 1] = upto - z;
      if (lane == 63) s_total[w] = upto;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint64_t o = __ballot(over >> i & 1), e = __ballot(equal >> i & 1);
      const int group = i * kSelectWaves + w;
      const int before = equals + s_equal[group];  // at the last rank, lower positions
      const int at = done + s_over[group] + min(before, want) - min(equals, want);
      const int ties = before + count(e & lower);
      const bool take = (over >> i & 1) || ((equal >> i & 1) && ties < want);
      if (take) {
        const int t = block * kBlock + i * kSelectThreads + tid;
        const int to = at + count(o & lower) + min(ties, want) - min(before, want);
        kept[to] = t;
        if (at_once) dst[to] = x[i];
      }
    }
    done += s_total[0] + min(equals + s_total[1], want) - min(equals, want);
    equals += s_total[1];
    __syncthreads();
  }
  for (int i = total + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
  if (kvh == 0 && tid == 0) p.new_lengths[b] = total;
  if (!p.out_weights || at_once) return;
  // In place the kept positions' weights go to the front 1024 at a time: a later
  // stretch's sources lie past every place written so far.
  __threadfence_block();
  __syncthreads();
  for (int i0 = 0; i0 < total; i0 += kSelectThreads) {
    const int i = i0 + tid;
    float y = 0.0f;
    if (i < total) y = weights[kept[i]];
    wait_loads();
    __syncthreads();
    if (i < total) dst[i] = y;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Packing.

struct MoveParams {
  char* arena[2];        // keys and values, or their scales; [1] may be null
  const int32_t* kept;   // [batch, hkv, keep]
  const int32_t* new_lengths;
  const int32_t* tables;
  const int32_t* out_tables;
  int64_t arena_pages;
  int64_t page_bytes;
  int64_t head_bytes;
  int64_t row_bytes;     // between rows of a page and head
  int32_t width;         // bytes of a row
  int32_t table_stride;
  int32_t out_stride;
  int32_t page_size;
  int32_t hkv;
  int32_t keep;
};

// Byte offset of position t's row, -1 if its page is not in the arena (or t is
// negative).
__device__ __forceinline__ int64_t row_at(const MoveParams& p, const int32_t* table, int stride,
                                          int t, int kvh) {
  const uint32_t pi = (uint32_t)t / (uint32_t)p.page_size;
  const uint32_t page = (uint32_t)table[min(pi, (uint32_t)stride - 1)];
  if (t < 0 || pi >= (uint32_t)stride || page >= (uint32_t)min(p.arena_pages, (int64_t)INT32_MAX))
    return -1;
  return page * p.page_bytes + kvh * p.head_bytes +
         (int64_t)(t - (int)pi * p.page_size) * p.row_bytes;
}

// Kept rows to other pages: a thread moves one piece of V of kEach rows, their
// positions, places and then the rows looked up together. Moves each byte once,
// which bounds it: 32 sequences' 2048 rows of 4 heads of 128 dims, keys and values,
// 268 MB in 58 us (4.6 TB/s; with rows kept in the caches, where nothing looks for
// them before they are gone, 60).
template <class V>
__global__ __launch_bounds__(256) void evict_copy_kernel(const MoveParams p) {
  constexpr int kEach = 8;
  const int kvh = blockIdx.y % p.hkv, b = blockIdx.z;
  char* arena = p.arena[blockIdx.y / p.hkv];
  const int pieces = p.width / (int)sizeof(V);
  const int across = min(pieces, 256), rows = 256 / across;  // threads a row, rows a pass
  const int total = min(p.new_lengths[b], p.keep);
  const int32_t* kept = p.kept + ((int64_t)b * p.hkv + kvh) * p.keep;
  const int32_t* from = p.tables + (int64_t)b * p.table_stride;
  const int32_t* to = p.out_tables + (int64_t)b * p.out_stride;
  const int mine = (int)threadIdx.x / across, first = (int)threadIdx.x % across;
  if (mine >= rows) return;
  for (int64_t r0 = (int64_t)blockIdx.x * (rows * kEach); r0 < total;
       r0 += (int64_t)gridDim.x * (rows * kEach)) {
    int64_t s[kEach], d[kEach];
    int pos[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int64_t row = r0 + rows * j + mine;
      pos[j] = row < total ? kept[row] : -1;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      s[j] = row_at(p, from, p.table_stride, pos[j], kvh);
      d[j] = row_at(p, to, p.out_stride, (int)(r0 + rows * j + mine), kvh);
      if (pos[j] < 0 || d[j] < 0 || d[j] == s[j]) s[j] = -1;
    }
    for (int c = first; c < pieces; c += across) {
      V x[kEach];
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (s[j] >= 0)
          x[j] = __builtin_nontemporal_load(
              reinterpret_cast<const V*>(arena + s[j] + c * (int64_t)sizeof(V)));
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (s[j] >= 0)
          __builtin_nontemporal_store(
              x[j], reinterpret_cast<V*>(arena + d[j] + c * (int64_t)sizeof(V)));
    }
  }
}

// Kept rows to the front of their own pages. A row's place lies at or before
// it, and rows keep their order, so a workgroup that owns a slice of the rows
// (kSlice bytes of every row of a sequence and kv head) may walk them in
// stretches: a stretch's places hold no source of a later one. Within a stretch
// all loads come before the first store. The rows above in place 102 us: one
// workgroup walks each slice, where the copy has as many as there are rows.
template <class V>
__global__ __launch_bounds__(256) void evict_pack_kernel(const MoveParams p) {
  constexpr int kSlice = sizeof(V) >= 4 ? 4 * sizeof(V) : sizeof(V);  // bytes
  constexpr int kPieces = kSlice / (int)sizeof(V);
  constexpr int kRows = 256 / kPieces;  // rows per pass
  constexpr int kEach = 8;
  const int slices = (p.width + kSlice - 1) / kSlice;
  const int slice = blockIdx.x % slices;
  char* arena = p.arena[blockIdx.x / slices];
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int c = slice * kSlice + (threadIdx.x % kPieces) * (int)sizeof(V);
  const bool mine = c < p.width;
  const int total = min(p.new_lengths[b], p.keep);
  const int32_t* kept = p.kept + ((int64_t)b * p.hkv + kvh) * p.keep;
  const int32_t* table = p.tables + (int64_t)b * p.table_stride;
  for (int r0 = 0; r0 < total; r0 += kRows * kEach) {
    V x[kEach];
    int64_t at[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int row = r0 + kRows * j + (int)threadIdx.x / kPieces;
      at[j] = -1;
      if (mine && row < total) {
        const int from = kept[row];
        if (from != row) {
          const int64_t s = row_at(p, table, p.table_stride, from, kvh);
          const int64_t d = row_at(p, table, p.table_stride, row, kvh);
          if (s >= 0 && d >= 0) {
            x[j] = *reinterpret_cast<const V*>(arena + s + c);
            at[j] = d + c;
          }
        }
      }
    }
    wait_loads();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (at[j] >= 0) *reinterpret_cast<V*>(arena + at[j]) = x[j];
    __syncthreads();
  }
}

}  // namespace

extern "C" {

int pda_attention_weights_workspace_bytes(int32_t batch, int32_t q_heads, int32_t capacity,
                                          size_t* bytes) {
  if (batch < 0 || q_heads <= 0 || capacity <= 0 || !bytes)
    return fail(PDA_ERR_INVALID_ARGUMENT, "batch=%d q_heads=%d capacity=%d", batch, q_heads,
                capacity);
  *bytes = weights_workspace(batch, q_heads, capacity);
  return ok();
}

int pda_attention_weights(const void* queries, const void* keys, const int32_t* tables,
                          const int32_t* lengths, const float* weights, float* out, int32_t batch,
                          int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t page_size,
                          int32_t table_stride, int64_t arena_rows, int32_t layout,
                          int32_t capacity, int32_t longest, float scale, int32_t window,
                          float softcap, int32_t fresh, void* workspace, size_t workspace_bytes,
                          void* stream) {
  return attention_weights(queries, keys, nullptr, false, tables, lengths, weights, out, batch,
                           q_heads, kv_heads, head_dim, page_size, table_stride, arena_rows,
                           layout, capacity, longest, scale, window, softcap, fresh, false,
                           workspace, workspace_bytes, stream);
}

int pda_attention_weights_bf16(const void* queries, const void* keys, const int32_t* tables,
                               const int32_t* lengths, const float* weights, float* out,
                               int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                               int32_t page_size, int32_t table_stride, int64_t arena_rows,
                               int32_t layout, int32_t capacity, int32_t longest, float scale,
                               int32_t window, float softcap, int32_t fresh, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return attention_weights(queries, keys, nullptr, false, tables, lengths, weights, out, batch,
                           q_heads, kv_heads, head_dim, page_size, table_stride, arena_rows,
                           layout, capacity, longest, scale, window, softcap, fresh, true,
                           workspace, workspace_bytes, stream);
}

int pda_attention_weights_q8(const void* queries, const void* keys, const void* key_scales,
                             const int32_t* tables, const int32_t* lengths, const float* weights,
                             float* out, int32_t batch, int32_t q_heads, int32_t kv_heads,
                             int32_t head_dim, int32_t page_size, int32_t table_stride,
                             int64_t arena_rows, int32_t layout, int32_t capacity,
                             int32_t longest, float scale, int32_t window, float softcap,
                             int32_t fresh, void* workspace, size_t workspace_bytes,
                             void* stream) {
  return attention_weights(queries, keys, key_scales, true, tables, lengths, weights, out, batch,
                           q_heads, kv_heads, head_dim, page_size, table_stride, arena_rows,
                           layout, capacity, longest, scale, window, softcap, fresh, false,
                           workspace, workspace_bytes, stream);
}

int pda_attention_weights_q8_bf16(const void* queries, const void* keys, const void* key_scales,
                                  const int32_t* tables, const int32_t* lengths,
                                  const float* weights, float* out, int32_t batch,
                                  int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                  int32_t page_size, int32_t table_stride, int64_t arena_rows,
                                  int32_t layout, int32_t capacity, int32_t longest, float scale,
                                  int32_t window, float softcap, int32_t fresh, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  return attention_weights(queries, keys, key_scales, true, tables, lengths, weights, out, batch,
                           q_heads, kv_heads, head_dim, page_size, table_stride, arena_rows,
                           layout, capacity, longest, scale, window, softcap, fresh, true,
                           workspace, workspace_bytes, stream);
}

int pda_evict_select(const float* weights, float* out_weights, const int32_t* tables,
                     const int32_t* lengths, int32_t* kept, int32_t* new_lengths, int32_t batch,
                     int32_t kv_heads, int32_t page_size, int32_t table_stride,
                     int64_t arena_rows, int32_t capacity, int32_t out_capacity, int32_t keep,
                     int32_t recent, int32_t sinks, void* stream) {
  if (batch < 0 || batch > 65535 || kv_heads <= 0 || page_size <= 0 || table_stride <= 0 ||
      capacity <= 0 || keep <= 0 || recent < 0 || sinks < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "batch=%d kv_heads=%d page_size=%d table_stride=%d capacity=%d keep=%d recent=%d "
                "sinks=%d",
                batch, kv_heads, page_size, table_stride, capacity, keep, recent, sinks);
  if ((int64_t)recent + sinks > keep)
    return fail(PDA_ERR_INVALID_ARGUMENT, "recent %d and sinks %d exceed keep %d", recent, sinks,
                keep);
  if (batch == 0) return ok();
  if (!weights || !tables || !lengths || !kept || !new_lengths)
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (out_weights && out_capacity < std::min(keep, capacity))
    return fail(PDA_ERR_INVALID_ARGUMENT, "out_capacity %d holds fewer than %d weights",
                out_capacity, std::min(keep, capacity));
  if (out_weights == weights && out_weights && out_capacity != capacity)
    return fail(PDA_ERR_INVALID_ARGUMENT, "weights packed in place keep their capacity");
  if (arena_rows < page_size)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld holds no whole page",
                (long long)arena_rows);
  if (capacity > kMaxPositions || keep > kMaxPositions)
    return fail(PDA_ERR_TOO_LONG, "capacity %d or keep %d next to 2^31", capacity, keep);
  if (((uintptr_t)weights | (uintptr_t)out_weights | (uintptr_t)tables | (uintptr_t)lengths |
       (uintptr_t)kept | (uintptr_t)new_lengths) & 3)
    return fail(PDA_ERR_ALIGNMENT, "all buffers must be 4-byte aligned");
  SelectParams prm;
  prm.weights = weights;
  prm.out_weights = out_weights;
  prm.tables = tables;
  prm.lengths = lengths;
  prm.kept = kept;
  prm.new_lengths = new_lengths;
  prm.arena_pages = arena_rows / page_size;
  prm.table_stride = table_stride;
  prm.page_size = page_size;
  prm.hkv = kv_heads;
  prm.capacity = capacity;
  prm.out_capacity = out_capacity;
  prm.keep = keep;
  prm.recent = recent;
  prm.sinks = sinks;
  void* args[] = {&prm};
  const hipError_t err =
      hipLaunchKernel((const void*)evict_select_kernel, dim3(kv_heads, batch),
                      dim3(kSelectThreads), args, 0, static_cast<hipStream_t>(stream));
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

int pda_evict_move(void* arena, void* arena2, int32_t width, const int32_t* kept,
                   const int32_t* new_lengths, const int32_t* tables, const int32_t* out_tables,
                   int32_t batch, int32_t kv_heads, int32_t page_size, int32_t table_stride,
                   int32_t out_stride, int64_t arena_rows, int32_t layout, int32_t keep,
                   void* stream) {
  if (batch < 0 || batch > 65535 || kv_heads <= 0 || kv_heads > 32767 || page_size <= 0 ||
      table_stride <= 0 || out_stride <= 0 || keep <= 0 || width <= 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "batch=%d kv_heads=%d page_size=%d table_stride=%d out_stride=%d keep=%d width=%d",
                batch, kv_heads, page_size, table_stride, out_stride, keep, width);
  if (batch == 0) return ok();
  if (!arena || !kept || !new_lengths || !tables || !out_tables)
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (layout != PDA_LAYOUT_ROWS && layout != PDA_LAYOUT_PAGES)
    return fail(PDA_ERR_INVALID_ARGUMENT, "unknown K/V layout %d", layout);
  if (arena_rows < page_size)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld holds no whole page",
                (long long)arena_rows);
  if (keep > kMaxPositions) return fail(PDA_ERR_TOO_LONG, "keep %d next to 2^31", keep);
  if (((uintptr_t)kept | (uintptr_t)new_lengths | (uintptr_t)tables | (uintptr_t)out_tables) & 3)
    return fail(PDA_ERR_ALIGNMENT, "index buffers must be 4-byte aligned");
  if (arena2 == arena) arena2 = nullptr;  // (once: two walks of one slice would race)
  MoveParams prm;
  prm.arena[0] = static_cast<char*>(arena);
  prm.arena[1] = static_cast<char*>(arena2);
  prm.kept = kept;
  prm.new_lengths = new_lengths;
  prm.tables = tables;
  prm.out_tables = out_tables;
  prm.arena_pages = arena_rows / page_size;
  prm.page_bytes = (int64_t)page_size * kv_heads * width;
  const bool rows = layout == PDA_LAYOUT_ROWS;
  prm.head_bytes = rows ? width : (int64_t)page_size * width;
  prm.row_bytes = rows ? (int64_t)kv_heads * width : width;
  prm.width = width;
  prm.table_stride = table_stride;
  prm.out_stride = out_stride;
  prm.page_size = page_size;
  prm.hkv = kv_heads;
  prm.keep = keep;
  // The widest piece that rows and buffers are aligned to.
  const uintptr_t mis = (uintptr_t)arena | (uintptr_t)arena2 | (uintptr_t)width;
  const int vec = mis % 16 == 0 ? 16 : mis % 4 == 0 ? 4 : mis % 2 == 0 ? 2 : 1;
  const int arenas = arena2 ? 2 : 1;
  void* args[] = {&prm};
  const void* fn;
  dim3 grid;
  if (tables == out_tables) {
    const int slice = vec >= 4 ? 4 * vec : vec;
    const int64_t gx = (int64_t)arenas * ((width + slice - 1) / slice);
    if (gx > INT32_MAX) return fail(PDA_ERR_INVALID_ARGUMENT, "width %d", width);
    fn = vec == 16  ? (const void*)evict_pack_kernel<u32x4>
         : vec == 4 ? (const void*)evict_pack_kernel<uint32_t>
         : vec == 2 ? (const void*)evict_pack_kernel<uint16_t>
                    : (const void*)evict_pack_kernel<uint8_t>;
    grid = dim3((unsigned)gx, kv_heads, batch);
  } else {
    const int rows = 256 / std::min(width / vec, 256);
    const int64_t per = ((int64_t)keep + 8 * rows - 1) / (8 * rows);
    fn = vec == 16  ? (const void*)evict_copy_kernel<u32x4>
         : vec == 4 ? (const void*)evict_copy_kernel<uint32_t>
         : vec == 2 ? (const void*)evict_copy_kernel<uint16_t>
                    : (const void*)evict_copy_kernel<uint8_t>;
    grid = dim3((unsigned)std::min<int64_t>(per, 4096), arenas * kv_heads, batch);
  }
  const hipError_t err =
      hipLaunchKernel(fn, grid, dim3(256), args, 0, static_cast<hipStream_t>(stream));
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

}  // extern "C"
