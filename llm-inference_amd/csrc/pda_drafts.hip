// Attention for trees of drafted tokens over the paged cache, and the step that
// keeps the accepted ones, for MI355X (gfx950), C-ABI in pda.h
// (pda_tree_attention, pda_commit_drafts). No counterpart in the reference, which
// decodes one token a sequence and step.
//
// Node i of a sequence's tree lies behind the l rows that the sequence holds, in
// row l + i, and attends to the held rows and to the nodes whose bits its mask has
// (itself and its ancestors): flops 4 D a (query head, node, visible key); the
// rows of a kv head are read once for up to 256 (node, query head) pairs of it.
//
// Rows of queries. A unit is (sequence, kv head, 128 or 256 of its node and head
// pairs); its keys come in tiles of 64. The tiles of all units form one stream that is
// cut into equal ranges, one a workgroup, whatever the lengths: a unit inside one
// range is written at once, the pieces of one that is cut are joined by a second
// kernel. The cuts depend on the lengths alone, so repeated calls give the same bits.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "pda.h"
#include "pda_internal.h"
#include "pda_tree.h"

namespace {

using pda_internal::fail;
using pda_internal::ok;
using pda_internal::overlap;
using pda_internal::Span;

using namespace pda_tree;

// Joins the pieces of the unit that is cut and ends in a workgroup's range: with M the
// largest of their maxima, the outputs are sum 2^(m - M) o / sum 2^(m - M) l. A wave
// takes 32 rows, a quarter of their dims and every PHASES-th piece, the lanes as in the
// kernel that left them; the waves' sums meet in LDS, in a fixed order.
//
// PHASES 1: a workgroup for each of the ranges, whether a cut unit ends there or not. 4:
// where a few units have many pieces each, a workgroup for each unit, which looks for its
// cut among the ranges' (one sequence of 40000 rows, 28/4 heads of 128, 78 pieces a unit:
// 67 -> 48 us a call; 16 pieces a unit in ranges without one: 22 -> 31 us the join).
constexpr int kManyPhases = 4;

// (m, sum, outputs) of some pieces plus those of others.
template <int N>
struct Joined {
  float top, sum;
  float4 o[N];
  __device__ __forceinline__ void clear() {
    top = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  // (Pieces of which the row sees nothing hold zeros; one of NaN is not empty.)
  __device__ __forceinline__ void add(float m, float l, const float4 (&x)[N]) {
    if (m == -INFINITY && l == 0.0f) return;
    const float now = fmaxf(top, m);
    const float f = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top - now);
    const float g = __builtin_amdgcn_exp2f(m - now);
    top = now;
    sum = fmaf(sum, f, l * g);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i].x = fmaf(o[i].x, f, x[i].x * g);
      o[i].y = fmaf(o[i].y, f, x[i].y * g);
      o[i].z = fmaf(o[i].z, f, x[i].z * g);
      o[i].w = fmaf(o[i].w, f, x[i].w * g);
    }
  }
};

template <int D, bool BF, int PHASES>
__global__ __launch_bounds__(256 * PHASES) void tree_join_kernel(const TreeParams p) {
  constexpr int kShare = D / 8 / 4;  // groups of 8 dims a wave takes
  constexpr int kAtOnce = kShare <= 4 ? 4 : 2;  // pieces loaded together
  const int w = blockIdx.y, waves = gridDim.y;
  const int lane = threadIdx.x & 63, part = (threadIdx.x >> 6) & 3, phase = threadIdx.x >> 8;
  int g = blockIdx.x;
  if constexpr (PHASES > 1) {
    // The range in which the blockIdx.x-th of the cut units ends.
    static_assert(256 * PHASES >= groups_for(128, 4), "a thread for each range");
    __shared__ int s_before[4 * PHASES], s_found;
    const int wave = threadIdx.x >> 6;
    const bool mine = (int)threadIdx.x < p.groups && p.cuts[threadIdx.x].rows > 0;
    const uint64_t all = __ballot(mine);
    if (lane == 0) s_before[wave] = __popcll(all);
    if (threadIdx.x == 0) s_found = -1;
    __syncthreads();
    int at = __popcll(all & ((1ull << lane) - 1));
    for (int i = 0; i < wave; ++i) at += s_before[i];
    if (mine && at == (int)blockIdx.x) s_found = threadIdx.x;
    __syncthreads();
    g = s_found;
    if (g < 0) return;
  }
  const Cut cut = p.cuts[g];
  if (cut.rows <= 32 * w) return;
  // Its pieces: the first, then those of the workgroups up to this one.
  const int count = g - cut.group + 2;
  auto piece = [&](int i) {
    return (int64_t)(i == 0 ? cut.piece : 2 * (cut.group + i - 1)) * waves + w;
  };
  Joined<kShare> all;
  all.clear();
  for (int i0 = phase; i0 < count; i0 += PHASES * kAtOnce) {
    float2 ml[kAtOnce];
    float4 o[kAtOnce][kShare];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t at = piece(min(i0 + PHASES * j, count - 1));
      ml[j] = p.part_ml[at * 32 + (lane & 31)];
      const float4* src = reinterpret_cast<const float4*>(p.part_o) + at * (D / 8 * 64) +
                          part * kShare * 64 + lane;
#pragma unroll
      for (int i = 0; i < kShare; ++i) o[j][i] = src[64 * i];
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (i0 + PHASES * j < count) all.add(ml[j].x, ml[j].y, o[j]);
  }
  if constexpr (PHASES > 1) {
    __shared__ float s_join[PHASES - 1][4][kShare * 4 + 2][64];
    if (phase > 0) {
      float (&to)[kShare * 4 + 2][64] = s_join[phase - 1][part];
      to[0][lane] = all.top;
      to[1][lane] = all.sum;
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        to[2 + 4 * i][lane] = all.o[i].x;
        to[3 + 4 * i][lane] = all.o[i].y;
        to[4 + 4 * i][lane] = all.o[i].z;
        to[5 + 4 * i][lane] = all.o[i].w;
      }
    }
    __syncthreads();
    if (phase > 0) return;
    for (int f = 1; f < min(PHASES, count); ++f) {
      const float (&from)[kShare * 4 + 2][64] = s_join[f - 1][part];
      float4 o[kShare];
#pragma unroll
      for (int i = 0; i < kShare; ++i)
        o[i] = make_float4(from[2 + 4 * i][lane], from[3 + 4 * i][lane], from[4 + 4 * i][lane],
                           from[5 + 4 * i][lane]);
      all.add(from[0][lane], from[1][lane], o);
    }
  }
  const int r = 32 * w + (lane & 31);
  if (r >= cut.rows) return;
  const int G = p.hq / p.hkv, row = cut.first + r;
  const float inv = all.sum == 0.0f ? 0.0f : 1.0f / all.sum;
  f16* dst = p.out + ((int64_t)(cut.token + row / G) * p.hq + cut.kvh * G + row % G) * p.dim;
#pragma unroll
  for (int i = 0; i < kShare; ++i) {
    const int d = 8 * (part * kShare + i) + 4 * (lane >> 5);
    const f16x4 y = {round16<BF>(all.o[i].x * inv), round16<BF>(all.o[i].y * inv),
                     round16<BF>(all.o[i].z * inv), round16<BF>(all.o[i].w * inv)};
    if (d < p.dim) *reinterpret_cast<f16x4*>(dst + d) = y;
  }
}

template <bool BF, int PHASES>
const void* tree_join_for(int width) {
  return width == 64    ? reinterpret_cast<const void*>(tree_join_kernel<64, BF, PHASES>)
         : width == 96  ? reinterpret_cast<const void*>(tree_join_kernel<96, BF, PHASES>)
         : width == 128 ? reinterpret_cast<const void*>(tree_join_kernel<128, BF, PHASES>)
                        : reinterpret_cast<const void*>(tree_join_kernel<256, BF, PHASES>);
}

// Pieces' outputs, (max, sum) pairs and the cuts: 2 pieces a workgroup, of 32 rows a
// wave. As many rows with four waves a workgroup as with eight.
size_t tree_workspace(int width) {
  const size_t rows = 2 * (size_t)groups_for(width, 4) * 4 * 32;
  return rows * width * 4 + rows * 8 + groups_for(width, 4) * sizeof(Cut);
}

int tree_attention(const void* queries, const void* keys, const void* values,
                   const void* key_scales, const void* value_scales, bool q8, bool bf16_elems,
                   const int32_t* tables, const int32_t* lengths, const int32_t* starts,
                   const uint64_t* masks, void* out, int32_t tokens, int32_t batch,
                   int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t page_size,
                   int32_t table_stride, int64_t arena_rows, int32_t layout, float scale,
                   int32_t window, float softcap, void* workspace, size_t workspace_bytes,
                   void* stream) {
  if (tokens < 0 || batch < 0 || q_heads <= 0 || kv_heads <= 0 || page_size <= 0 ||
      table_stride < 0 || window < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "tokens=%d batch=%d q_heads=%d kv_heads=%d page_size=%d table_stride=%d window=%d",
                tokens, batch, q_heads, kv_heads, page_size, table_stride, window);
  if (q_heads % kv_heads)
    return fail(PDA_ERR_HEAD_RATIO, "query heads must be a multiple of kv heads");
  const int width = width_for(head_dim);
  if (width == 0)
    return fail(PDA_ERR_HEAD_DIM, "head_dim %d: trees are served at multiples of 8 up to 256",
                head_dim);
  if (!(scale == scale) || isinf(scale) || !(softcap >= 0.0f) || isinf(softcap))
    return fail(PDA_ERR_INVALID_ARGUMENT, "scale must be finite and softcap >= 0");
  if (layout != PDA_LAYOUT_ROWS && layout != PDA_LAYOUT_PAGES)
    return fail(PDA_ERR_INVALID_ARGUMENT, "unknown K/V layout %d", layout);
  if ((int64_t)page_size * kv_heads > INT32_MAX / head_dim)
    return fail(PDA_ERR_INVALID_ARGUMENT, "a page of one layer holds more than 2^31 elements");
  if (arena_rows < page_size)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld holds no whole page",
                (long long)arena_rows);
  // Rows of a sequence's trees are counted in 32 bits.
  const int G = q_heads / kv_heads;
  if ((int64_t)tokens * q_heads > INT32_MAX)
    return fail(PDA_ERR_TOO_LONG, "%d nodes of %d query heads exceed one launch", tokens, q_heads);
  if (tokens == 0) return ok();
  if (!queries || !out || (batch > 0 && (!keys || !values || !tables || !lengths || !starts ||
                                         !masks || (q8 && (!key_scales || !value_scales)))))
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (batch > 0 && table_stride == 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "empty page tables hold no node");
  if (((uintptr_t)queries | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)out) & 15)
    return fail(PDA_ERR_ALIGNMENT, "query, K/V and output buffers must be 16-byte aligned");
  if (q8 && (((uintptr_t)key_scales | (uintptr_t)value_scales) & 1))
    return fail(PDA_ERR_ALIGNMENT, "fp16 scale arenas must be 2-byte aligned");
  if ((((uintptr_t)tables | (uintptr_t)lengths | (uintptr_t)starts) & 3) || ((uintptr_t)masks & 7))
    return fail(PDA_ERR_ALIGNMENT, "int32 buffers must be 4-byte aligned, masks 8-byte aligned");
  const size_t need = tree_workspace(width);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))
    return fail(PDA_ERR_WORKSPACE, "a 256-byte aligned workspace of %zu bytes is needed (got %zu)",
                need, workspace ? workspace_bytes : (size_t)0);

  TreeParams prm;
  prm.q = static_cast<const f16*>(queries);
  prm.k = keys;
  prm.v = values;
  prm.kscale = static_cast<const f16*>(key_scales);
  prm.vscale = static_cast<const f16*>(value_scales);
  prm.tables = tables;
  prm.lengths = lengths;
  prm.starts = starts;
  prm.masks = masks;
  prm.out = static_cast<f16*>(out);
  // Eight waves, two to a SIMD, where the sequences' trees have more rows than four
  // waves hold: their keys and values are then read once where they were read twice.
  const bool exact = width == head_dim;
  const int waves =
      exact && width <= 128 && (int64_t)tokens * G > 4 * 32 * (int64_t)batch ? 8 : 4;
  prm.groups = groups_for(width, waves);
  prm.rows = 32 * waves;
  const size_t pieces = 2 * (size_t)prm.groups * prm.rows;
  char* ws = static_cast<char*>(workspace);
  prm.part_o = reinterpret_cast<float*>(ws);
  ws += pieces * width * 4;
  prm.part_ml = reinterpret_cast<float2*>(ws);
  ws += pieces * 8;
  prm.cuts = reinterpret_cast<Cut*>(ws);
  prm.arena_pages = arena_rows / page_size;
  prm.page_elems = (int64_t)page_size * kv_heads * head_dim;
  prm.scale_page = (int64_t)page_size * kv_heads;
  const bool rows = layout == PDA_LAYOUT_ROWS;
  prm.row_elems = rows ? kv_heads * head_dim : head_dim;
  prm.head_elems = rows ? head_dim : page_size * head_dim;
  prm.scale_row = rows ? kv_heads : 1;
  prm.scale_head = rows ? 1 : page_size;
  prm.stride = table_stride;
  prm.page_size = page_size;
  prm.tokens = tokens;
  prm.batch = batch;
  prm.hq = q_heads;
  prm.hkv = kv_heads;
  prm.dim = head_dim;
  prm.window = window;
  prm.shape = shape_of(scale, softcap);
  void* args[] = {&prm};
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  const void* fn = q8 ? (bf16_elems ? tree_kernel_q8_bf16 : tree_kernel_q8)(width, waves, exact)
                      : (bf16_elems ? tree_kernel_bf16 : tree_kernel_f16)(width, waves, exact);
  hipError_t err = hipLaunchKernel(fn, dim3(prm.groups), dim3(64 * waves), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  if (batch == 0) return ok();
  // (As many units as there may be, each of some groups / units pieces.)
  const int64_t units =
      ((int64_t)tokens * G + (int64_t)(prm.rows - 1) * batch) / prm.rows * kv_heads;
  const bool many = 8 * units < prm.groups;
  const void* join = many ? (bf16_elems ? tree_join_for<true, kManyPhases>(width)
                                        : tree_join_for<false, kManyPhases>(width))
                          : (bf16_elems ? tree_join_for<true, 1>(width)
                                        : tree_join_for<false, 1>(width));
  err = hipLaunchKernel(join, dim3(many ? (unsigned)units : (unsigned)prm.groups, waves),
                        dim3(many ? 256 * kManyPhases : 256), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "join launch failed: %s", hipGetErrorString(err));
  return ok();
}

// ---------------------------------------------------------------------------
// Acceptance and the move of the accepted rows.

constexpr int kCommitLayers = 48;  // a launch's arguments hold as many

struct CommitParams {
  const int32_t* tables;   // [batch, stride]
  const int32_t* lengths;  // [batch]
  const int32_t* starts;   // [batch + 1]
  const int32_t* parents;  // [tokens]
  const void* drafted;     // [tokens] int64 or int32
  const void* targets;
  int32_t* out_lengths;    // [batch]
  int32_t* accepted;       // [batch]
  int32_t* path;           // [batch, 64]
  int64_t* following;      // [batch]
  int64_t arena_pages;
  int32_t wide;            // tokens of 64 bits
  int32_t tokens;
  int32_t batch;
  int32_t stride;
  int32_t page_size;
  int32_t hkv;
  int32_t layout;
  int32_t width;           // bytes of a row of keys or values
  int32_t stores;          // of a layer: 2, or 4 with scales
  void* store[4 * kCommitLayers];
};

// A workgroup takes one sequence and one store (a layer's keys, values or scales).
// Every wave walks the tree by itself: a lane holds a node, a turn finds the first
// child whose token is what the model chose after the last accepted node. Then the
// accepted rows move to the places behind the held rows, in order: entry i of the
// path is at least i, so a row's place was read by the rows before it or by itself,
// and what a wave moves at once it reads before it writes. Bound by that chain of reads: a
// sequence, 8 layers of 4 stores 4.5 us; 64 sequences, 12 layers of 4 heads of 128 9.9 us.
__global__ __launch_bounds__(kThreads) void commit_drafts_kernel(const CommitParams p) {
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int first = max(0, min(p.starts[b], p.tokens));
  const int n = min(max(first, min(p.starts[b + 1], p.tokens)) - first, kNodes);
  const int held = max(0, p.lengths[b]);
  int parent = -2;
  int64_t token = 0, target = 0;
  if (lane < n) {
    const int at = first + lane;
    parent = p.parents[at];
    token = p.wide ? static_cast<const int64_t*>(p.drafted)[at]
                   : static_cast<const int32_t*>(p.drafted)[at];
    target = p.wide ? static_cast<const int64_t*>(p.targets)[at]
                    : static_cast<const int32_t*>(p.targets)[at];
  }
  int count = n > 0 ? 1 : 0, last = 0, mine = lane == 0 && n > 0 ? 0 : -1;  // lane i: entry i
  while (count > 0 && count < kNodes) {
    const int64_t want = __shfl(target, last);
    const uint64_t fits = __ballot(lane > last && parent == last && token == want);
    if (fits == 0) break;
    last = __builtin_ctzll(fits);
    if (lane == count) mine = last;
    ++count;
  }
  if (blockIdx.y == 0 && w == 0) {
    p.path[(int64_t)b * kNodes + lane] = mine;
    if (lane == (count > 0 ? last : 0)) {
      p.following[b] = count > 0 ? target : -1;
      p.accepted[b] = count;
      p.out_lengths[b] = (int)min((int64_t)held + count, (int64_t)INT32_MAX);
    }
  }
  // Lane i: the rows that entry i moves from and to, in rows of the arena (-1: none).
  int64_t from = -1, to = -1;
  if (lane < count && mine != lane) {
    const int64_t src = (int64_t)held + mine, dst = (int64_t)held + lane;
    const int64_t sp = src / p.page_size, dp = dst / p.page_size;
    if (sp < p.stride && dp < p.stride) {
      const int s = p.tables[(int64_t)b * p.stride + sp], d = p.tables[(int64_t)b * p.stride + dp];
      if (s >= 0 && s < p.arena_pages && d >= 0 && d < p.arena_pages) {
        from = (int64_t)s * p.page_size + src % p.page_size;
        to = (int64_t)d * p.page_size + dst % p.page_size;
      }
    }
  }
  const uint64_t moves = __ballot(to >= 0);
  if (moves == 0) return;

  char* store = static_cast<char*>(p.store[blockIdx.y]);
  const int width = blockIdx.y % p.stores < 2 ? p.width : 2;
  auto place = [&](int64_t row, int head) {
    const int64_t page = row / p.page_size, slot = row - page * p.page_size;
    return (p.layout == PDA_LAYOUT_ROWS
                ? row * p.hkv + head
                : (page * p.hkv + head) * p.page_size + slot) * width;
  };
  // Units of the widest load that rows are multiples of.
  auto move = [&](auto zero) {
    typedef decltype(zero) U;
    const int units = width / (int)sizeof(U);  // of a row
    const int each = units < 64 ? 64 / units : 1;  // rows that the wave moves at once
    for (int head = w; head < p.hkv; head += kThreads / 64) {
      uint64_t left = moves;
      while (left) {
        // Lane: a row of the next `each` and its unit there.
        const int which = units < 64 ? lane / units : 0;
        uint64_t mask = left;
        int entry = -1;
        for (int i = 0; i < each && mask; ++i) {
          const int e = __builtin_ctzll(mask);
          if (i == which) entry = e;
          mask &= mask - 1;
        }
        left = mask;
        const int64_t rf = __shfl(from, entry < 0 ? 0 : entry);
        const int64_t rt = __shfl(to, entry < 0 ? 0 : entry);
        const bool on = entry >= 0 && which < each;
        // (Rows of over 64 units go in turns; each lane reads and writes its own.)
        for (int u = units < 64 ? lane % units : lane; u < units; u += 64) {
          if (on) {
            const U x = *reinterpret_cast<const U*>(store + place(rf, head) + (int64_t)u * sizeof(U));
            *reinterpret_cast<U*>(store + place(rt, head) + (int64_t)u * sizeof(U)) = x;
          }
        }
      }
    }
  };
  const uint32_t fit = (uint32_t)width | (uint32_t)(uintptr_t)store;
  if (fit % 16 == 0)
    move(u32x4{});
  else if (fit % 4 == 0)
    move((uint32_t)0);
  else if (fit % 2 == 0)
    move((uint16_t)0);
  else
    move((uint8_t)0);
}

}  // namespace

extern "C" {

int pda_tree_workspace_bytes(int32_t head_dim, size_t* bytes) {
  if (!bytes) return fail(PDA_ERR_INVALID_ARGUMENT, "null pointer");
  const int width = width_for(head_dim);
  if (width == 0)
    return fail(PDA_ERR_HEAD_DIM, "head_dim %d: trees are served at multiples of 8 up to 256",
                head_dim);
  *bytes = tree_workspace(width);
  return ok();
}

#define PDA_TREE_ARGS                                                                          \
  const int32_t *tables, const int32_t *lengths, const int32_t *starts, const uint64_t *masks, \
      void *out, int32_t tokens, int32_t batch, int32_t q_heads, int32_t kv_heads,             \
      int32_t head_dim, int32_t page_size, int32_t table_stride, int64_t arena_rows,           \
      int32_t layout, float scale, int32_t window, float softcap, void *workspace,             \
      size_t workspace_bytes, void *stream
#define PDA_TREE_PASS                                                                          \
  tables, lengths, starts, masks, out, tokens, batch, q_heads, kv_heads, head_dim, page_size,  \
      table_stride, arena_rows, layout, scale, window, softcap, workspace, workspace_bytes, stream

int pda_tree_attention(const void* queries, const void* keys, const void* values, PDA_TREE_ARGS) {
  return tree_attention(queries, keys, values, nullptr, nullptr, false, false, PDA_TREE_PASS);
}
int pda_tree_attention_bf16(const void* queries, const void* keys, const void* values,
                            PDA_TREE_ARGS) {
  return tree_attention(queries, keys, values, nullptr, nullptr, false, true, PDA_TREE_PASS);
}
int pda_tree_attention_q8(const void* queries, const void* keys, const void* values,
                          const void* key_scales, const void* value_scales, PDA_TREE_ARGS) {
  return tree_attention(queries, keys, values, key_scales, value_scales, true, false,
                        PDA_TREE_PASS);
}
int pda_tree_attention_q8_bf16(const void* queries, const void* keys, const void* values,
                               const void* key_scales, const void* value_scales, PDA_TREE_ARGS) {
  return tree_attention(queries, keys, values, key_scales, value_scales, true, true,
                        PDA_TREE_PASS);
}

int pda_commit_drafts(void* const* stores, int32_t layers, int32_t stores_per_layer,
                      int32_t width, const int32_t* tables, const int32_t* lengths,
                      const int32_t* starts, const int32_t* parents, const void* drafted,
                      const void* targets, int32_t token_bytes, int32_t* out_lengths,
                      int32_t* accepted, int32_t* path, int64_t* following, int32_t tokens,
                      int32_t batch, int32_t kv_heads, int32_t page_size, int32_t table_stride,
                      int64_t arena_rows, int32_t layout, void* stream) {
  if (layers <= 0 || (stores_per_layer != 2 && stores_per_layer != 4) || width <= 0 ||
      tokens < 0 || batch < 0 || kv_heads <= 0 || page_size <= 0 || table_stride <= 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "layers=%d stores_per_layer=%d width=%d tokens=%d batch=%d kv_heads=%d "
                "page_size=%d table_stride=%d",
                layers, stores_per_layer, width, tokens, batch, kv_heads, page_size, table_stride);
  if (token_bytes != 4 && token_bytes != 8)
    return fail(PDA_ERR_INVALID_ARGUMENT, "tokens have 4 or 8 bytes, got %d", token_bytes);
  if (layout != PDA_LAYOUT_ROWS && layout != PDA_LAYOUT_PAGES)
    return fail(PDA_ERR_INVALID_ARGUMENT, "unknown K/V layout %d", layout);
  if (arena_rows < page_size)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld holds no whole page",
                (long long)arena_rows);
  if (batch == 0) return ok();
  if (batch >= 1 << 18)
    return fail(PDA_ERR_TOO_LONG, "%d sequences exceed one launch", batch);
  if (!stores || !tables || !lengths || !starts || !out_lengths || !accepted || !path ||
      !following || (tokens > 0 && (!parents || !drafted || !targets)))
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (out_lengths == lengths)
    return fail(PDA_ERR_INVALID_ARGUMENT, "out_lengths must not be lengths: others still read them");
  if (((uintptr_t)tables | (uintptr_t)lengths | (uintptr_t)starts | (uintptr_t)parents |
       (uintptr_t)out_lengths | (uintptr_t)accepted | (uintptr_t)path) & 3)
    return fail(PDA_ERR_ALIGNMENT, "int32 buffers must be 4-byte aligned");
  if ((((uintptr_t)drafted | (uintptr_t)targets) & (token_bytes - 1)) || ((uintptr_t)following & 7))
    return fail(PDA_ERR_ALIGNMENT, "tokens must be aligned to their size");
  // (The workgroups of other stores read the inputs while one writes the results.)
  const Span in[] = {{"tables", tables, 4 * (int64_t)batch * table_stride},
                     {"lengths", lengths, 4 * (int64_t)batch},
                     {"starts", starts, 4 * ((int64_t)batch + 1)},
                     {"parents", parents, 4 * (int64_t)tokens},
                     {"drafted", drafted, (int64_t)token_bytes * tokens},
                     {"targets", targets, (int64_t)token_bytes * tokens}};
  const Span results[] = {{"out_lengths", out_lengths, 4 * (int64_t)batch},
                          {"accepted", accepted, 4 * (int64_t)batch},
                          {"path", path, 4 * (int64_t)kNodes * batch},
                          {"following", following, 8 * (int64_t)batch}};
  for (const Span& r : results) {
    for (const Span& x : in)
      if (overlap(r, x)) return fail(PDA_ERR_INVALID_ARGUMENT, "%s overlaps %s", r.name, x.name);
    for (const Span& x : results)
      if (&x != &r && overlap(r, x))
        return fail(PDA_ERR_INVALID_ARGUMENT, "%s overlaps %s", r.name, x.name);
  }
  const int64_t count = (int64_t)layers * stores_per_layer;
  for (int64_t i = 0; i < count; ++i)
    if (!stores[i]) return fail(PDA_ERR_INVALID_ARGUMENT, "null arena pointer");
  for (int32_t l0 = 0; l0 < layers; l0 += kCommitLayers) {
    const int n = std::min(kCommitLayers, layers - l0) * stores_per_layer;
    CommitParams prm{tables,   lengths, starts, parents,    drafted, targets, out_lengths,
                     accepted, path,    following, arena_rows / page_size, token_bytes == 8,
                     tokens,   batch,   table_stride, page_size, kv_heads, layout, width,
                     stores_per_layer, {}};
    for (int i = 0; i < n; ++i) prm.store[i] = stores[(int64_t)l0 * stores_per_layer + i];
    void* args[] = {&prm};
    const hipError_t err =
        hipLaunchKernel(reinterpret_cast<const void*>(commit_drafts_kernel), dim3(batch, n),
                        dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
    if (err != hipSuccess)
      return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  }
  return ok();
}

}  // extern "C"
