// Attention for trees of drafted tokens over the paged cache, and the step that
// keeps the accepted ones, for MI355X (gfx950), C-ABI in pda.h
// (pda_tree_attention, pda_commit_drafts). No counterpart in the reference, which
// decodes one token a sequence and step.
//
// Node i of a sequence's tree lies behind the l rows that the sequence holds, in
// row l + i, and attends to the held rows and to the nodes whose bits its mask has
// (itself and its ancestors): flops 4 D a (query head, node, visible key); the
// rows of a kv head are read once for up to 128 (node, query head) pairs of it.
//
// Rows of queries. A unit is (sequence, kv head, 128 of its node and head pairs);
// its keys come in tiles of 64. The tiles of all units form one stream that is cut
// into equal ranges, one a workgroup, whatever the lengths: a unit inside one range
// is written at once, the pieces of one that is cut are joined by a second kernel.
// The cuts depend on the lengths alone, so repeated calls give the same bits.

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

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kRows = 128;   // of a unit
constexpr int kNodes = 64;   // of a tree
constexpr int kCus = 256;
constexpr int groups_for(int width) { return width <= 128 ? 2 * kCus : kCus; }

struct TreeParams {
  const f16* q;          // [tokens, hq, dim]
  const void* k;         // arena: 16-bit, or int8 with scales
  const void* v;
  const f16* kscale;
  const f16* vscale;
  const int32_t* tables;   // [batch, stride]
  const int32_t* lengths;  // [batch] rows held before the tree
  const int32_t* starts;   // [batch + 1]
  const uint64_t* masks;   // [tokens]
  f16* out;                // [tokens, hq, dim]
  int64_t* seq_tiles;      // [batch + 1] first tile of each sequence in the stream,
  int32_t* seq_units;      // [batch + 1]   and its first unit
  float* part_o;           // [2 groups, 4 waves, D / 8, 64 lanes, 4]
  float2* part_ml;         // [2 groups, 128]
  int64_t arena_pages;
  int64_t page_elems, scale_page;  // elements between pages,
  int32_t head_elems, scale_head;  //   kv heads of a page,
  int32_t row_elems, scale_row;    //   rows of a page and head
  int32_t stride;
  int32_t page_size;
  int32_t tokens;
  int32_t batch;
  int32_t groups;  // workgroups that take ranges
  int32_t hq;
  int32_t hkv;
  int32_t dim;
  int32_t window;
  Shape shape;
};

// A sequence's tree: its tokens [first, first + n), the rows before it, the tiles
// [t0, t0 + nt) of its keys and its units a kv head.
struct Seq {
  int first, n, held, t0, nt, blocks;
};
__device__ __forceinline__ Seq seq_of(const TreeParams& p, int b) {
  Seq s;
  s.first = max(0, min(p.starts[b], p.tokens));
  s.n = max(s.first, min(p.starts[b + 1], p.tokens)) - s.first;
  const int64_t room = min((int64_t)p.stride * p.page_size, (int64_t)INT32_MAX - 2 * kNodes);
  s.held = (int)max((int64_t)0, min((int64_t)p.lengths[b], room));
  // (The first row that any node sees: a node is at least at position `held`.)
  s.t0 = p.window > 0 ? max(0, s.held - p.window + 1) / kKeys : 0;
  const int end = s.held + min(s.n, kNodes);
  s.nt = s.n > 0 ? (end + kKeys - 1) / kKeys - s.t0 : 0;
  s.blocks = (int)(((int64_t)s.n * (p.hq / p.hkv) + kRows - 1) / kRows);
  return s;
}
__device__ __forceinline__ Seq uniform_seq(const Seq& s) {
  return {uniform(s.first), uniform(s.n),  uniform(s.held),
          uniform(s.t0),    uniform(s.nt), uniform(s.blocks)};
}
__device__ __forceinline__ int64_t tiles_of(const TreeParams& p, const Seq& s) {
  return (int64_t)s.nt * s.blocks * p.hkv;
}

// Workgroups that take ranges of a stream of `tiles`, and the first tile of one's.
__device__ __forceinline__ int64_t ranges(const TreeParams& p, int64_t tiles) {
  return min(tiles, (int64_t)p.groups);
}
__device__ __forceinline__ int64_t range_begin(int64_t tiles, int64_t n, int64_t g) {
  return tiles * g / n;
}

// Prefix sums over the sequences: the stream's length, and sequence `seq` that
// holds tile x, which is its `rest`-th. Workgroup 0 leaves the sums for the join.
// (x is past the stream's end: seq is batch.)
template <class F>
__device__ __forceinline__ int64_t locate(const TreeParams& p, F pick, int& seq, int64_t& rest) {
  __shared__ int64_t s_tiles[kThreads / 64];
  __shared__ int32_t s_units[kThreads / 64];
  __shared__ int s_seq;
  __shared__ int64_t s_rest;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  int64_t mine = 0;
  int32_t units = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = seq_of(p, b);
    mine += tiles_of(p, s);
    units += s.blocks * p.hkv;
  }
  int64_t upto = mine;
  int32_t upto_units = units;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(upto, d);
    const int32_t z = __shfl_up(upto_units, d);
    if (lane >= d) upto += y, upto_units += z;
  }
  if (lane == 63) s_tiles[w] = upto, s_units[w] = upto_units;
  if (tid == 0) s_seq = p.batch;
  __syncthreads();
  int64_t before = upto - mine, all = 0;
  int32_t before_units = upto_units - units, all_units = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < w) before += s_tiles[i], before_units += s_units[i];
    all += s_tiles[i];
    all_units += s_units[i];
  }
  const int64_t x = pick(uniform64(all));
  if (blockIdx.x == 0) {
    int64_t t = before;
    int32_t u = before_units;
    for (int b = b0; b < b1; ++b) {
      const Seq s = seq_of(p, b);
      p.seq_tiles[b] = t;
      p.seq_units[b] = u;
      t += tiles_of(p, s);
      u += s.blocks * p.hkv;
    }
    if (tid == 0) {
      p.seq_tiles[p.batch] = all;
      p.seq_units[p.batch] = all_units;
    }
  }
  if (x >= before && x < before + mine) {
    int64_t left = x - before;
    for (int b = b0; b < b1; ++b) {
      const int64_t n = tiles_of(p, seq_of(p, b));
      if (left < n) {
        s_seq = b;
        s_rest = left;
        break;
      }
      left -= n;
    }
  }
  __syncthreads();
  seq = uniform(s_seq);
  rest = uniform64(s_rest);
  return uniform64(all);
}

// Eight int8 values as elements of the queries' type, exactly.
template <bool BF>
__device__ __forceinline__ f16x8 from_bytes(const u32x2& y) {
  f16x8 x;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = round16<BF>((float)(int)__builtin_amdgcn_sbfe((int)y[i / 4], 8 * (i % 4), 8));
  return x;
}
// Times the row's scale, rounded once.
template <bool BF>
__device__ __forceinline__ f16x8 from_bytes(const u32x2& y, float scale) {
  f16x8 x;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = round16<BF>((float)(int)__builtin_amdgcn_sbfe((int)y[i / 4], 8 * (i % 4), 8) * scale);
  return x;
}

template <int D, bool BF, bool Q8>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void tree_attention_kernel(
    const TreeParams p) {
  constexpr int kPlanes = D / 32;
  constexpr int kTileHalves = kPlanes * kPlane;
  __shared__ __align__(1024) f16 s_k[2][kTileHalves];
  __shared__ __align__(1024) f16 s_v[2][kTileHalves];
  __shared__ __align__(16) float s_scale[2][kKeys];  // the keys' scales
  __shared__ uint16_t s_ok[2][4], s_bad[2][4];  // usable keys; values not finite

  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int G = p.hq / p.hkv;

  // Rows behind the last sequence: zeros.
  {
    const int real = p.batch > 0 ? max(0, min(p.starts[p.batch], p.tokens)) : 0;
    const int64_t from = (int64_t)real * p.hq * p.dim / 8, to = (int64_t)p.tokens * p.hq * p.dim / 8;
    for (int64_t i = from + blockIdx.x * kThreads + tid; i < to; i += (int64_t)gridDim.x * kThreads)
      reinterpret_cast<f16x8*>(p.out)[i] = f16x8{};
  }
  int seq;
  int64_t rest, begin = 0, end = 0;
  locate(p, [&](int64_t all) -> int64_t {
    const int64_t n = ranges(p, all);
    if (blockIdx.x >= n) return all;
    begin = range_begin(all, n, blockIdx.x);
    end = range_begin(all, n, blockIdx.x + 1);
    return begin;
  }, seq, rest);
  if (begin >= end) return;

  if (p.dim != D) {  // what no copy writes
    f16* flat_k = &s_k[0][0];
    f16* flat_v = &s_v[0][0];
    for (int i = 8 * tid; i < 2 * kTileHalves; i += 8 * kThreads) {
      *reinterpret_cast<f16x8*>(flat_k + i) = f16x8{};
      *reinterpret_cast<f16x8*>(flat_v + i) = f16x8{};
    }
    __syncthreads();
  }

  Rows<D, BF> r;
  r.init(p.shape);
  const bool special = p.shape.cap_out > 0.0f || !(p.shape.scale_log2 > 0.0f);
  const uint32_t pages = (uint32_t)min(p.arena_pages, (int64_t)INT32_MAX);

  // Copies: thread tid moves key tid / 4 of a tile, one 8-element chunk a plane.
  const int gk = tid >> 2;
  const int kchunk = 8 * ((lane & 3) ^ ((lane >> 4) & 3)), vchunk = 8 * (lane & 3);
  const uint32_t k_dst = uniform(lds_address(&s_k[0][0]) + 1024 * w);
  const uint32_t v_dst = uniform(lds_address(&s_v[0][0]) + 1024 * w);

  int64_t left = end - begin;
  bool first_piece = true;
  while (left > 0) {
    const Seq s = uniform_seq(seq_of(p, seq));
    const int unit = uniform((int)(rest / s.nt));
    const int ta = s.t0 + (int)(rest - (int64_t)unit * s.nt);
    const int tb = s.t0 + (int)min((int64_t)s.nt, rest - (int64_t)unit * s.nt + left);
    const int kvh = uniform(unit / s.blocks), block = unit - kvh * s.blocks;
    const int32_t* table = p.tables + (int64_t)seq * p.stride;

    // This lane's row: a node and a query head. (Rows past the last see what that
    // one sees, and are not stored.)
    const int all_rows = s.n * G;
    const int row = kRows * block + 32 * w + (lane & 31);
    const bool wave_live = kRows * block + 32 * w < all_rows;
    const bool live = row < all_rows;
    const int at = min(row, all_rows - 1);
    const int node = at / G;
    const int64_t q_row = (int64_t)(s.first + node) * p.hq + kvh * G + at % G;
    r.clear();
    r.load(p.q + q_row * p.dim, p.dim, true);
    uint64_t mask = p.masks[s.first + node];
    const int depth = max(0, (int)__popcll(mask) - 1);
    int lo = 0;  // first held row the node sees
    if (p.window > 0) {
      lo = max(0, s.held + depth - p.window + 1);
      while ((int)__popcll(mask) > p.window) mask &= mask - 1;
    }
    const int last = s.held + min(s.n, kNodes) - 1;

    int page = 0;
    bool in = false;
    uint32_t slot = 0;
    auto lookup = [&](int t) {
      const uint32_t kp = (uint32_t)t * kKeys + gk;
      const uint32_t pi = kp / (uint32_t)p.page_size;
      slot = kp - pi * (uint32_t)p.page_size;
      in = kp <= (uint32_t)last && pi < (uint32_t)p.stride;
      page = table[min(pi, (uint32_t)p.stride - 1)];
    };
    u32x2 raw_k[kPlanes], raw_v[kPlanes];
    f16 raw_ks = (f16)0.0f, raw_vs = (f16)0.0f;
    bool mine_ok = false;  // this thread's key of the tile under way
    auto copies = [&](int t) {
      const uint32_t buf = (t - ta) & 1;
      mine_ok = in && (uint32_t)page < pages;
      const int64_t from = mine_ok ? page : 0;
      const int64_t src = from * p.page_elems + (int64_t)slot * p.row_elems + (int64_t)kvh * p.head_elems;
      if constexpr (Q8) {
        const int64_t sc = from * p.scale_page + (int64_t)slot * p.scale_row + (int64_t)kvh * p.scale_head;
        raw_ks = p.kscale[sc];
        raw_vs = p.vscale[sc];
#pragma unroll
        for (int i = 0; i < kPlanes; ++i) {
          if (D == p.dim || 32 * i + kchunk < p.dim)
            raw_k[i] = *reinterpret_cast<const u32x2*>(static_cast<const int8_t*>(p.k) + src + kchunk + 32 * i);
          if (D == p.dim || 32 * i + vchunk < p.dim)
            raw_v[i] = *reinterpret_cast<const u32x2*>(static_cast<const int8_t*>(p.v) + src + vchunk + 32 * i);
        }
      } else {
        const f16* src_k = static_cast<const f16*>(p.k) + src + kchunk;
        const f16* src_v = static_cast<const f16*>(p.v) + src + vchunk;
        const uint32_t off = buf * (2 * kTileHalves);
#pragma unroll
        for (int i = 0; i < kPlanes; ++i) {
          if (D == p.dim || 32 * i + kchunk < p.dim)
            copy_to_lds(src_k + 32 * i, k_dst + off + 2 * kPlane * i);
          if (D == p.dim || 32 * i + vchunk < p.dim)
            copy_to_lds(src_v + 32 * i, v_dst + off + 2 * kPlane * i);
        }
      }
    };
    // Tiles with keys that not every row sees.
    auto edge = [&](int t) {
      return t * kKeys + kKeys > s.held ||
             (p.window > 0 && t * kKeys < s.held + kNodes - p.window);
    };
    // What was copied becomes readable: rows that are not usable as zeros (their
    // weight is 0, but 0 times what an arena holds there need not be); on an edge,
    // values that are not finite as zeros too, their keys remembered.
    auto arrive = [&](int t) {
      const int buf = (t - ta) & 1;
      wait_vmem<0>();
      const bool check = edge(t);
      bool bad = false;
      f16* dst_k = &s_k[buf][32 * gk + 8 * (lane & 3)];
      f16* dst_v = &s_v[buf][32 * gk + 8 * (lane & 3)];
      if constexpr (Q8) {
        if ((lane & 3) == 0) s_scale[buf][gk] = (float)raw_ks;
        const float vs = (float)raw_vs;
#pragma unroll
        for (int i = 0; i < kPlanes; ++i) {
          if (D == p.dim || 32 * i + kchunk < p.dim)
            *reinterpret_cast<f16x8*>(dst_k + kPlane * i) = from_bytes<BF>(raw_k[i]);
          if (D == p.dim || 32 * i + vchunk < p.dim) {
            f16x8 x = from_bytes<BF>(raw_v[i], vs);
            if (!mine_ok) x = f16x8{};
            if (check && not_finite<BF>(x)) {
              bad = true;
              x = finite_only<BF>(x);
            }
            *reinterpret_cast<f16x8*>(dst_v + kPlane * i) = x;
          }
        }
      } else if (!mine_ok) {
#pragma unroll
        for (int i = 0; i < kPlanes; ++i)
          *reinterpret_cast<f16x8*>(dst_v + kPlane * i) = f16x8{};
      } else if (check) {
#pragma unroll
        for (int i = 0; i < kPlanes; ++i) {
          const f16x8 x = *reinterpret_cast<const f16x8*>(dst_v + kPlane * i);
          if (not_finite<BF>(x)) {
            bad = true;
            *reinterpret_cast<f16x8*>(dst_v + kPlane * i) = finite_only<BF>(x);
          }
        }
      }
      const uint32_t usable = keys_of(__ballot(mine_ok)), not_fin = keys_of(__ballot(bad));
      if (lane == 0) {
        s_ok[buf][w] = (uint16_t)usable;
        s_bad[buf][w] = (uint16_t)not_fin;
      }
    };

    lookup(ta);
    copies(ta);
    if (ta + 1 < tb) lookup(ta + 1);
    arrive(ta);
    __syncthreads();
    for (int t = ta; t < tb; ++t) {
      if (t + 1 < tb) copies(t + 1);
      if (t + 2 < tb) lookup(t + 2);
      const int buf = (t - ta) & 1;
      if (wave_live) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k0 = t * kKeys + 32 * j;
          f32x16 x;
          f16x8 weights[2];
          r.scores(x, s_k[buf] + 1024 * j);
          if constexpr (Q8) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float4 ks = *reinterpret_cast<const float4*>(&s_scale[buf][32 * j + 8 * g + 4 * r.hh]);
              x[4 * g] *= ks.x;
              x[4 * g + 1] *= ks.y;
              x[4 * g + 2] *= ks.z;
              x[4 * g + 3] *= ks.w;
            }
          }
          if (special) r.shape(x, p.shape);
          const uint32_t usable = uniform((int)(s_ok[buf][2 * j] | s_ok[buf][2 * j + 1] << 16));
          uint32_t see = usable;
          if (usable != 0xFFFFFFFFu || edge(t)) {
            const int d = s.held - k0;  // the tree's first row in the block
            uint32_t nodes = 0;
            if (d >= 0 && d < 32) nodes = (uint32_t)(mask << d);
            if (d < 0 && d > -64) nodes = (uint32_t)(mask >> -d);
            see &= (below(d) & ~below(lo - k0)) | nodes;
            r.mask(x, see);
          }
          r.weigh(x, weights);
          r.accumulate(weights, s_v[buf] + 1024 * j);
          if (edge(t)) {
            const uint32_t bad = uniform((int)(s_bad[buf][2 * j] | s_bad[buf][2 * j + 1] << 16));
            if (bad)
              r.add_not_finite(weights, bad, see, p.dim, [&](int k, int d) {
                const uint32_t pi = (uint32_t)(k0 + k) / (uint32_t)p.page_size;
                const uint32_t sl = (uint32_t)(k0 + k) - pi * (uint32_t)p.page_size;
                const int64_t from = table[pi];  // (the key is usable)
                const int64_t src = from * p.page_elems + (int64_t)sl * p.row_elems +
                                    (int64_t)kvh * p.head_elems + d;
                if constexpr (Q8) {
                  const float vs = (float)p.vscale[from * p.scale_page + (int64_t)sl * p.scale_row +
                                                   (int64_t)kvh * p.scale_head];
                  const int8_t* y = static_cast<const int8_t*>(p.v) + src;
                  return make_float4(y[0] * vs, y[1] * vs, y[2] * vs, y[3] * vs);
                } else {
                  return widen4<BF>(static_cast<const f16*>(p.v) + src);
                }
              });
          }
        }
      }
      if (t + 1 < tb) arrive(t + 1);
      __syncthreads();
    }

    if (tb - ta == s.nt) {
      const float inv = r.inverse();
      if (live) r.store(p.out + q_row * p.dim, p.dim, inv);
    } else if (wave_live) {
      // A piece of a unit that is cut, as it is.
      const int64_t piece = 2 * (int64_t)blockIdx.x + (first_piece ? 0 : 1);
      const float sum = r.l + __shfl_xor(r.l, 32);
      if (lane < 32) p.part_ml[piece * kRows + 32 * w + lane] = make_float2(r.m, sum);
      float4* dst = reinterpret_cast<float4*>(p.part_o) + (piece * 4 + w) * (D / 8 * 64) + lane;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        dst[64 * i] = make_float4(r.o[i / 4][4 * (i % 4)], r.o[i / 4][4 * (i % 4) + 1],
                                  r.o[i / 4][4 * (i % 4) + 2], r.o[i / 4][4 * (i % 4) + 3]);
    }
    left -= tb - ta;
    rest += tb - ta;
    if (rest >= tiles_of(p, s)) {  // the next sequence that has a tree
      rest = 0;
      ++seq;
      while (left > 0 && uniform(seq_of(p, seq).nt) == 0) ++seq;
    }
    first_piece = false;
  }
}

// Joins the pieces of a cut unit: with M the largest of their maxima, the outputs
// are sum 2^(m - M) o / sum 2^(m - M) l. A wave takes 32 rows and a few of their
// dims, the lanes as in the kernel that left them.
template <int D, bool BF>
__global__ __launch_bounds__(kThreads) void tree_join_kernel(const TreeParams p) {
  constexpr int kShare = D / 8 / 4;  // groups of 8 dims a wave takes: a quarter
  const int unit = blockIdx.x >> 2;
  const int lane = threadIdx.x & 63, w = blockIdx.x & 3, part = threadIdx.x >> 6;
  if (unit >= p.seq_units[p.batch]) return;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.seq_units[mid] <= unit)
      lo = mid;
    else
      hi = mid - 1;
  }
  const Seq s = seq_of(p, lo);
  const int64_t all = p.seq_tiles[p.batch];
  const int64_t n = ranges(p, all);
  const int64_t begin = p.seq_tiles[lo] + (int64_t)(unit - p.seq_units[lo]) * s.nt;
  const int64_t end = begin + s.nt;
  const int64_t g0 = ((begin + 1) * n - 1) / all, g1 = (end * n - 1) / all;
  if (g0 == g1) return;  // written where it was computed
  const int G = p.hq / p.hkv;
  const int kvh = (unit - p.seq_units[lo]) / s.blocks, block = (unit - p.seq_units[lo]) % s.blocks;
  const int row = kRows * block + 32 * w + (lane & 31);
  if (kRows * block + 32 * w >= s.n * G) return;
  auto piece = [&](int64_t g) {
    return 2 * g + (g == g0 && begin > range_begin(all, n, g) ? 1 : 0);
  };
  float top = -INFINITY;
  for (int64_t g = g0; g <= g1; ++g)
    top = fmaxf(top, p.part_ml[piece(g) * kRows + 32 * w + (lane & 31)].x);
  float4 acc[kShare];
#pragma unroll
  for (int i = 0; i < kShare; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
  for (int64_t g = g0; g <= g1; ++g) {
    const float2 ml = p.part_ml[piece(g) * kRows + 32 * w + (lane & 31)];
    // (A piece of which the row sees nothing holds zeros. One of NaN is not empty.)
    const float f = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
    const float4* src = reinterpret_cast<const float4*>(p.part_o) +
                        (piece(g) * 4 + w) * (D / 8 * 64) + part * kShare * 64 + lane;
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
      const float4 x = src[64 * i];
      acc[i].x = fmaf(x.x, f, acc[i].x);
      acc[i].y = fmaf(x.y, f, acc[i].y);
      acc[i].z = fmaf(x.z, f, acc[i].z);
      acc[i].w = fmaf(x.w, f, acc[i].w);
    }
    sum = fmaf(ml.y, f, sum);
  }
  if (row >= s.n * G) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  f16* dst = p.out + ((int64_t)(s.first + row / G) * p.hq + kvh * G + row % G) * p.dim;
#pragma unroll
  for (int i = 0; i < kShare; ++i) {
    const int d = 8 * (part * kShare + i) + 4 * (lane >> 5);
    const f16x4 y = {round16<BF>(acc[i].x * inv), round16<BF>(acc[i].y * inv),
                     round16<BF>(acc[i].z * inv), round16<BF>(acc[i].w * inv)};
    if (d < p.dim) *reinterpret_cast<f16x4*>(dst + d) = y;
  }
}

template <bool BF, bool Q8>
const void* tree_kernel_for(int width) {
  return width == 64    ? reinterpret_cast<const void*>(tree_attention_kernel<64, BF, Q8>)
         : width == 96  ? reinterpret_cast<const void*>(tree_attention_kernel<96, BF, Q8>)
         : width == 128 ? reinterpret_cast<const void*>(tree_attention_kernel<128, BF, Q8>)
                        : reinterpret_cast<const void*>(tree_attention_kernel<256, BF, Q8>);
}
template <bool BF>
const void* tree_join_for(int width) {
  return width == 64    ? reinterpret_cast<const void*>(tree_join_kernel<64, BF>)
         : width == 96  ? reinterpret_cast<const void*>(tree_join_kernel<96, BF>)
         : width == 128 ? reinterpret_cast<const void*>(tree_join_kernel<128, BF>)
                        : reinterpret_cast<const void*>(tree_join_kernel<256, BF>);
}

constexpr size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

size_t tree_workspace(int64_t batch, int width) {
  const size_t pieces = 2 * (size_t)groups_for(width);
  return aligned((batch + 1) * 8) + aligned((batch + 1) * 4) + pieces * kRows * 8 +
         pieces * kRows * width * 4;
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
  // Rows of a sequence's tree, and all units, are counted in 32 bits.
  const int G = q_heads / kv_heads;
  const int64_t units = ((int64_t)tokens * G + (int64_t)(kRows - 1) * batch) / kRows * kv_heads;
  if ((int64_t)tokens * G > INT32_MAX || units >= (int64_t)1 << 22)
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
  const size_t need = tree_workspace(batch, width);
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
  const size_t pieces = 2 * (size_t)groups_for(width);
  char* ws = static_cast<char*>(workspace);
  prm.part_o = reinterpret_cast<float*>(ws);
  ws += pieces * kRows * width * 4;
  prm.part_ml = reinterpret_cast<float2*>(ws);
  ws += pieces * kRows * 8;
  prm.seq_tiles = reinterpret_cast<int64_t*>(ws);
  ws += aligned(((size_t)batch + 1) * 8);
  prm.seq_units = reinterpret_cast<int32_t*>(ws);
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
  prm.groups = groups_for(width);
  prm.hq = q_heads;
  prm.hkv = kv_heads;
  prm.dim = head_dim;
  prm.window = window;
  prm.shape = shape_of(scale, softcap);
  void* args[] = {&prm};
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  const void* fn = q8 ? (bf16_elems ? tree_kernel_for<true, true>(width)
                                    : tree_kernel_for<false, true>(width))
                      : (bf16_elems ? tree_kernel_for<true, false>(width)
                                    : tree_kernel_for<false, false>(width));
  hipError_t err = hipLaunchKernel(fn, dim3(prm.groups), dim3(kThreads), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  if (batch == 0) return ok();
  err = hipLaunchKernel(bf16_elems ? tree_join_for<true>(width) : tree_join_for<false>(width),
                        dim3((unsigned)(4 * units)), dim3(kThreads), args, 0, hs);
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
// and what a wave moves at once it reads before it writes.
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

int pda_tree_workspace_bytes(int32_t batch, int32_t head_dim, size_t* bytes) {
  if (batch < 0 || !bytes) return fail(PDA_ERR_INVALID_ARGUMENT, "batch=%d", batch);
  const int width = width_for(head_dim);
  if (width == 0)
    return fail(PDA_ERR_HEAD_DIM, "head_dim %d: trees are served at multiples of 8 up to 256",
                head_dim);
  *bytes = tree_workspace(batch, width);
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
