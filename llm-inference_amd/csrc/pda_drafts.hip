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
#include "pda_rows.h"

namespace {

using namespace pda_rows;
using pda_internal::fail;
using pda_internal::ok;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;  // of a workgroup of four waves, and of the join's
constexpr int kNodes = 64;     // of a tree
constexpr int kCus = 256;
// Workgroups: as many as the GPU holds at once.
constexpr int groups_for(int width, int waves) { return width <= 128 && waves == 4 ? 2 * kCus : kCus; }
// Tiles that a range has at least.
constexpr int kLeastTiles = 2;

// What the join has to know of a unit that ends in a workgroup's range and began in
// an earlier one.
struct Cut {
  int32_t rows;     // of the unit (0: no such unit)
  int32_t first;    // its first (token, query head) row, without the kv head's
  int32_t token;    // the sequence's first token
  int32_t kvh;
  int32_t piece;    // its first piece
  int32_t group;    // the workgroup after that piece's
  int32_t pad[2];
};

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
  float* part_o;           // [2 groups, waves, D / 8, 64 lanes, 4]
  float2* part_ml;         // [2 groups, waves, 32]
  Cut* cuts;               // [groups]
  int64_t arena_pages;
  int64_t page_elems, scale_page;  // elements between pages,
  int32_t head_elems, scale_head;  //   kv heads of a page,
  int32_t row_elems, scale_row;    //   rows of a page and head
  int32_t stride;
  int32_t page_size;
  int32_t tokens;
  int32_t batch;
  int32_t groups;  // workgroups that take ranges
  int32_t rows;    // of a unit: 32 a wave
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
  s.blocks = (int)(((int64_t)s.n * (p.hq / p.hkv) + p.rows - 1) / p.rows);
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
  return min((tiles + kLeastTiles - 1) / kLeastTiles, (int64_t)p.groups);
}
__device__ __forceinline__ int64_t range_begin(int64_t tiles, int64_t n, int64_t g) {
  return tiles * g / n;
}

// The workgroup's range of the stream of all sequences' tiles, and the sequence that
// its first tile belongs to, of which it is the `rest`-th. Every wave finds them by
// itself, a lane for a few sequences.
struct Range {
  int64_t all, n, begin, end, rest;
  int seq;
};
__device__ __forceinline__ Range range_of(const TreeParams& p) {
  const int lane = threadIdx.x & 63;
  const int per = (p.batch + 63) / 64;
  const int b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of(p, seq_of(p, b));
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
  }
  Range r;
  r.all = uniform64(__shfl(upto, 63));
  r.n = ranges(p, r.all);
  if (blockIdx.x >= r.n) {
    r.begin = r.end = r.rest = 0;
    r.seq = 0;
    return r;
  }
  r.begin = range_begin(r.all, r.n, blockIdx.x);
  r.end = range_begin(r.all, r.n, blockIdx.x + 1);
  const bool here = r.begin >= upto - mine && r.begin < upto;
  int64_t left = r.begin - (upto - mine);
  int seq = b0;
  if (here)
    for (; seq < b1 - 1; ++seq) {
      const int64_t n = tiles_of(p, seq_of(p, seq));
      if (left < n) break;
      left -= n;
    }
  const int owner = __builtin_ctzll(__ballot(here));
  r.seq = uniform(__shfl(seq, owner));
  r.rest = uniform64(__shfl(left, owner));
  return r;
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

// A unit's keys and values on their way from the pages through LDS, and their masks.
// W waves: with eight the first four copy V and the others K.
// EXACT: the head dim is D.
template <int D, bool BF, bool Q8, int W, bool EXACT>
struct TreeTiles {
  static constexpr int kPlanes = D / 32;
  static constexpr int kHalves = kPlanes * kPlane;  // of a tile
  static constexpr int kCopies = W == 4 ? 2 * kPlanes : kPlanes;

  const TreeParams& p;
  f16* s_k;          // [2][kHalves]
  f16* s_v;
  float* s_scale;    // [4][64] the keys' scales, by tile
  uint16_t* s_ok;    // [4][4] usable keys, by tile and wave
  int* s_left;       // whether values that are not finite were taken as zeros
  bool special;
  int lane, w, gk, kchunk, vchunk;
  uint32_t k_dst, v_dst, pages;

  // The piece's.
  const int32_t* table;
  int kvh, held, last;
  uint64_t mask;  // nodes that the lane's row sees
  int lo;         // and the first row held
  // This thread's key of the tiles whose V and K are copied next, and the looked-up
  // page of the tile after them.
  int64_t at_v, at_k, scale_v, scale_k;
  bool ok_v, ok_k, in;
  int page;
  uint32_t slot;
  uint64_t usable, usable_before;  // keys of the tile that is scored, and of the last
  u32x2 raw_k[Q8 ? kPlanes : 1], raw_v[Q8 ? kPlanes : 1];
  f16 raw_ks, raw_vs;

  __device__ __forceinline__ bool moves_v() const { return W == 4 || w < 4; }
  __device__ __forceinline__ bool moves_k() const { return W == 4 || w >= 4; }

  __device__ __forceinline__ void init() {
    const int tid = threadIdx.x;
    lane = tid & 63;
    w = uniform(tid >> 6);
    // Copies: a thread moves key (tid / 4) % 64 of a tile, one 8-element chunk a plane.
    gk = (tid >> 2) & 63;
    kchunk = 8 * ((lane & 3) ^ ((lane >> 4) & 3));
    vchunk = 8 * (lane & 3);
    k_dst = uniform(lds_address(s_k) + 1024 * (w & 3));
    v_dst = uniform(lds_address(s_v) + 1024 * (w & 3));
    pages = (uint32_t)min(p.arena_pages, (int64_t)INT32_MAX);
    special = p.shape.cap_out > 0.0f || !(p.shape.scale_log2 > 0.0f);
    if constexpr (!EXACT) {  // what no copy writes
      for (int i = 8 * tid; i < 2 * kHalves; i += 8 * 64 * W) {
        *reinterpret_cast<f16x8*>(s_k + i) = f16x8{};
        *reinterpret_cast<f16x8*>(s_v + i) = f16x8{};
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ const f16* keys(int t) const { return s_k + (t & 1) * kHalves; }
  __device__ __forceinline__ const f16* values(int t) const { return s_v + (t & 1) * kHalves; }

  __device__ __forceinline__ void lookup(int t) {
    const uint32_t kp = (uint32_t)t * kKeys + gk;
    const uint32_t pi = kp / (uint32_t)p.page_size;
    slot = kp - pi * (uint32_t)p.page_size;
    in = kp <= (uint32_t)last && pi < (uint32_t)p.stride;
    page = table[min(pi, (uint32_t)p.stride - 1)];
  }
  // The looked-up tile becomes the next K to copy, the one before it the next V.
  __device__ __forceinline__ void turn() {
    at_v = at_k;
    ok_v = ok_k;
    ok_k = in && (uint32_t)page < pages;
    const int64_t from = ok_k ? page : 0;
    at_k = from * p.page_elems + (int64_t)slot * p.row_elems + (int64_t)kvh * p.head_elems;
    if constexpr (Q8) {
      scale_v = scale_k;
      scale_k = from * p.scale_page + (int64_t)slot * p.scale_row + (int64_t)kvh * p.scale_head;
    }
  }
  __device__ __forceinline__ void copy_k(int t, int i) {
    if constexpr (Q8) {
      if (i == 0) raw_ks = p.kscale[scale_k];
    }
    if (!EXACT && 32 * i + kchunk >= p.dim) return;
    if constexpr (Q8) {
      raw_k[i] = *reinterpret_cast<const u32x2*>(static_cast<const int8_t*>(p.k) + at_k + kchunk + 32 * i);
    } else {
      copy_to_lds(static_cast<const f16*>(p.k) + at_k + kchunk + 32 * i,
                  k_dst + (t & 1) * (2 * kHalves) + 2 * kPlane * i);
    }
  }
  __device__ __forceinline__ void copy_v(int t, int i) {
    if (!EXACT && 32 * i + vchunk >= p.dim) return;
    if constexpr (Q8) {
      raw_v[i] = *reinterpret_cast<const u32x2*>(static_cast<const int8_t*>(p.v) + at_v + vchunk + 32 * i);
      if (i == 0) raw_vs = p.vscale[scale_v];
    } else {
      copy_to_lds(static_cast<const f16*>(p.v) + at_v + vchunk + 32 * i,
                  v_dst + (t & 1) * (2 * kHalves) + 2 * kPlane * i);
    }
  }
  template <int j>
  __device__ __forceinline__ void copy(int t) {
    if constexpr (W == 4) {
      if constexpr (j < kPlanes)
        copy_v(t, j);
      else
        copy_k(t + 1, j - kPlanes);
    } else {
      if (w < 4)
        copy_v(t, j);
      else
        copy_k(t + 1, j);
    }
  }
  // 8 bits: what was loaded goes to LDS, the keys as they are (their scales beside
  // them, for the scores), the values times their scale.
  __device__ __forceinline__ void put_k(int t) {
    if constexpr (Q8) {
      if (!moves_k()) return;
      f16* dst = s_k + (t & 1) * kHalves + 32 * gk + 8 * (lane & 3);
      if ((lane & 3) == 0) s_scale[kKeys * (t & 3) + gk] = (float)raw_ks;
#pragma unroll
      for (int i = 0; i < kPlanes; ++i)
        if (EXACT || 32 * i + kchunk < p.dim)
          *reinterpret_cast<f16x8*>(dst + kPlane * i) = from_bytes<BF>(raw_k[i]);
    }
  }

  // Tiles with keys that not every row sees.
  __device__ __forceinline__ bool edge(int t) const {
    return t * kKeys + kKeys > held || (p.window > 0 && t * kKeys < held + kNodes - p.window);
  }
  // V of tile t as it arrived: rows that are not usable become zeros (their weight is
  // 0, but 0 times what an arena holds there need not be); on an edge, values that are
  // not finite too.
  __device__ __forceinline__ void put_v(int t) {
    if (!moves_v()) return;
    const bool check = edge(t);
    f16* dst = s_v + (t & 1) * kHalves + 32 * gk + 8 * (lane & 3);
    if constexpr (Q8) {
      const float vs = (float)raw_vs;
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) {
        if (!EXACT && 32 * i + vchunk >= p.dim) continue;
        f16x8 x = from_bytes<BF>(raw_v[i], vs);
        if (!ok_v) x = f16x8{};
        if (check && not_finite<BF>(x)) {
          *s_left = 1;
          x = finite_only<BF>(x);
        }
        *reinterpret_cast<f16x8*>(dst + kPlane * i) = x;
      }
    } else if (!ok_v) {
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) *reinterpret_cast<f16x8*>(dst + kPlane * i) = f16x8{};
    } else if (check) {
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) {
        const f16x8 x = *reinterpret_cast<const f16x8*>(dst + kPlane * i);
        if (not_finite<BF>(x)) {
          *s_left = 1;
          *reinterpret_cast<f16x8*>(dst + kPlane * i) = finite_only<BF>(x);
        }
      }
    }
  }
  __device__ __forceinline__ void put_usable(int t) {
    if (!moves_k()) return;
    const uint32_t flags = keys_of(__ballot(ok_k));
    if (lane == 0) s_ok[4 * (t & 3) + (w & 3)] = (uint16_t)flags;
  }
  __device__ __forceinline__ void take_usable(int t) {
    usable_before = usable;
    usable = (uint64_t)uniform64((int64_t)*reinterpret_cast<const uint64_t*>(s_ok + 4 * (t & 3)));
  }

  __device__ __forceinline__ void first(int t) {
    lookup(t);
    turn();
    lookup(t + 1);
    if (moves_k())
#pragma unroll
      for (int i = 0; i < kPlanes; ++i) copy_k(t, i);
    put_usable(t);
    if constexpr (Q8) put_k(t);
    turn();
    auto one = [&](auto j) { copy<j.value>(t); };
    each(one, std::make_integer_sequence<int, kCopies>{});
    if constexpr (!Q8 && EXACT && W == 4)
      wait_vmem<kCopies>();  // the first K alone
    else
      wait_vmem<0>();
    __syncthreads();
    take_usable(t);
    lookup(t + 2);
  }
  __device__ __forceinline__ void close(int t) {
    wait_vmem<0>();
    put_v(t);
    put_k(t + 1);
    put_usable(t + 1);
    __syncthreads();
    take_usable(t + 1);
    turn();
    lookup(t + 3);
  }

  __device__ __forceinline__ uint32_t visible(int k0, uint32_t ok) const {
    const int d = held - k0;  // the tree's first row in the block
    uint32_t nodes = 0;
    if (d >= 0 && d < 32) nodes = (uint32_t)(mask << d);
    if (d < 0 && d > -kNodes) nodes = (uint32_t)(mask >> -d);
    return ok & ((below(d) & ~below(lo - k0)) | nodes);
  }
  // Usable keys of the block from k0 on, of the tile that is scored or the one before.
  __device__ __forceinline__ uint32_t ok_of(int k0) const {
    return k0 & 32 ? (uint32_t)(usable_before >> 32) : (uint32_t)usable;
  }
  __device__ __forceinline__ bool rough(int t) const {
    return Q8 || special || edge(t) || edge(t - 1) ||
           ((uint32_t)usable & (uint32_t)(usable_before >> 32)) != 0xFFFFFFFFu;
  }
  __device__ __forceinline__ void shape(f32x16& x, int k0) const {
    if constexpr (Q8) {
      const float* ks = s_scale + (k0 & (4 * kKeys - 1)) + 4 * (lane >> 5);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 y = *reinterpret_cast<const float4*>(ks + 8 * g);
        x[4 * g] *= y.x;
        x[4 * g + 1] *= y.y;
        x[4 * g + 2] *= y.z;
        x[4 * g + 3] *= y.w;
      }
    }
    if (special) Rows<D, BF>::shape(x, p.shape);
    const uint32_t ok = ok_of(k0);
    if (edge(k0 / kKeys) || ok != 0xFFFFFFFFu) Rows<D, BF>::mask(x, visible(k0, ok));
  }
  // After the piece's last tile: the values that were taken as zeros, to the rows that
  // see them.
  __device__ __forceinline__ void add_left_out(Rows<D, BF>& r, int ta, int tb) const {
    __syncthreads();
    if (uniform(*s_left) == 0) return;
    for (int t = ta; t < tb; ++t) {
      if (!edge(t)) continue;
      for (int k = t * kKeys; k <= min(t * kKeys + kKeys - 1, last); ++k) {
        const uint32_t pi = (uint32_t)k / (uint32_t)p.page_size;
        const uint32_t sl = (uint32_t)k - pi * (uint32_t)p.page_size;
        const int from = pi < (uint32_t)p.stride ? table[pi] : -1;
        if ((uint32_t)from >= pages) continue;
        const int64_t at = from * p.page_elems + (int64_t)sl * p.row_elems +
                           (int64_t)kvh * p.head_elems;
        const bool seen = k < held ? k >= lo : (mask >> (k - held) & 1) != 0;
        r.add_not_finite(seen, p.dim, [&](int d) {
          if constexpr (Q8) {
            const float vs = (float)p.vscale[from * p.scale_page + (int64_t)sl * p.scale_row +
                                             (int64_t)kvh * p.scale_head];
            const int8_t* y = static_cast<const int8_t*>(p.v) + at + d;
            return make_float4(y[0] * vs, y[1] * vs, y[2] * vs, y[3] * vs);
          } else {
            return widen4<BF>(static_cast<const f16*>(p.v) + at + d);
          }
        });
      }
    }
  }
};

// What a piece leaves to the one after it; in LDS, for the registers are the tiles'.
struct Walk {
  int64_t left, rest;  // tiles of the range, and where in the sequence's
  int seq, pieces;
};

template <int D, bool BF, bool Q8, int W, bool EXACT>
__global__ __launch_bounds__(64 * W, D <= 128 ? 2 : 1) void tree_attention_kernel(
    const TreeParams p) {
  using Tiles = TreeTiles<D, BF, Q8, W, EXACT>;
  __shared__ __align__(1024) f16 s_k[2 * Tiles::kHalves];
  __shared__ __align__(1024) f16 s_v[2 * Tiles::kHalves];
  __shared__ __align__(16) float s_scale[Q8 ? 4 * kKeys : 4];
  __shared__ __align__(8) uint16_t s_ok[4 * 4];
  __shared__ int s_left;

  const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
  const int G = p.hq / p.hkv;
  // Rows behind the last sequence: zeros.
  {
    const int real = p.batch > 0 ? max(0, min(p.starts[p.batch], p.tokens)) : 0;
    const int64_t from = (int64_t)real * p.hq * p.dim / 8, to = (int64_t)p.tokens * p.hq * p.dim / 8;
    for (int64_t i = from + blockIdx.x * (64 * W) + tid; i < to; i += (int64_t)gridDim.x * (64 * W))
      reinterpret_cast<f16x8*>(p.out)[i] = f16x8{};
  }
  __shared__ Walk s_walk;
  {
    const Range range = range_of(p);
    if (tid == 0) {
      p.cuts[blockIdx.x] = Cut{};
      s_walk = {range.end - range.begin, range.rest, range.seq, 0};
    }
    if (range.begin >= range.end) return;
  }
  Rows<D, BF> r;
  r.init(p.shape);
  Tiles x{p, s_k, s_v, s_scale, s_ok, &s_left};
  x.init();
  __syncthreads();
  for (;;) {
    int ta, tb;
    {
      const int64_t left = uniform64(s_walk.left), rest = uniform64(s_walk.rest);
      const int seq = uniform(s_walk.seq);
      const Seq s = uniform_seq(seq_of(p, seq));
      const int unit = uniform((int)(rest / s.nt));
      const int begin = (int)(rest - (int64_t)unit * s.nt);
      ta = s.t0 + begin;
      tb = s.t0 + (int)min((int64_t)s.nt, begin + left);
      x.kvh = uniform(unit / s.blocks);
      x.held = s.held;
      x.last = s.held + min(s.n, kNodes) - 1;
      x.table = p.tables + (int64_t)seq * p.stride;
      // This lane's row: a node and a query head. (Rows past the last see what that
      // one sees, and are not stored.)
      const int row = 32 * W * (unit - x.kvh * s.blocks) + 32 * w + (lane & 31);
      const int at = min(row, s.n * G - 1);
      const int node = at / G;
      r.clear();
      r.load(p.q + ((int64_t)(s.first + node) * p.hq + x.kvh * G + at % G) * p.dim, p.dim, true);
      x.mask = p.masks[s.first + node];
      x.lo = 0;
      if (p.window > 0) {
        x.lo = max(0, s.held + max(0, (int)__popcll(x.mask) - 1) - p.window + 1);
        while ((int)__popcll(x.mask) > p.window) x.mask &= x.mask - 1;
      }
      // (A wave that has no row sees no tile.)
      const bool live = uniform(row - (lane & 31)) < s.n * G;
      if (tid == 0) s_left = 0;
      attend(r, x, ta, tb, ta, live ? tb : ta, x.last >= (tb - 1) * kKeys + 32);
    }
    x.add_left_out(r, ta, tb);

    // (All of it anew: what was held over the tiles cost their registers.)
    const int64_t left = uniform64(s_walk.left), rest = uniform64(s_walk.rest);
    const int seq = uniform(s_walk.seq), pieces = uniform(s_walk.pieces);
    const Seq s = uniform_seq(seq_of(p, seq));
    const int unit = uniform((int)(rest / s.nt));
    const int begin = ta - s.t0, end = tb - s.t0;
    const int kvh = uniform(unit / s.blocks);
    const int first_row = 32 * W * (unit - kvh * s.blocks), all_rows = s.n * G;
    const int row = first_row + 32 * w + (lane & 31);
    if (end - begin == s.nt) {
      const float inv = r.inverse();
      if (row < all_rows)
        r.store(p.out + ((int64_t)(s.first + row / G) * p.hq + kvh * G + row % G) * p.dim, p.dim,
                inv);
    } else if (first_row + 32 * w < all_rows) {
      // A piece of a unit that is cut, as it is.
      const int64_t piece = (2 * (int64_t)blockIdx.x + (pieces ? 1 : 0)) * W + w;
      const float sum = r.l + __shfl_xor(r.l, 32);
      if (lane < 32) p.part_ml[piece * 32 + lane] = make_float2(r.m, sum);
      float4* dst = reinterpret_cast<float4*>(p.part_o) + piece * (D / 8 * 64) + lane;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        dst[64 * i] = make_float4(r.o[i / 4][4 * (i % 4)], r.o[i / 4][4 * (i % 4) + 1],
                                  r.o[i / 4][4 * (i % 4) + 2], r.o[i / 4][4 * (i % 4) + 3]);
    }
    if (pieces == 0 && begin > 0 && end == s.nt) {
      // The unit began in an earlier range: its first tile, and the workgroup of that.
      const Range range = range_of(p);
      const int64_t from = range.begin - begin;
      const int64_t g = ((from + 1) * range.n - 1) / range.all;
      if (tid == 0)
        p.cuts[blockIdx.x] = {min(all_rows - first_row, 32 * W), first_row, s.first, kvh,
                              (int)(2 * g + (from > range_begin(range.all, range.n, g) ? 1 : 0)),
                              (int)g + 1, {}};
    }
    const int64_t now = left - (end - begin);
    if (now <= 0) break;
    int64_t on = rest + (end - begin);
    int next = seq;
    if (on >= tiles_of(p, s)) {  // the next sequence that has a tree
      on = 0;
      do ++next;
      while (uniform(seq_of(p, next).nt) == 0);
    }
    __syncthreads();  // (others may still read the state and the last tile)
    if (tid == 0) s_walk = {now, on, next, pieces + 1};
    __syncthreads();
  }
}

// Joins the pieces of the unit that is cut and ends in a workgroup's range: with M the
// largest of their maxima, the outputs are sum 2^(m - M) o / sum 2^(m - M) l. A wave
// takes 32 rows and a quarter of their dims, the lanes as in the kernel that left them.
template <int D, bool BF>
__global__ __launch_bounds__(kThreads) void tree_join_kernel(const TreeParams p) {
  constexpr int kShare = D / 8 / 4;  // groups of 8 dims a wave takes
  constexpr int kAtOnce = 4;         // pieces loaded together
  const int g = blockIdx.x, w = blockIdx.y, waves = gridDim.y;
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const Cut cut = p.cuts[g];
  if (cut.rows <= 32 * w) return;
  // Its pieces: the first, then those of the workgroups up to this one.
  const int count = g - cut.group + 2;
  auto piece = [&](int i) {
    return (int64_t)(i == 0 ? cut.piece : 2 * (cut.group + i - 1)) * waves + w;
  };
  float top = -INFINITY;
  float4 acc[kShare];
#pragma unroll
  for (int i = 0; i < kShare; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
  for (int i0 = 0; i0 < count; i0 += kAtOnce) {
    float2 ml[kAtOnce];
    float4 o[kAtOnce][kShare];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t at = piece(min(i0 + j, count - 1));
      ml[j] = p.part_ml[at * 32 + (lane & 31)];
      const float4* src = reinterpret_cast<const float4*>(p.part_o) + at * (D / 8 * 64) +
                          part * kShare * 64 + lane;
#pragma unroll
      for (int i = 0; i < kShare; ++i) o[j][i] = src[64 * i];
    }
    float now = top;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) now = fmaxf(now, ml[j].x);
    const float f0 = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - now);
    top = now;
    // (Before any key was seen sums and outputs are zeros, or NaN where a piece was.)
    if (f0 != 0.0f || sum == 0.0f) {
      sum *= f0;
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        acc[i].x *= f0;
        acc[i].y *= f0;
        acc[i].z *= f0;
        acc[i].w *= f0;
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      // (A piece of which the row sees nothing holds zeros. One of NaN is not empty.)
      const bool empty = i0 + j >= count || (ml[j].x == -INFINITY && ml[j].y == 0.0f);
      const float f = empty ? 0.0f : __builtin_amdgcn_exp2f(ml[j].x - top);
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        acc[i].x = fmaf(empty ? 0.0f : o[j][i].x, f, acc[i].x);
        acc[i].y = fmaf(empty ? 0.0f : o[j][i].y, f, acc[i].y);
        acc[i].z = fmaf(empty ? 0.0f : o[j][i].z, f, acc[i].z);
        acc[i].w = fmaf(empty ? 0.0f : o[j][i].w, f, acc[i].w);
      }
      sum = empty ? sum : fmaf(ml[j].y, f, sum);
    }
  }
  const int r = 32 * w + (lane & 31);
  if (r >= cut.rows) return;
  const int G = p.hq / p.hkv, row = cut.first + r;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  f16* dst = p.out + ((int64_t)(cut.token + row / G) * p.hq + cut.kvh * G + row % G) * p.dim;
#pragma unroll
  for (int i = 0; i < kShare; ++i) {
    const int d = 8 * (part * kShare + i) + 4 * (lane >> 5);
    const f16x4 y = {round16<BF>(acc[i].x * inv), round16<BF>(acc[i].y * inv),
                     round16<BF>(acc[i].z * inv), round16<BF>(acc[i].w * inv)};
    if (d < p.dim) *reinterpret_cast<f16x4*>(dst + d) = y;
  }
}

// Other head dims than the widths take the four-wave kernels.
template <bool BF, bool Q8>
const void* tree_kernel_for(int width, int waves, bool exact) {
  if (!exact)
    return width == 64   ? reinterpret_cast<const void*>(tree_attention_kernel<64, BF, Q8, 4, false>)
           : width == 96 ? reinterpret_cast<const void*>(tree_attention_kernel<96, BF, Q8, 4, false>)
           : width == 128
               ? reinterpret_cast<const void*>(tree_attention_kernel<128, BF, Q8, 4, false>)
               : reinterpret_cast<const void*>(tree_attention_kernel<256, BF, Q8, 4, false>);
  if (waves == 8)
    return width == 64   ? reinterpret_cast<const void*>(tree_attention_kernel<64, BF, Q8, 8, true>)
           : width == 96 ? reinterpret_cast<const void*>(tree_attention_kernel<96, BF, Q8, 8, true>)
                         : reinterpret_cast<const void*>(tree_attention_kernel<128, BF, Q8, 8, true>);
  return width == 64    ? reinterpret_cast<const void*>(tree_attention_kernel<64, BF, Q8, 4, true>)
         : width == 96  ? reinterpret_cast<const void*>(tree_attention_kernel<96, BF, Q8, 4, true>)
         : width == 128 ? reinterpret_cast<const void*>(tree_attention_kernel<128, BF, Q8, 4, true>)
                        : reinterpret_cast<const void*>(tree_attention_kernel<256, BF, Q8, 4, true>);
}
template <bool BF>
const void* tree_join_for(int width) {
  return width == 64    ? reinterpret_cast<const void*>(tree_join_kernel<64, BF>)
         : width == 96  ? reinterpret_cast<const void*>(tree_join_kernel<96, BF>)
         : width == 128 ? reinterpret_cast<const void*>(tree_join_kernel<128, BF>)
                        : reinterpret_cast<const void*>(tree_join_kernel<256, BF>);
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
  const void* fn = q8 ? (bf16_elems ? tree_kernel_for<true, true>(width, waves, exact)
                                    : tree_kernel_for<false, true>(width, waves, exact))
                      : (bf16_elems ? tree_kernel_for<true, false>(width, waves, exact)
                                    : tree_kernel_for<false, false>(width, waves, exact));
  hipError_t err = hipLaunchKernel(fn, dim3(prm.groups), dim3(64 * waves), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  if (batch == 0) return ok();
  err = hipLaunchKernel(bf16_elems ? tree_join_for<true>(width) : tree_join_for<false>(width),
                        dim3(prm.groups, waves), dim3(kThreads), args, 0, hs);
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
