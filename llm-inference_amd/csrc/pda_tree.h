// The kernel of attention for drafted trees (pda_tree_attention), instantiated by
// element type in pda_tree_*.hip so that they compile side by side.
//
// What bounds it (64 sequences of 512-8192 rows, trees of 8-24 nodes, 28/4 heads of 128,
// bf16: 619 MB of keys and values; the split kernel 173-186 us, the join 10-14): without
// the math it takes 170 us, without the copies 129, with neither pages nor copies 102. Of
// the 170 the pieces of cut units are 16 (512 ranges over 256 units) and every piece's
// chain of lengths, table entries, first rows some 5. A ring of blocks of 32 keys with two
// to three always under way streamed faster (161 us; 2 sequences of 116000 rows 194
// instead of 245) but its barrier every 32 keys cost the math more than that (205 and
// 372 us instead of 188 and 330), as did touching the tile after next ahead of its copies
// (222); whole 128-byte lines a copy or non-temporal ones changed nothing or lost (176,
// 196). Two sequences of 100000-131072 rows, trees of 48-64 nodes, 32/8 heads: 290-330
// us, 680-750 TFLOP/s, 3.1-3.4 TB/s: copies alone 230, math alone 250.
#ifndef PDA_TREE_H
#define PDA_TREE_H

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "pda_rows.h"

namespace pda_tree {

using namespace pda_rows;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;  // of a workgroup of four waves
constexpr int kNodes = 64;     // of a tree
constexpr int kCus = 256;
// Workgroups: as many as the GPU holds at once.
constexpr int groups_for(int width, int waves) { return width <= 128 && waves == 4 ? 2 * kCus : kCus; }
// A unit of n tiles in ranges of r takes about r tiles' time and then n / r pieces', of
// some kPieceCost tile times each, to join: least at r = sqrt(kPieceCost n).
constexpr float kPieceCost = 0.2f;

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
  const int64_t room = min((int64_t)p.stride * p.page_size, (int64_t)INT32_MAX - 1024);
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

// Workgroups that take ranges of a stream of `tiles` in `units`, and the first tile of
// one's.
__device__ __forceinline__ int64_t ranges(const TreeParams& p, int64_t tiles, int64_t units) {
  const int64_t least = max(1, (int)sqrtf(kPieceCost * ((float)tiles / (float)max(units, (int64_t)1))));
  const int64_t n = min((tiles + least - 1) / least, (int64_t)p.groups);
  // (One workgroup a CU rather than a second one on some: 4 sequences of 1000-2000 rows,
  // 32/8 heads of 128, 384 ranges 35 us a call, 256 30.)
  return n > kCus && n < p.groups ? (int64_t)kCus : n;
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
  int64_t mine = 0, units = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = seq_of(p, b);
    mine += tiles_of(p, s);
    units += s.nt > 0 ? (int64_t)s.blocks * p.hkv : 0;
  }
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(upto, d);
    if (lane >= d) upto += y;
    units += __shfl_xor(units, d);
  }
  Range r;
  r.all = uniform64(__shfl(upto, 63));
  r.n = uniform64(ranges(p, r.all, uniform64(units)));
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
  static constexpr bool kSpread = false;  // the copies are issued at once: they are waited for
  // 8 bits: the keys are exact in either type, the values times their scales are rounded,
  // to fp16 also under bf16 queries (to bf16, and the weights with them, the outputs were
  // 1.65 times as far from 64 bits as their own rounding puts them: 0.0028 and 0.0017).
  static constexpr bool kVbf = BF && !Q8;
  using R = Rows<D, BF, kVbf>;

  const TreeParams& p;
  f16* s_k;          // [2][kHalves]
  f16* s_v;
  float* s_scale;    // [4][64] the keys' scales, by tile
  uint16_t* s_ok;    // [4][4] usable keys, by tile and wave
  int* s_left;       // whether values that are not finite were taken as zeros
  bool special;
  int lane, w, gk, kchunk, vchunk, shift;
  uint32_t k_dst, v_dst, pages;

  // The piece's.
  const int32_t* table;
  int kvh, held, last;
  uint64_t mask;  // nodes that the lane's row sees
  int lo;         // and the first row held
  // This thread's key of the tiles whose V and K are copied next, and the looked-up
  // page of the tile after them.
  const char* from_k;
  const char* from_v;
  uint64_t at_k;
  int64_t scale_v, scale_k;
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
    shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
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

  // (Page sizes are powers of two as a rule: no division then.)
  __device__ __forceinline__ void lookup(int t) {
    const uint32_t kp = (uint32_t)t * kKeys + gk;
    const uint32_t pi = shift >= 0 ? kp >> shift : kp / (uint32_t)p.page_size;
    slot = kp - pi * (uint32_t)p.page_size;
    in = kp <= (uint32_t)last && pi < (uint32_t)p.stride;
    page = table[min(pi, (uint32_t)p.stride - 1)];
  }
  // The looked-up tile becomes the next K to copy, the one before it the next V. (An
  // element of either arena is a byte at 8 bits, else two.)
  __device__ __forceinline__ void turn() {
    constexpr int kBytes = Q8 ? 1 : 2;
    from_v = static_cast<const char*>(p.v) + at_k + kBytes * vchunk;
    ok_v = ok_k;
    ok_k = in && (uint32_t)page < pages;
    const uint32_t from = ok_k ? page : 0;
    at_k = kBytes * ((uint64_t)from * (uint32_t)p.page_elems +
                     (uint64_t)(uint32_t)((int)slot * p.row_elems + kvh * p.head_elems));
    from_k = static_cast<const char*>(p.k) + at_k + kBytes * kchunk;
    if constexpr (Q8) {
      scale_v = scale_k;
      scale_k = (int64_t)from * p.scale_page + (int)slot * p.scale_row + kvh * p.scale_head;
    }
  }
  template <int i>
  __device__ __forceinline__ void copy_k(int t) {
    if constexpr (Q8) {
      if (i == 0) raw_ks = p.kscale[scale_k];
    }
    if (!EXACT && 32 * i + kchunk >= p.dim) return;
    if constexpr (Q8)
      raw_k[i] = *reinterpret_cast<const u32x2*>(from_k + 32 * i);
    else
      copy_plane_to_lds<i>(from_k, k_dst + (t & 1) * (2 * kHalves));
  }
  template <int i>
  __device__ __forceinline__ void copy_v(int t) {
    if constexpr (Q8) {
      if (i == 0) raw_vs = p.vscale[scale_v];
    }
    if (!EXACT && 32 * i + vchunk >= p.dim) return;
    if constexpr (Q8)
      raw_v[i] = *reinterpret_cast<const u32x2*>(from_v + 32 * i);
    else
      copy_plane_to_lds<i>(from_v, v_dst + (t & 1) * (2 * kHalves));
  }
  template <int j>
  __device__ __forceinline__ void copy(int t) {
    if constexpr (W == 4) {
      if constexpr (j < kPlanes)
        copy_v<j>(t);
      else
        copy_k<j - kPlanes>(t + 1);
    } else {
      if (w < 4)
        copy_v<j>(t);
      else
        copy_k<j>(t + 1);
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
        f16x8 x = from_bytes<kVbf>(raw_v[i], vs);
        if (!ok_v) x = f16x8{};
        if (check && not_finite<kVbf>(x)) {
          *s_left = 1;
          x = finite_only<kVbf>(x);
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
        if (not_finite<kVbf>(x)) {
          *s_left = 1;
          *reinterpret_cast<f16x8*>(dst + kPlane * i) = finite_only<kVbf>(x);
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
    if (moves_k()) {
      auto one = [&](auto i) { copy_k<i.value>(t); };
      each(one, std::make_integer_sequence<int, kPlanes>{});
    }
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
  __device__ __forceinline__ void aim(int) const {}  // (turn has)
  __device__ __forceinline__ void ahead(R&) const {}
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
    if (special) R::shape(x, p.shape);
    const uint32_t ok = ok_of(k0);
    if (edge(k0 / kKeys) || ok != 0xFFFFFFFFu) R::mask(x, visible(k0, ok));
  }
  // After the piece's last tile: the values that were taken as zeros, to the rows that
  // see them.
  __device__ __forceinline__ void add_left_out(R& r, int ta, int tb) const {
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
            auto value = [&](int i) { return widen16<kVbf>(round16<kVbf>(y[i] * vs)); };
            return make_float4(value(0), value(1), value(2), value(3));
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
  using Tiles = TreeTiles<D, BF, Q8, W, EXACT>;  // EXACT: the head dim is D
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
  typename Tiles::R r;
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
      r.settle_queries();
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

const void* tree_kernel_f16(int width, int waves, bool exact);
const void* tree_kernel_bf16(int width, int waves, bool exact);
const void* tree_kernel_q8(int width, int waves, bool exact);
const void* tree_kernel_q8_bf16(int width, int waves, bool exact);

}  // namespace pda_tree

#endif  // PDA_TREE_H
