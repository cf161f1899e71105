// Latent attention for MI355X (gfx950): the append of latent rows and the
// decode attention over them in the absorbed form, C-ABI in pda.h
// (pda_latent_append, pda_latent_decode_attention). No reference counterpart:
// the reference keeps keys and values per kv head.
//
// A token's cache row is [c | k]: its normalised latent c (latent_dim wide),
// from which every head's keys and values are projected, and one rotated key k
// (rope_dim wide) that all heads share. With W_h = kv_b[h] = [U_h; D_h]
// (nope_dim and value_dim rows over the latent) head h has
//   key(t) = [U_h c_t ; k_t],  value(t) = D_h c_t,
//   score(t) = scale (q_nope . U_h c_t + q_rope . k_t).
// Absorbed: q_nope . U_h c = (U_h^T q_nope) . c, and the weighted values are
// D_h applied once to the weighted latents. So a step projects its queries
// (latent_absorb_kernel), attends over the rows themselves, all heads from one
// read (latent_decode_kernel), and projects what comes out
// (latent_merge_kernel, which joins the parts of a sequence on the way).

#include <algorithm>
#include <type_traits>
#include <utility>

#include "pda_latent.h"

namespace {

using namespace pda_latent;
using pda_internal::fail;
using pda_internal::ok;

// ---------------------------------------------------------------------------
// Append.

constexpr int kAppendHeads = 16;  // query heads of one token a workgroup takes

struct LatentAppendParams {
  const f16* q;       // [n, hq, nope + rope], or null
  f16* q_out;
  const f16* c;       // [n, latent], rows c_stride apart
  const f16* k;       // [n, rope], rows k_stride apart
  const f16* norm;    // [latent], or null: latents are stored as they are
  f16* arena;         // [arena_rows, latent + rope]
  const int32_t* positions;
  const int32_t* rows;
  const float* inv_freq;  // [rope / 2], or null: no rotation
  int64_t c_stride;
  int64_t k_stride;
  int64_t arena_rows;
  int32_t n;
  int32_t hq;
  int32_t latent;
  int32_t rope;
  int32_t nope;
  int32_t head_groups;  // workgroups of query heads per token
  float eps;
};

// The rotation of 8 pairs (a[i], b[i]) by the angles whose cosines and sines
// are given: separately rounded float32 products and sums, as the other
// append's, rounded to the element type.
template <bool BF>
__device__ __forceinline__ void rotate(f16x8& a, f16x8& b, const float* cs, const float* sn) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = widen<BF>(a[i]), y = widen<BF>(b[i]);
    a[i] = round16<BF>(__fsub_rn(__fmul_rn(x, cs[i]), __fmul_rn(y, sn[i])));
    b[i] = round16<BF>(__fadd_rn(__fmul_rn(y, cs[i]), __fmul_rn(x, sn[i])));
  }
}

// The first workgroups write the rows, a wave a token (a lane 8 latent dims);
// the others rotate the queries, kAppendHeads heads of a token each, in
// 16-byte pieces: a piece of the nope part is copied (left alone when q_out is
// q), a pair of pieces half the rotary part apart is rotated. A token's angles
// are computed once a workgroup. Moves every byte once, which bounds it: 4096
// tokens of 128 heads 82 us for 413 MB (5.0 TB/s), 8 of 16 heads 3.7 us (a
// launch's latency).
template <bool BF>
__global__ __launch_bounds__(256) void latent_append_kernel(const LatentAppendParams p) {
  __shared__ float s_cos[4][kMaxRope / 2], s_sin[4][kMaxRope / 2];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int half = p.rope / 2;
  const int row_groups = p.c ? (p.n + 3) / 4 : 0;
  auto angles = [&](int token, int slot, int i) {
    if (i < half) {
      float sn, cs;
      sincosf(__fmul_rn((float)p.positions[token], p.inv_freq[i]), &sn, &cs);
      s_cos[slot][i] = cs;
      s_sin[slot][i] = sn;
    }
  };
  if ((int)blockIdx.x < row_groups) {
    const int token = blockIdx.x * 4 + w;
    const bool live = token < p.n;
    if (live && p.inv_freq) angles(token, w, lane);
    __syncthreads();
    if (!live) return;
    const int64_t row = p.rows[token];
    if (row < 0 || row >= p.arena_rows) return;
    f16* dst = p.arena + row * (p.latent + p.rope);
    const bool mine = 8 * lane < p.latent;
    f16x8 x = {};
    if (mine) x = *reinterpret_cast<const f16x8*>(p.c + token * p.c_stride + 8 * lane);
    if (p.norm) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(widen<BF>(x[i]), widen<BF>(x[i]), sum);
#pragma unroll
      for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
      const float r = 1.0f / sqrtf(sum / (float)p.latent + p.eps);
      if (mine) {
        const f16x8 g = *reinterpret_cast<const f16x8*>(p.norm + 8 * lane);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = round16<BF>(widen<BF>(x[i]) * r * widen<BF>(g[i]));
      }
    }
    if (mine) *reinterpret_cast<f16x8*>(dst + 8 * lane) = x;
    if (8 * lane < half) {
      const f16* src = p.k + token * p.k_stride;
      f16x8 a = *reinterpret_cast<const f16x8*>(src + 8 * lane);
      f16x8 b = *reinterpret_cast<const f16x8*>(src + half + 8 * lane);
      if (p.inv_freq) rotate<BF>(a, b, &s_cos[w][8 * lane], &s_sin[w][8 * lane]);
      *reinterpret_cast<f16x8*>(dst + p.latent + 8 * lane) = a;
      *reinterpret_cast<f16x8*>(dst + p.latent + half + 8 * lane) = b;
    }
    return;
  }
  const int item = blockIdx.x - row_groups;
  const int token = item / p.head_groups, h0 = (item % p.head_groups) * kAppendHeads;
  if (p.inv_freq) {
    angles(token, 0, tid);
    __syncthreads();
  }
  const int heads = min(kAppendHeads, p.hq - h0);
  const int width = p.nope + p.rope;
  const int64_t at = ((int64_t)token * p.hq + h0) * width;
  const int pairs = half / 8, pieces = p.nope / 8 + pairs;  // a head's work items
  const bool in_place = p.q == p.q_out;
  for (int i = tid; i < heads * pieces; i += 256) {
    const int h = i / pieces, j = i - h * pieces;
    if (j >= pairs) {
      const int64_t e = at + h * width + 8 * (j - pairs);
      if (!in_place)
        *reinterpret_cast<f16x8*>(p.q_out + e) = *reinterpret_cast<const f16x8*>(p.q + e);
      continue;
    }
    const int64_t e = at + h * width + p.nope + 8 * j;
    f16x8 a = *reinterpret_cast<const f16x8*>(p.q + e);
    f16x8 b = *reinterpret_cast<const f16x8*>(p.q + e + half);
    if (p.inv_freq) rotate<BF>(a, b, &s_cos[0][8 * j], &s_sin[0][8 * j]);
    *reinterpret_cast<f16x8*>(p.q_out + e) = a;
    *reinterpret_cast<f16x8*>(p.q_out + e + half) = b;
  }
}

// ---------------------------------------------------------------------------
// Decode.

constexpr int kTileKeys = 32;     // keys per tile
constexpr int kChunkTiles = 64;   // tiles whose rows are looked up at once
constexpr int kChunkKeys = kTileKeys * kChunkTiles;
constexpr int kMaxGroups = 256;   // workgroups of a launch: one per CU of an MI355X
constexpr float kSlack = 8.0f;    // scores may pass the running max by 2^8
// What a workgroup spends on a sequence besides its tiles (queries, rows, the
// partial), in tiles: the cuts of the stream count it. (Counted as 2, 64 sequences
// of 64 heads 107 us a call for 101, of 128 heads 139 for 131.)
constexpr int kSequenceTiles = 8;

struct LatentDecodeParams {
  const f16* q;          // [batch, hq, nope + rope]
  const f16* kv_b;       // [hq, nope + value, latent]
  const f16* arena;      // [arena_rows, latent + rope]
  const int32_t* tables; // [batch, table_stride]
  const int32_t* lengths;
  f16* out;              // [batch, hq, value]
  f16* q_lat;            // [batch, hq, latent + rope]: absorbed queries
  float* q_size;         // [batch, hq]: the absorbed queries times this are true (fp16)
  int32_t* prefix;       // [batch + 1] tiles, kSequenceTiles a sequence, before each
  float* part_o;         // [groups + batch, hq, latent] unnormalised partial sums
  float2* part_ml;       // [groups + batch, hq] (running max, sum)
  int64_t arena_pages;
  int32_t table_stride;
  int32_t page_size;
  int32_t batch;
  int32_t hq;
  int32_t latent;
  int32_t rope;
  int32_t nope;
  int32_t value;
  int32_t groups;        // workgroups the stream of tiles is cut over
  int32_t merge_batch;   // sequences a merge workgroup takes
  int32_t once;          // rows past the caches
  float scale_log2;
};

__device__ __forceinline__ int64_t keys_of(const LatentDecodeParams& p, int b) {
  const int64_t cap = (int64_t)p.table_stride * p.page_size;
  return max((int64_t)0, min((int64_t)p.lengths[b], cap));
}

// Units of the stream that sequence b takes.
__device__ __forceinline__ int units_of(const LatentDecodeParams& p, int b) {
  const int tiles = (int)((keys_of(p, b) + kTileKeys - 1) / kTileKeys);
  return tiles ? tiles + kSequenceTiles : 0;
}

// The value of the lane kBy on in a row of 16 lanes.
template <int kBy>
__device__ __forceinline__ uint32_t row_turned(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + kBy, 0xf, 0xf, false);
}

// Queries into the latent: q_lat[b, h] = [U_h^T q_nope | q_rope], rounded to
// the element type, because the matrix cores take 16-bit operands (the products
// and their sum are float32). It moves the result by about as much as the
// output's own rounding: in bf16 1.6e-3 of its 2-norm beside 1.7e-3. In fp16
// q_lat may pass the type's range where queries and projections are far inside
// it: a query with elements from 2^7 on is taken down by a power of two, which the
// scores are multiplied by again (q_size); a latent dim whose |U_h| sum to less
// than 512 then stays finite whatever the query. As products: (U_h^T) (32 latent
// dims x nope) by (q_nope)^T (nope x 32 sequences); a wave has 32 latent dims,
// whose columns of U_h it keeps in LDS and reads transposed. U_h is read once per
// 32 sequences.
// The first workgroup also leaves the sequences' tile prefix for the kernels
// after it. 64 sequences of 128 heads 11 us (26 MB; the reads in turn of U_h, q
// and the rows bound it), one of 16 heads 4 us.
template <bool BF>
__global__ __launch_bounds__(256) void latent_absorb_kernel(const LatentDecodeParams p) {
  __shared__ __align__(1024) f16 s_u[4][kMaxHead * 32];
  __shared__ __align__(16) f16 s_q[32 * (kMaxHead + 8)];
  __shared__ int s_scan[256];
  __shared__ f16 s_down[32];
  const int tid = threadIdx.x, w = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 31, hh = lane >> 5;
  const int h = blockIdx.y, b0 = blockIdx.z * 32;
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
    const int each = (p.batch + 255) / 256, first = min(tid * each, p.batch);
    const int end = min(first + each, p.batch);
    int sum = 0;
    for (int b = first; b < end; ++b) sum += units_of(p, b);
    s_scan[tid] = sum;
    __syncthreads();
    for (int d = 1; d < 256; d <<= 1) {
      const int x = tid >= d ? s_scan[tid - d] : 0;
      __syncthreads();
      s_scan[tid] += x;
      __syncthreads();
    }
    int at = s_scan[tid] - sum;
    for (int b = first; b < end; ++b) {
      p.prefix[b] = at;
      at += units_of(p, b);
    }
    if (tid == 255) p.prefix[p.batch] = s_scan[255];
  }
  const int width = p.latent + p.rope, qwidth = p.nope + p.rope;
  // The rotary part is copied, in fp16 taken down like the rest: a piece a thread.
  static_assert(32 * (kMaxRope / 8) <= 256, "a piece a thread");
  const int pieces = max(p.rope / 8, 1), rot_row = tid / pieces;
  const bool rotary = blockIdx.x == 0 && tid < 32 * (p.rope / 8) && b0 + rot_row < p.batch;
  const int64_t rot_head = (int64_t)(b0 + rot_row) * p.hq + h;
  const int rot_dim = 8 * (tid % pieces);
  f16x8 rot = {};
  if (rotary) rot = *reinterpret_cast<const f16x8*>(p.q + rot_head * qwidth + p.nope + rot_dim);
  const int d0 = (blockIdx.x * 4 + w) * 32;
  // The wave's columns of U_h: rows of 64 bytes, zeros past either edge.
  const f16* u = p.kv_b + (int64_t)h * (p.nope + p.value) * p.latent;
  const int col = d0 + 8 * (lane & 3);
  f16x8 rows[kMaxHead / 16];
#pragma unroll
  for (int i = 0; i < kMaxHead / 16; ++i) {
    const int r = 16 * i + (lane >> 2);
    rows[i] = f16x8{};
    if (r < p.nope && col < p.latent)
      rows[i] = *reinterpret_cast<const f16x8*>(u + (int64_t)r * p.latent + col);
  }
  // The queries of 32 sequences, by rows, zeros past either edge.
  constexpr int kQPitch = kMaxHead + 8;
#pragma unroll
  for (int i = tid; i < 32 * (kMaxHead / 8); i += 256) {
    const int r = i / (kMaxHead / 8), d = 8 * (i % (kMaxHead / 8));
    f16x8 x = {};
    if (b0 + r < p.batch && d < p.nope)
      x = *reinterpret_cast<const f16x8*>(p.q + ((int64_t)(b0 + r) * p.hq + h) * qwidth + d);
    if constexpr (!BF) {
      // The largest of a query's elements, whose 16 lanes are a row of the wave:
      // without their signs fp16 numbers have the order of their bits.
      u16x8 bits = __builtin_bit_cast(u16x8, x) & (unsigned short)0x7FFF;
      unsigned int top = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) top = max(top, (unsigned int)bits[t]);
      top = max(top, row_turned<8>(top));
      top = max(top, row_turned<4>(top));
      top = max(top, row_turned<2>(top));
      top = max(top, row_turned<1>(top));
      const int e = max(0, (int)(top >> 10) - (15 + 6));  // 2^7 and up: 1 and up
      const f16 f = __builtin_bit_cast(f16, (unsigned short)((15 - e) << 10));
#pragma unroll
      for (int t = 0; t < 8; ++t) x[t] *= f;
      if (d == 0) {
        s_down[r] = f;
        if (blockIdx.x == 0 && b0 + r < p.batch)
          p.q_size[(int64_t)(b0 + r) * p.hq + h] = __uint_as_float((uint32_t)(127 + e) << 23);
      }
    }
    *reinterpret_cast<f16x8*>(s_q + r * kQPitch + d) = x;
  }
  f16* su = s_u[w];
#pragma unroll
  for (int i = 0; i < kMaxHead / 16; ++i)
    *reinterpret_cast<f16x8*>(su + (16 * i + (lane >> 2)) * 32 + 8 * (lane & 3)) = rows[i];
  __syncthreads();
  const int g16 = lane >> 4, s16 = lane & 15;
  const f16* vp = su + (4 * (g16 >> 1) + (s16 >> 2)) * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
  const f16* qp = s_q + n * kQPitch + 4 * hh;
  f32x16 acc = {};
#pragma unroll
  for (int i = 0; i < kMaxHead / 16; ++i) {
    if (16 * i >= p.nope) break;
    const f16x4 lo = read_tr(vp + 512 * i), hi = read_tr(vp + 512 * i + 256);
    const f16x4 ql = *reinterpret_cast<const f16x4*>(qp + 16 * i);
    const f16x4 qh = *reinterpret_cast<const f16x4*>(qp + 16 * i + 8);
    acc = mfma16<BF>(f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]},
                     f16x8{ql[0], ql[1], ql[2], ql[3], qh[0], qh[1], qh[2], qh[3]}, acc);
  }
  // The workgroup's 32 x 128 results through LDS, written along the rows.
  constexpr int kPitch = 136;
  __syncthreads();
  f16* so = s_u[0];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    f16x4 y;
#pragma unroll
    for (int t = 0; t < 4; ++t) y[t] = round16<BF>(acc[4 * g + t]);
    *reinterpret_cast<f16x4*>(so + n * kPitch + 32 * w + 8 * g + 4 * hh) = y;
  }
  __syncthreads();
#pragma unroll
  for (int i = tid; i < 32 * 16; i += 256) {
    const int b = b0 + i / 16, d = blockIdx.x * 128 + 8 * (i % 16);
    if (b < p.batch && d < p.latent)
      *reinterpret_cast<f16x8*>(p.q_lat + ((int64_t)b * p.hq + h) * width + d) =
          *reinterpret_cast<const f16x8*>(so + (i / 16) * kPitch + 8 * (i % 16));
  }
  if (rotary) {
    if constexpr (!BF) rot *= s_down[rot_row];
    *reinterpret_cast<f16x8*>(p.q_lat + rot_head * width + p.latent + rot_dim) = rot;
  }
}

// Attention over the latent rows. The tiles (32 keys) of all sequences form
// one stream, cut into `groups` equal ranges, so that ragged batches and single
// long sequences load the CUs alike; a workgroup walks its range and writes one
// partial (max, sum, weighted latents) per sequence it meets, to slot group +
// sequence (both only grow along the stream, so no two share one).
//
// A wave holds 32 heads entire: queries (72 half2 a lane at 512 + 64 dims) and
// weighted latents (32 x 512 in 256 accumulator registers), so the weights go
// from the scores' registers to the next product without LDS: scores S^T = K
// Q^T leave a lane 16 keys of one head, which are the B operand of O^T += V^T
// P^T when V's rows are read in that order (two transposed reads). K and V are
// the same rows: one copy in LDS serves both, in planes of 64 dims whose 16-byte
// pieces are swizzled so that neither read meets a bank twice (swizzle). A copy
// instruction moves 128 bytes of 8 rows: at 64 bytes of 16 rows the L2 was asked
// twice as often, and its requests bound the launch.
// The weights are rounded to 16 bits for the second product, and the sum that
// divides it is of the rounded ones; in bf16 that moves the result by 1.2e-3 of its
// 2-norm. (Two 16-bit numbers a weight would take that to nothing and a third
// more time: 64 x 128 heads 132 us for 101, and the result from 2.5e-3 to 2.3e-3.)
// 64 sequences of 512 to 8192 keys, 128 heads: 102 us for 82 GFLOP and 339 MB of
// rows, the products and the rows about alike; 32 heads, two sequences of 228
// thousand keys together 56 us (263 MB, 4.7 TB/s: the rows).
// NHG: waves side by side over heads, sharing a tile; 4 / NHG groups of waves
// take tiles in turn. The LDS holds four tiles: a ring of NHG per group.
template <int WP, int OB, int NHG, bool BF>
__global__ __launch_bounds__(256, 1) void latent_decode_kernel(const LatentDecodeParams p) {
  constexpr int kGroups = 4 / NHG;           // tiles under way side by side
  constexpr int kPlane = kTileKeys * 64;     // halves of a 64-dim plane of a tile
  constexpr int kTile = WP * kPlane;
  constexpr int kChunks = 4 * WP;            // 16-dim steps of a row
  constexpr int kRows = 4 / NHG;             // 8-row parts of a tile a wave copies
  constexpr int kJoin = OB > 8 ? 256 : 128;  // dims joined at once
  constexpr int kPitch = kJoin + 4;          // floats of a head's
  // Operands read early: as many as the registers hold beside the queries.
  constexpr int kAhead = NHG == 1 ? 2 : NHG == 2 ? 3 : 4;
  __shared__ __align__(1024) f16 s_t[4][kTile];
  __shared__ int s_row[kChunkKeys];
  __shared__ float2 s_ml[4][32];
  __shared__ int s_at[4];
  static_assert(4 * 32 * kPitch * 4 <= sizeof(s_t), "the joined sums use the tiles' LDS");

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int n = lane & 31, hh = lane >> 5;
  const int hg = w % NHG, kg = w / NHG;
  const int head0 = blockIdx.y * 32 * NHG;
  const int h = head0 + 32 * hg + n;
  const bool live = h < p.hq;
  const int width = p.latent + p.rope;

  const int total = scalar_load(p.prefix, p.batch);
  const int per = (int)(((uint32_t)total + p.groups - 1) / (uint32_t)p.groups);
  const int64_t from = (int64_t)blockIdx.x * per;
  if (from >= total) return;
  const int t0 = (int)from, t1 = (int)min((int64_t)total, from + per);
  // The sequence that holds unit t0: those that end at or before it lie before it.
  int before = 0;
  for (int i = tid; i < p.batch; i += 256) before += p.prefix[i + 1] <= t0 ? 1 : 0;
#pragma unroll
  for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d);
  if (lane == 0) s_at[w] = before;
  __syncthreads();
  int b = uniform(s_at[0] + s_at[1] + s_at[2] + s_at[3]);

  // A lane's places in a tile's plane for the two reads: steps of 16 dims, and 8
  // rows or 32 dims on, differ in bits of the swizzled place.
  const int g16 = lane >> 4, s16 = lane & 15;
  const int k_place = 64 * n + 8 * (hh ^ swizzle(n));
  const int v_row = 4 * hh + (s16 >> 2);
  const int v_place = 64 * v_row + 4 * (s16 & 1) +
                      8 * ((2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ swizzle(v_row));
  // The copies: lane i of an instruction moves a 16-byte piece of row i / 8 (of
  // 8); pieces past the row's end (widths below the kernel's) are another
  // piece of the row, whose query elements are zeros. The wave has the rows of
  // parts hg, hg + NHG, ..
  const int last_piece = width / 8 - 1;
  const bool whole = width == 64 * WP;
  auto each_plane = [&](auto f) { each(f, std::make_integer_sequence<int, WP>{}); };
  const int row0 = 8 * hg + (lane >> 3), piece0 = (lane & 7) ^ swizzle(row0);
  // Row 8 (hg + NHG i) + lane / 8 and its piece's place.
  auto part_row = [&](int i) { return row0 + 8 * NHG * i; };
  auto piece = [&](int i) { return piece0 ^ 2 * (NHG * i & 1); };
  const uint32_t lds = uniform(lds_address(&s_t[0][0]));
  const uint32_t pages = (uint32_t)min(p.arena_pages, (int64_t)INT32_MAX);

  // A positive scale is applied with the maximum's subtraction, another one to
  // the scores.
  const bool direct = p.scale_log2 > 0.0f;
  float c = direct ? p.scale_log2 : 1.0f;

  for (; b < p.batch; ++b) {
    const int seq0 = scalar_load(p.prefix, b), seq1 = scalar_load(p.prefix, b + 1);
    const int keys =
        (int)max((int64_t)0, min((int64_t)scalar_load(p.lengths, b),
                                 (int64_t)p.table_stride * p.page_size));
    if (seq0 >= t1) break;
    const int tb = min(t1, seq1) - seq0 - kSequenceTiles;
    const int ta = max(0, t0 - seq0 - kSequenceTiles);
    if (ta >= tb) continue;  // none of the sequence's tiles

    // Arena rows of a chunk's keys; -1: no such key, or no such page.
    constexpr int kEach = kChunkKeys / 256;
    uint32_t page[kEach];
    auto look_up = [&](int c0) {
      const int64_t table = (int64_t)b * p.table_stride;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint32_t key = (uint32_t)c0 * kTileKeys + 256 * i + tid;  // (may pass 2^31)
        page[i] = ~0u;
        if (256 * i < min(tb - c0, kChunkTiles) * kTileKeys && key < (uint32_t)keys)
          page[i] = (uint32_t)p.tables[table + key / (uint32_t)p.page_size];
      }
    };
    auto put_rows = [&](int c0) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint32_t r = ((uint32_t)c0 * kTileKeys + 256 * i + tid) % (uint32_t)p.page_size;
        s_row[256 * i + tid] = page[i] < pages ? (int)(page[i] * (uint32_t)p.page_size + r) : -1;
      }
    };
    look_up(ta);
    if constexpr (!BF)
      c = (direct ? p.scale_log2 : 1.0f) * p.q_size[(int64_t)b * p.hq + min(h, p.hq - 1)];
    // The queries by way of the tiles' LDS, laid out as a tile: head group hg's in
    // slot hg, parts kg NHG .. copied by this wave. (Operands straight from memory,
    // 16 bytes of a row a lane, take the cache 4 times as long, each wave's anew: 32
    // heads, 64 sequences of 512 to 8192 keys 86.5 us a call for 84.2, one of 777
    // 26.7 for 24.7.)
#pragma unroll 1
    for (int i = 0; i < NHG; ++i) {
      const int r = 8 * (kg * NHG + i) + (lane >> 3), at = (lane & 7) ^ swizzle(r);
      const f16* src =
          p.q_lat + ((int64_t)b * p.hq + min(head0 + 32 * hg + r, p.hq - 1)) * width;
      const uint32_t dst = lds + hg * (2 * kTile) + 1024 * (kg * NHG + i);
#pragma unroll 1
      for (int j = 0; j < WP; ++j)
        copy_to_lds<0, 0>(src + 8 * min(8 * j + at, last_piece), dst + j * (2 * kPlane));
    }
    put_rows(ta);
    wait_vmem<0>();
    __syncthreads();
    f16x8 qf[kChunks];
    {
      // (The places are formed here for every sequence: kept through the loop they
      // were spilled, and 50 reloads in turn took 15 us.)
      int k0 = k_place, part = 8 * hh;
      asm volatile("" : "+v"(k0), "+v"(part));
      const f16* t = s_t[hg];
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const f16x8 x =
            *reinterpret_cast<const f16x8*>(t + (k0 ^ 16 * (i & 3)) + kPlane * (i >> 2));
        qf[i] = live && 16 * i + part < width ? x : f16x8{};
      }
    }
    wait_lds();
    __syncthreads();
    f32x16 o[OB];
#pragma unroll
    for (int i = 0; i < OB; ++i) o[i] = f32x16{};
    outputs_settle(o);
    float m = -INFINITY, l = 0.0f;

    for (int c0 = ta; c0 < tb; c0 += kChunkTiles) {
      const int tiles = min(kChunkTiles, tb - c0);
      if (c0 > ta) {
        look_up(c0);
        __syncthreads();  // (everyone is past the chunk before)
        put_rows(c0);
        __syncthreads();
      }
      // Tile `tile` of the chunk into slot `slot` of the wave's ring: this
      // wave's parts, their arena rows in `row`.
      auto copy = [&](const int (&row)[kRows], int slot) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const uint32_t dst =
              lds + (kg * NHG + slot) * (2 * kTile) + 1024 * (hg + NHG * i);
          const f16* src = p.arena + (int64_t)max(row[i], 0) * width;
          auto plane = [&](auto j, auto once) {
            copy_to_lds<128 * j.value, (2 * kPlane - 128) * j.value, once.value>(
                src + 8 * piece(i), dst);
          };
          if (whole && p.once) {
            each_plane([&](auto j) { plane(j, std::true_type{}); });
          } else if (whole) {
            each_plane([&](auto j) { plane(j, std::false_type{}); });
          } else {
#pragma unroll 1
            for (int j = 0; j < WP; ++j)
              copy_to_lds<0, 0>(src + 8 * min(8 * j + piece(i), last_piece), dst + j * (2 * kPlane));
          }
        }
      };
      auto rows_of = [&](int tile, int (&row)[kRows]) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) row[i] = s_row[tile * kTileKeys + part_row(i)];
      };
      // Rows of no key become zeros once they have landed (their weight is 0;
      // zero rows keep 0 * V finite whatever the arena holds).
      auto clean = [&](uint32_t okm, int slot) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          if (okm >> part_row(i) & 1) continue;
          f16* t = s_t[kg * NHG + slot] + 64 * part_row(i) + 8 * (lane & 7);
          for (int j = 0; j < WP; ++j) *reinterpret_cast<f16x8*>(t + j * kPlane) = f16x8{};
        }
      };
      auto math = [&](uint32_t okm, int slot) {
        const f16* t = s_t[kg * NHG + slot];
        // Operands are read kAhead products early (the reads and products
        // would else wait for each other in turn).
        // (The places are formed per tile: kept, they cost 8 registers of the
        // few left beside the queries, and what was spilled for them 8 us.)
        int k0 = k_place, v0 = v_place;
        asm volatile("" : "+v"(k0), "+v"(v0));
        f32x16 s = {};
        f16x8 a[kChunks];
        auto read_k = [&](int i) {
          a[i] = *reinterpret_cast<const f16x8*>(t + (k0 ^ 16 * (i & 3)) + kPlane * (i >> 2));
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) read_k(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          s = mfma16<BF>(a[i], qf[i], s);
          if (i + kAhead < kChunks) read_k(i + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
        f16x8 va[2 * OB];
        auto read_v = [&](int j) {
          const f16* vp = t + kPlane * (j % OB / 2) + 1024 * (j / OB);
          const f16x4 lo = read_tr(vp + (v0 ^ 32 * (j & 1)));
          const f16x4 hi = read_tr(vp + (v0 ^ (16 + 32 * (j & 1))) + 512);
          va[j] = f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
#pragma unroll
        for (int j = 0; j < kAhead; ++j) read_v(j);
        if (!direct) {
#pragma unroll
          for (int v = 0; v < 16; ++v) s[v] *= p.scale_log2;
        }
        if (okm != 0xFFFFFFFFu) {
          const uint32_t see = okm >> (4 * hh);
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (!(see >> (8 * (v / 4) + v % 4) & 1)) s[v] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) top = fmaxf(top, s[v]);
        top = max_halves(top) * c;
        const bool grow = top > m + kSlack;
        if (__ballot(grow)) {
          // (Sums of a lane that has seen no key are zeros: a sequence's first
          // tile scales nothing.)
          const bool seen = __ballot(grow && m != -INFINITY) != 0;
          const float f = grow ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
          m = grow ? top : m;
          l *= f;
          if (seen) {
            outputs_settle(o);
#pragma unroll
            for (int i = 0; i < OB; ++i) {
#pragma unroll
              for (int v = 0; v < 16; ++v) o[i][v] *= f;
              asm volatile("" : "+a"(o[i]));
            }
          }
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        f16x8 pb[2];
#pragma unroll
        for (int v = 0; v < 16; ++v)
          pb[v / 8][v % 8] = round16<BF>(__builtin_amdgcn_exp2f(fmaf(s[v], c, -mu)));
#pragma unroll
        for (int v = 0; v < 16; v += 2) l = add_pair<BF>(pb[v / 8][v % 8], pb[v / 8][v % 8 + 1], l);
        operands_settle(pb);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2 * OB; ++j) {
          mfma_acc<BF>(va[j], pb[j / OB], o[j % OB]);
          if (j + kAhead < 2 * OB) read_v(j + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      const int rounds = (tiles + kGroups - 1) / kGroups;
      // Copies of the first ring - 1 rounds; then per round: this round's rows
      // have landed, everyone is past the round before, whose slot takes the
      // next copies. The rows of those copies and this tile's mask were read a
      // round before.
      constexpr int kFirst = NHG > 1 ? NHG - 1 : 1;
      auto landed = [&](auto later) { wait_vmem<later.value * kRows * WP>(); };  // all but
      // those of `later` tiles
      constexpr int kTwo = NHG > 3 ? 2 : 0, kOne = NHG > 2 ? 1 : 0;
      int row[kRows];
      for (int r = 0; r < min(kFirst, rounds); ++r)
        if (r * kGroups + kg < tiles) {
          rows_of(r * kGroups + kg, row);
          copy(row, r % NHG);
        }
      // (Reads past the last tile stay in the chunk's rows; what they give is
      // not used.)
      constexpr int kLast = kChunkTiles - 1;
      rows_of(min(kFirst * kGroups + kg, kLast), row);
      int key_row = s_row[min(kg, kLast) * kTileKeys + n];
      for (int r = 0; r < rounds; ++r) {
        const int tile = r * kGroups + kg;
        const bool here = tile < tiles;
        const int next = tile + kFirst * kGroups;
        const uint32_t okm = (uint32_t)__ballot(key_row >= 0);
        if (NHG > 3 && tile + 2 * kGroups < tiles)
          landed(std::integral_constant<int, kTwo>{});
        else if (NHG > 2 && tile + kGroups < tiles)
          landed(std::integral_constant<int, kOne>{});
        else
          wait_vmem<0>();
        if (here && okm != 0xFFFFFFFFu) clean(okm, r % NHG);
        if constexpr (NHG > 1) {
          __syncthreads();
          if (next < tiles) copy(row, (r + kFirst) % NHG);
        }
        key_row = s_row[min(tile + kGroups, kLast) * kTileKeys + n];
        if constexpr (NHG > 1) rows_of(min(next + kGroups, kLast), row);
        if (here) math(okm, r % NHG);
        wait_lds();
        if constexpr (NHG == 1) {
          if (next < tiles) copy(row, 0);
          rows_of(min(next + kGroups, kLast), row);
        }
      }
    }

    // One partial of the wave groups' sums: each scaled to their common max,
    // kJoin dims a round through LDS, added and written along the rows.
    outputs_settle(o);
    l += __shfl_xor(l, 32);
    if (hh == 0) s_ml[w][n] = make_float2(m, l);
    __syncthreads();
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) mm = fmaxf(mm, s_ml[g * NHG + hg][n].x);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float2 x = s_ml[g * NHG + hg][n];
      if (x.x != -INFINITY) ll += x.y * __builtin_amdgcn_exp2f(x.x - mm);
    }
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mm);
    const int64_t slot = (int64_t)blockIdx.x + b;
    if (kg == 0 && hh == 0 && live) p.part_ml[slot * p.hq + h] = make_float2(mm, ll);
    float* join = reinterpret_cast<float*>(&s_t[0][0]);
#pragma unroll
    for (int q = 0; q < 32 * OB / kJoin; ++q) {
      const int d0 = kJoin * q;
      if (d0 >= p.latent) break;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kJoin / 32; ++i) {
        f32x16& x = o[kJoin / 32 * q + i];
        asm volatile("" : "+a"(x));
        float* at = join + (32 * w + n) * kPitch + 32 * i + 4 * hh;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(at + 8 * g) =
              make_float4(x[4 * g] * f, x[4 * g + 1] * f, x[4 * g + 2] * f, x[4 * g + 3] * f);
      }
      __syncthreads();
      constexpr int kWide = kJoin / 4;  // threads along a row
#pragma unroll 4
      for (int i = 0; i < 32 * NHG * kWide / 256; ++i) {
        const int hd = i * (256 / kWide) + tid / kWide, d = 4 * (tid % kWide);
        float4 x = *reinterpret_cast<const float4*>(join + hd * kPitch + d);
#pragma unroll
        for (int g = 1; g < kGroups; ++g) {
          const float4 y =
              *reinterpret_cast<const float4*>(join + (32 * NHG * g + hd) * kPitch + d);
          x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        if (head0 + hd < p.hq && d0 + d < p.latent)
          *reinterpret_cast<float4*>(p.part_o + (slot * p.hq + head0 + hd) * p.latent + d0 + d) = x;
      }
    }
    __syncthreads();
  }
}

// Joins the partials of each sequence and projects the result: out[b, h] = D_h
// o / sum. A workgroup has one head and up to 32 sequences. D_h's rows are
// under way while the partials are joined: a wave has the rows of 32 value dims
// over half the latent.
// A wave joins a whole row of partials (512 dims) of one sequence, several
// waves share a sequence's partials where there are few sequences. The joined
// latents go to LDS as two 16-bit numbers each (the value and what its rounding
// left), so the product loses nothing that the output's rounding would show. 64
// sequences of 128 heads 22 us (84 MB of partials, 3.8 TB/s), one of 16 heads 8 us
// (six reads and meetings in turn).
template <bool BF>
__global__ __launch_bounds__(512, 2) void latent_merge_kernel(const LatentDecodeParams p) {
  constexpr int kWaves = 8;
  constexpr int kRow = kMaxLatent + 8;        // halves between sequences
  constexpr int kSlices = 8;                  // loads of 4 rows for a wave's 32
  __shared__ __align__(16) f16 s_hi[32 * kRow];
  __shared__ __align__(16) f16 s_lo[32 * kRow];
  __shared__ __align__(16) float s_part[kWaves][kMaxLatent];
  __shared__ __align__(1024) f16 s_d[kWaves][32 * 128];
  const int tid = threadIdx.x, w = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 31, hh = lane >> 5;
  const int h = blockIdx.x, b0 = blockIdx.y * p.merge_batch;
  const int count = min(p.merge_batch, p.batch - b0);
  const int v0 = 32 * (w & 3), k0 = (w >> 2) * (kMaxLatent / 2);
  // Lane i: the stream's place before sequence b0 + i, the ranges of its units
  // on either side.
  const uint32_t place = (uint32_t)p.prefix[b0 + min(lane, count)];
  const uint32_t per =
      max(1u, ((uint32_t)scalar_load(p.prefix, p.batch) + p.groups - 1) / (uint32_t)p.groups);
  const int range_in = (int)((place + kSequenceTiles) / per), range_end = (int)((place - 1) / per);
  const int share = count >= 8 ? 1 : count >= 4 ? 2 : count >= 2 ? 4 : 8;  // waves a sequence
  const int d = 8 * lane;
  // A wave's slice of D_h: rows v0 .. v0 + 31, dims k0 .. k0 + 255, in two halves
  // of 128. A load moves 256 bytes of 4 rows (lanes side by side read 16 bytes
  // side by side: a product's operand straight from memory, 32 rows an
  // instruction, takes the cache 4 times as long); row r has piece p at place
  // p ^ (r % 16).
  auto weights_at = [&](int i, int from) {
    const int r = 4 * i + (lane >> 4), piece = (lane & 15) ^ (r & 15);
    return reinterpret_cast<const f16x8*>(
        p.kv_b +
        ((int64_t)h * (p.nope + p.value) + p.nope + min(v0 + r, p.value - 1)) * p.latent +
        min(k0 + from + 8 * piece, p.latent - 8));
  };
  const uint32_t lds = uniform(lds_address(&s_d[w][0]));
  f16x8 a[kSlices];
  for (int r0 = 0; r0 < count; r0 += kWaves / share) {
    const int r = r0 + w / share, part = w % share;
    const bool have = r < count;
    const int b = b0 + (have ? r : 0);
    const int at = have ? r : 0;
    const bool some = __builtin_amdgcn_readlane(place, at + 1) !=
                      __builtin_amdgcn_readlane(place, at);  // it has keys
    const int g0 = __builtin_amdgcn_readlane(range_in, at);
    const int slots = have && some ? __builtin_amdgcn_readlane(range_end, at + 1) - g0 + 1 : 0;
    const float2* ml = p.part_ml + ((int64_t)g0 + b) * p.hq + h;
    const float* po = p.part_o + (((int64_t)g0 + b) * p.hq + h) * p.latent;
    // This wave's partials part + share i, kEach of them under way, the first
    // before what they weigh is known.
    constexpr int kEach = 8;
    float4 x[kEach][2];
    auto load = [&](int g) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        x[j][0] = x[j][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (g + share * j < slots && d < p.latent) {
          const float4* src =
              reinterpret_cast<const float4*>(po + (int64_t)(g + share * j) * p.hq * p.latent + d);
          x[j][0] = src[0];
          x[j][1] = src[1];
        }
      }
    };
    // A lane looks at every 64th partial's maximum and sum.
    float2 mine = make_float2(-INFINITY, 0.0f);
    if (lane < slots) mine = ml[(int64_t)lane * p.hq];
    load(part);
    if (r0 == 0) {  // (loads return in their order: behind the first partials)
      auto copy = [&](auto i) __attribute__((always_inline)) {
        copy_to_lds<0, decltype(i)::value * 1024>(weights_at(i, 0), lds);
      };
      each(copy, std::make_integer_sequence<int, kSlices>{});
#pragma unroll
      for (int i = 0; i < kSlices; ++i) a[i] = *weights_at(i, 128);
    }
    float top = mine.x;
    for (int g = lane + 64; g < slots; g += 64) top = fmaxf(top, ml[(int64_t)g * p.hq].x);
#pragma unroll
    for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    float sum = 0.0f, f = 0.0f, acc[8] = {};
    for (int base = 0; base < slots; base += share * kEach) {
      if (base % 64 == 0) {  // (share * kEach divides 64)
        f = 0.0f;
        if (base + lane < slots && top != -INFINITY) {
          const float2 y = base ? ml[(int64_t)(base + lane) * p.hq] : mine;
          f = y.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y.x - top);
          sum = fmaf(y.y, f, sum);
        }
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        // (A partial without a key holds zeros: nothing to leave out.)
        const float fg = __shfl(f, (base + part + share * j) % 64);
        acc[0] = fmaf(x[j][0].x, fg, acc[0]);
        acc[1] = fmaf(x[j][0].y, fg, acc[1]);
        acc[2] = fmaf(x[j][0].z, fg, acc[2]);
        acc[3] = fmaf(x[j][0].w, fg, acc[3]);
        acc[4] = fmaf(x[j][1].x, fg, acc[4]);
        acc[5] = fmaf(x[j][1].y, fg, acc[5]);
        acc[6] = fmaf(x[j][1].z, fg, acc[6]);
        acc[7] = fmaf(x[j][1].w, fg, acc[7]);
      }
      if (base + share * kEach < slots) load(base + share * kEach + part);
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    if (share > 1) {
      if (r0) __syncthreads();
      *reinterpret_cast<float4*>(&s_part[w][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(&s_part[w][d + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      __syncthreads();
      if (part == 0)
        for (int i = 1; i < share; ++i) {
          const float4 y = *reinterpret_cast<const float4*>(&s_part[w + i][d]);
          const float4 z = *reinterpret_cast<const float4*>(&s_part[w + i][d + 4]);
          acc[0] += y.x, acc[1] += y.y, acc[2] += y.z, acc[3] += y.w;
          acc[4] += z.x, acc[5] += z.y, acc[6] += z.z, acc[7] += z.w;
        }
    }
    if (part || !have || d >= p.latent) continue;
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    f16x8 hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = acc[j] * inv;
      hi[j] = round16<BF>(x);
      lo[j] = round16<BF>(x - widen<BF>(hi[j]));
    }
    *reinterpret_cast<f16x8*>(&s_hi[r * kRow + d]) = hi;
    *reinterpret_cast<f16x8*>(&s_lo[r * kRow + d]) = lo;
  }
  wait_vmem<0>();
  __syncthreads();
  const bool have = n < count;  // (other columns hold anything)
  f32x16 acc = {}, rest = {};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half) {  // (a wave's own reads and writes of LDS keep their order)
#pragma unroll
      for (int i = 0; i < kSlices; ++i)
        *reinterpret_cast<f16x8*>(&s_d[w][512 * i + 8 * lane]) = a[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + 128 * half + 16 * i + 8 * hh, at = n * kRow + min(k, p.latent - 8);
      f16x8 x = *reinterpret_cast<const f16x8*>(&s_d[w][128 * n + 8 * ((2 * i + hh) ^ (n & 15))]);
      f16x8 hi = *reinterpret_cast<const f16x8*>(&s_hi[at]);
      f16x8 lo = *reinterpret_cast<const f16x8*>(&s_lo[at]);
      if (k >= p.latent) x = hi = lo = f16x8{};
      acc = mfma16<BF>(x, hi, acc);
      rest = mfma16<BF>(x, lo, rest);
    }
  }
  // The two halves of the latent.
  float* join = &s_part[0][0];
  __syncthreads();
  if (w >= 4) {
#pragma unroll
    for (int v = 0; v < 16; ++v) join[((w - 4) * 16 + v) * 64 + lane] = acc[v] + rest[v];
  }
  __syncthreads();
  if (w >= 4 || !have) return;
  f16* dst = p.out + ((int64_t)(b0 + n) * p.hq + h) * p.value + v0 + 4 * hh;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (v0 + 8 * g >= p.value) break;
    f16x4 y;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      y[t] = round16<BF>(acc[4 * g + t] + rest[4 * g + t] + join[(w * 16 + 4 * g + t) * 64 + lane]);
    *reinterpret_cast<f16x4*>(dst + 8 * g) = y;
  }
}

// ---------------------------------------------------------------------------
// Host.

constexpr int kMaxBatch = 8184;
// Rows of so many bytes go past the caches: a quarter of what an MI355X's last
// cache holds, so that from four layers on it would not have them at the next step.
// (32 sequences of 4000 keys, 147 MB a layer, us a call kept and past: 8 layers in
// turn, 16 heads 57 and 53, 64 heads 67 and 61; one layer again and again 55 and 57,
// 63 and 67. Widths below the kernel's gain nothing and stay.)
constexpr int64_t kOnceBytes = (int64_t)64 << 20;

// Waves side by side over heads: as many as the heads fill, so that a tile is
// copied once for all of them. (64 sequences of 512 to 8192 keys, us a call with 1,
// 2 and 4: 16 heads 79, 84, 100; 32 heads 87, 89, 99; 64 heads 110, 101, 108; 128
// heads 162, 143, 131.)
int waves_over_heads(int q_heads) { return q_heads <= 32 ? 1 : q_heads <= 64 ? 2 : 4; }

struct Plan {
  int head_groups;  // grid y
  int groups;       // ranges of the stream: grid x
  size_t q_lat, q_size, prefix, part_ml, part_o, bytes;
};

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

Plan plan_for(int batch, int q_heads, int latent, int rope, int page_size, int table_stride,
              int longest) {
  Plan r;
  const int nhg = waves_over_heads(q_heads);
  r.head_groups = (q_heads + 32 * nhg - 1) / (32 * nhg);
  const int64_t cap = (int64_t)page_size * table_stride;
  const int64_t keys = std::max<int64_t>(1, std::min<int64_t>(longest, cap));
  const int64_t tiles = (int64_t)batch * ((keys + kTileKeys - 1) / kTileKeys + kSequenceTiles);
  // A workgroup has a tile for each of its wave groups at least.
  const int64_t most = std::max(1, kMaxGroups / r.head_groups);
  r.groups = (int)std::max<int64_t>(1, std::min(most, (tiles + 4 / nhg - 1) / (4 / nhg)));
  const size_t slots = (size_t)r.groups + batch;
  size_t at = 0;
  r.q_lat = at;
  at = up256(at + (size_t)batch * q_heads * (latent + rope) * 2);
  r.q_size = at;
  at = up256(at + (size_t)batch * q_heads * 4);
  r.prefix = at;
  at = up256(at + (size_t)(batch + 1) * 4);
  r.part_ml = at;
  at = up256(at + slots * q_heads * 8);
  r.part_o = at;
  r.bytes = up256(at + slots * q_heads * latent * 4);
  return r;
}

template <int WP, int OB, bool BF>
const void* decode_kernel(int nhg) {
  switch (nhg) {
    case 1: return (const void*)latent_decode_kernel<WP, OB, 1, BF>;
    case 2: return (const void*)latent_decode_kernel<WP, OB, 2, BF>;
    default: return (const void*)latent_decode_kernel<WP, OB, 4, BF>;
  }
}

// The kernel of 256 latent dims (and 64 rotary ones) for rows that it holds: two
// thirds of the copies and products. (256 + 32 dims, the sequences above, us a call
// with it and with the wide one: 14 heads 56 and 64, 128 heads 77 and 100.)
template <bool BF>
const void* decode_kernel_for(int nhg, int latent) {
  return latent <= 256 ? decode_kernel<5, 8, BF>(nhg) : decode_kernel<9, 16, BF>(nhg);
}

int check_decode(int32_t batch, int32_t q_heads, int32_t latent_dim, int32_t rope_dim,
                 int32_t nope_dim, int32_t value_dim, int32_t page_size, int32_t table_stride) {
  const int rc = check_shape(q_heads, latent_dim, rope_dim, nope_dim, value_dim);
  if (rc != PDA_OK) return rc;
  if (batch < 0 || batch > kMaxBatch || page_size <= 0 || table_stride <= 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "batch=%d (at most %d) page_size=%d table_stride=%d",
                batch, kMaxBatch, page_size, table_stride);
  const int64_t keys = std::min<int64_t>((int64_t)page_size * table_stride, INT32_MAX);
  if ((int64_t)batch * ((keys + kTileKeys - 1) / kTileKeys + kSequenceTiles) > INT32_MAX)
    return fail(PDA_ERR_TOO_LONG, "batch x keys exceeds the tile stream (2^31 tiles of %d keys)",
                kTileKeys);
  return PDA_OK;
}

int latent_append(const void* q, void* q_out, const void* latent, int64_t latent_stride,
                  const void* k_rope, int64_t k_stride, const void* norm_weight, float eps,
                  void* arena, const int32_t* positions, const int32_t* rows, int32_t n,
                  int32_t q_heads, int32_t latent_dim, int32_t rope_dim, int32_t nope_dim,
                  int64_t arena_rows, const float* inv_freq, bool bf, void* stream) {
  const bool queries = q != nullptr || q_out != nullptr;
  const int rc = check_shape(queries ? q_heads : 1, latent_dim, rope_dim, queries ? nope_dim : 8, 8);
  if (rc != PDA_OK) return rc;
  if (n < 0 || arena_rows < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "n=%d arena_rows=%lld", n, (long long)arena_rows);
  if (n == 0) return ok();
  if (queries && (!q || !q_out)) return fail(PDA_ERR_INVALID_ARGUMENT, "q and q_out go together");
  const bool write = latent || arena || rows || (k_rope && rope_dim);
  if (write && (!latent || !arena || !rows || (rope_dim && !k_rope)))
    return fail(PDA_ERR_INVALID_ARGUMENT, "latent, k_rope, arena and rows go together");
  if (!queries && !write) return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (inv_freq && !positions)
    return fail(PDA_ERR_INVALID_ARGUMENT, "the rotation needs positions");
  if (write && (latent_stride < latent_dim || latent_stride % 8 ||
                (rope_dim && (k_stride < rope_dim || k_stride % 8))))
    return fail(PDA_ERR_ALIGNMENT, "row strides must hold a row and be multiples of 8 elements");
  if (norm_weight && !(eps >= 0.0f && eps < INFINITY))
    return fail(PDA_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  const uintptr_t mis = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)latent |
                        (rope_dim ? (uintptr_t)k_rope : 0) | (uintptr_t)arena |
                        (uintptr_t)norm_weight;
  if (mis & 15) return fail(PDA_ERR_ALIGNMENT, "16-bit buffers must be 16-byte aligned");
  if (((uintptr_t)positions | (uintptr_t)rows | (uintptr_t)inv_freq) & 3)
    return fail(PDA_ERR_ALIGNMENT, "positions, rows and inv_freq must be 4-byte aligned");
  LatentAppendParams prm;
  prm.q = static_cast<const f16*>(q);
  prm.q_out = static_cast<f16*>(q_out);
  prm.c = write ? static_cast<const f16*>(latent) : nullptr;
  prm.k = static_cast<const f16*>(k_rope);
  prm.norm = static_cast<const f16*>(norm_weight);
  prm.arena = static_cast<f16*>(arena);
  prm.positions = positions;
  prm.rows = rows;
  prm.inv_freq = rope_dim ? inv_freq : nullptr;
  prm.c_stride = latent_stride;
  prm.k_stride = k_stride;
  prm.arena_rows = arena_rows;
  prm.n = n;
  prm.hq = q_heads;
  prm.latent = latent_dim;
  prm.rope = rope_dim;
  prm.nope = nope_dim;
  prm.head_groups = (q_heads + kAppendHeads - 1) / kAppendHeads;
  prm.eps = eps;
  const int64_t blocks =
      (write ? ((int64_t)n + 3) / 4 : 0) + (queries ? (int64_t)n * prm.head_groups : 0);
  if (blocks > kMaxGrid)
    return fail(PDA_ERR_INVALID_ARGUMENT, "tokens x query heads beyond one launch's workgroups");
  void* args[] = {&prm};
  const hipError_t err =
      hipLaunchKernel(bf ? (const void*)latent_append_kernel<true>
                         : (const void*)latent_append_kernel<false>,
                      dim3((unsigned)blocks), dim3(256), args, 0, static_cast<hipStream_t>(stream));
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

int latent_decode(const void* queries, const void* arena, const void* kv_b, const int32_t* tables,
                  const int32_t* lengths, void* out, int32_t batch, int32_t q_heads,
                  int32_t latent_dim, int32_t rope_dim, int32_t nope_dim, int32_t value_dim,
                  int32_t page_size, int32_t table_stride, int64_t arena_rows, int32_t longest,
                  float scale, bool bf, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_decode(batch, q_heads, latent_dim, rope_dim, nope_dim, value_dim, page_size,
                              table_stride);
  if (rc != PDA_OK) return rc;
  if (batch == 0) return ok();
  if (!queries || !arena || !kv_b || !tables || !lengths || !out)
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (arena_rows < page_size || arena_rows > INT32_MAX)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld: a whole page at least, below 2^31",
                (long long)arena_rows);
  if (!(scale == scale) || isinf(scale))
    return fail(PDA_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (((uintptr_t)queries | (uintptr_t)arena | (uintptr_t)kv_b | (uintptr_t)out) & 15)
    return fail(PDA_ERR_ALIGNMENT, "16-bit buffers must be 16-byte aligned");
  if (((uintptr_t)tables | (uintptr_t)lengths) & 3)
    return fail(PDA_ERR_ALIGNMENT, "tables and lengths must be 4-byte aligned");
  const Plan plan =
      plan_for(batch, q_heads, latent_dim, rope_dim, page_size, table_stride, longest);
  if (!workspace || workspace_bytes < plan.bytes)
    return fail(PDA_ERR_WORKSPACE, "a workspace of %zu bytes is needed (got %zu)", plan.bytes,
                workspace ? workspace_bytes : (size_t)0);
  if ((uintptr_t)workspace & 255)
    return fail(PDA_ERR_ALIGNMENT, "the workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  const int nhg = waves_over_heads(q_heads);
  LatentDecodeParams prm;
  prm.q = static_cast<const f16*>(queries);
  prm.kv_b = static_cast<const f16*>(kv_b);
  prm.arena = static_cast<const f16*>(arena);
  prm.tables = tables;
  prm.lengths = lengths;
  prm.out = static_cast<f16*>(out);
  prm.q_lat = reinterpret_cast<f16*>(ws + plan.q_lat);
  prm.q_size = reinterpret_cast<float*>(ws + plan.q_size);
  prm.prefix = reinterpret_cast<int32_t*>(ws + plan.prefix);
  prm.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
  prm.part_o = reinterpret_cast<float*>(ws + plan.part_o);
  prm.arena_pages = arena_rows / page_size;
  prm.table_stride = table_stride;
  prm.page_size = page_size;
  prm.batch = batch;
  prm.hq = q_heads;
  prm.latent = latent_dim;
  prm.rope = rope_dim;
  prm.nope = nope_dim;
  prm.value = value_dim;
  prm.groups = plan.groups;
  prm.scale_log2 = scale * kLog2e;
  // Sequences a merge workgroup takes: fewer while the CUs are not all used.
  prm.once = (int64_t)batch * longest * (latent_dim + rope_dim) * 2 > kOnceBytes;
  // As many sequences a merging workgroup as leave one for each CU, 32 at most, the
  // columns of a product. (64 sequences, us a call with 8, with 32 and by the rule: 16
  // heads 78, 83, 78; 128 heads 147, 129, 129.)
  prm.merge_batch = 32;
  while (prm.merge_batch > 1 &&
         (int64_t)q_heads * ((batch + prm.merge_batch - 1) / prm.merge_batch) < kMaxGroups)
    prm.merge_batch /= 2;
  void* args[] = {&prm};
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  hipError_t err = hipLaunchKernel(
      bf ? (const void*)latent_absorb_kernel<true> : (const void*)latent_absorb_kernel<false>,
      dim3((latent_dim + 127) / 128, q_heads, (batch + 31) / 32), dim3(256), args, 0, hs);
  if (err == hipSuccess)
    err = hipLaunchKernel(bf ? decode_kernel_for<true>(nhg, latent_dim)
                             : decode_kernel_for<false>(nhg, latent_dim),
                          dim3(plan.groups, plan.head_groups), dim3(256), args, 0, hs);
  if (err == hipSuccess)
    err = hipLaunchKernel(
        bf ? (const void*)latent_merge_kernel<true> : (const void*)latent_merge_kernel<false>,
        dim3(q_heads, (batch + prm.merge_batch - 1) / prm.merge_batch), dim3(512), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

}  // namespace

extern "C" {

int pda_latent_append(const void* q, void* q_out, const void* latent, int64_t latent_stride,
                      const void* k_rope, int64_t k_stride, const void* norm_weight, float eps,
                      void* arena, const int32_t* positions, const int32_t* rows, int32_t n,
                      int32_t q_heads, int32_t latent_dim, int32_t rope_dim, int32_t nope_dim,
                      int64_t arena_rows, const float* inv_freq, void* stream) {
  return latent_append(q, q_out, latent, latent_stride, k_rope, k_stride, norm_weight, eps, arena,
                       positions, rows, n, q_heads, latent_dim, rope_dim, nope_dim, arena_rows,
                       inv_freq, false, stream);
}

int pda_latent_append_bf16(const void* q, void* q_out, const void* latent, int64_t latent_stride,
                           const void* k_rope, int64_t k_stride, const void* norm_weight,
                           float eps, void* arena, const int32_t* positions, const int32_t* rows,
                           int32_t n, int32_t q_heads, int32_t latent_dim, int32_t rope_dim,
                           int32_t nope_dim, int64_t arena_rows, const float* inv_freq,
                           void* stream) {
  return latent_append(q, q_out, latent, latent_stride, k_rope, k_stride, norm_weight, eps, arena,
                       positions, rows, n, q_heads, latent_dim, rope_dim, nope_dim, arena_rows,
                       inv_freq, true, stream);
}

int pda_latent_decode_workspace_bytes(int32_t batch, int32_t q_heads, int32_t latent_dim,
                                      int32_t rope_dim, int32_t page_size, int32_t table_stride,
                                      int32_t longest, size_t* bytes) {
  const int rc = check_decode(batch, q_heads, latent_dim, rope_dim, 8, 8, page_size, table_stride);
  if (rc != PDA_OK) return rc;
  if (!bytes) return fail(PDA_ERR_INVALID_ARGUMENT, "null result pointer");
  *bytes = batch == 0 ? 0
                      : plan_for(batch, q_heads, latent_dim, rope_dim, page_size, table_stride,
                                 longest)
                            .bytes;
  return ok();
}

int pda_latent_decode_attention(const void* queries, const void* arena, const void* kv_b,
                                const int32_t* tables, const int32_t* lengths, void* out,
                                int32_t batch, int32_t q_heads, int32_t latent_dim,
                                int32_t rope_dim, int32_t nope_dim, int32_t value_dim,
                                int32_t page_size, int32_t table_stride, int64_t arena_rows,
                                int32_t longest, float scale, void* workspace,
                                size_t workspace_bytes, void* stream) {
  return latent_decode(queries, arena, kv_b, tables, lengths, out, batch, q_heads, latent_dim,
                       rope_dim, nope_dim, value_dim, page_size, table_stride, arena_rows, longest,
                       scale, false, workspace, workspace_bytes, stream);
}

int pda_latent_decode_attention_bf16(const void* queries, const void* arena, const void* kv_b,
                                     const int32_t* tables, const int32_t* lengths, void* out,
                                     int32_t batch, int32_t q_heads, int32_t latent_dim,
                                     int32_t rope_dim, int32_t nope_dim, int32_t value_dim,
                                     int32_t page_size, int32_t table_stride, int64_t arena_rows,
                                     int32_t longest, float scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  return latent_decode(queries, arena, kv_b, tables, lengths, out, batch, q_heads, latent_dim,
                       rope_dim, nope_dim, value_dim, page_size, table_stride, arena_rows, longest,
                       scale, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
