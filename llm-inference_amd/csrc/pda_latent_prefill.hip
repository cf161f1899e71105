// Latent attention for MI355X (gfx950): prefill attention of a prompt's chunk
// in the expanded form, C-ABI in pda.h (pda_latent_prefill_attention). No
// reference counterpart.
//
// With many queries per key it is cheaper to project every head's keys and
// values out of the latents once, 2 latent (nope + value) operations a key and
// head, and to attend in nope + rope and value dims, than to attend in the
// latent (2 latent + rope dims a query, key and head): 320 against 1088
// operations a pair at 512 + 64 and 128 dims, so the projection's 262 thousand
// are paid for from some 170 queries on. Two launches per group of heads:
// latent_expand_kernel (a matrix product over the gathered rows) and
// latent_prefill_kernel (causal attention, a key range split over workgroups
// and merged where a chunk has few).

#include <algorithm>

#include "pda_latent.h"

namespace {

using namespace pda_latent;
using pda_internal::fail;
using pda_internal::ok;

constexpr int kQueries = 128;   // queries per workgroup
constexpr int kKeys = 64;       // keys per tile
constexpr int kTokenTile = 128; // tokens an expanding workgroup keeps
constexpr int kMaxSplits = 64;
constexpr float kSlack = 8.0f;
constexpr int kXcds = 8;
constexpr int kCus = 256;
constexpr int kSlots = 2 * kCus;  // workgroups resident on an MI355X, two a CU

struct PrefillParams {
  const f16* q;         // [count, hq, nope + rope]
  const f16* arena;     // [arena_rows, latent + rope]
  const f16* kv_b;      // [hq, nope + value, latent]
  const int32_t* table;
  f16* out;             // [count, hq, value]
  f16* keys;            // [heads of the group, span, kdim] expanded
  f16* values;          // [heads of the group, span, vdim]
  f16* rope_keys;       // [span, rdim]
  uint64_t* seen;       // [span / 64] bits of keys that have a row
  float* part_o;        // [splits, count, hq, value]
  float2* part_ml;      // [splits, count, hq]
  int64_t arena_pages;
  int32_t table_len;
  int32_t page_size;
  int32_t start;
  int32_t count;
  int32_t span;         // start + count, up to a whole tile
  int32_t hq;
  int32_t head0;        // first head of the group
  int32_t heads;        // heads of the group
  int32_t latent;
  int32_t rope;
  int32_t nope;
  int32_t value;
  int32_t kdim, vdim, rdim;  // widths of the expanded rows (planes of 32)
  int32_t tiles;        // query tiles
  int32_t paired;       // two query tiles of a head a workgroup
  int32_t splits;
  int32_t shares;       // workgroups that share a token tile's projected dims
  float scale_log2;
};

// ---------------------------------------------------------------------------
// Expansion.

// keys[h, t] = U_h c_t, values[h, t] = D_h c_t, rounded to the element type, as a
// cache of keys and values per head would hold them (in bf16 that moves the result
// by 1.0e-3 and 1.2e-3 of its 2-norm, beside 1.7e-3 for its own rounding): a matrix
// product in which the tokens stay and the projections stream. A wave
// keeps 32 tokens' whole latents as operands (128 registers at 512 dims, gathered
// from the pages once); the workgroup walks the projected dims of its heads 32 at
// a time through two LDS blocks, each read once by every wave. Two workgroups a
// CU, so that one's products run beside the other's waits. (Two token blocks a
// wave, which halve the LDS reads, and one workgroup a CU were slower: 128 heads,
// 512 tokens 63 us a call against 59, 16 heads, 256 at 30000 272 against 257.)
// The next block's copies and the last one's stores go out among the products:
// issued together they held the wave for as long as the products. 16 heads of
// 128 + 128 dims, 8289 tokens 49 us, 128 heads, 4096 tokens 150 to 162 us by the
// clock (0.85 to 0.92 PFLOP/s); the products and the copies' rate into LDS bound it
// about alike.
// Results are stored a block late. Tokens without a row are zeros from the start.
// The workgroups of the group's first heads also gather the rotary keys and the
// mask of keys that have a row. PL: planes of 64 latent dims.
template <int PL, bool BF>
__global__ __launch_bounds__(256, 2) void latent_expand_kernel(const PrefillParams p) {
  constexpr int kPlane = 32 * 64;  // halves of 64 latent dims of a block
  constexpr int kPlanes = PL;
  constexpr int kChunks = 4 * kPlanes;
  constexpr int kPitch = 40;        // halves of a token's 32 results
  __shared__ __align__(1024) f16 s_w[2][kPlanes * kPlane];
  __shared__ __align__(16) f16 s_out[4][32 * kPitch];
  __shared__ int s_row[kTokenTile];
  const int tid = threadIdx.x, w = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 31, hh = lane >> 5;
  const int outs = p.nope + p.value;
  const int share = blockIdx.x % p.shares;
  const int t0 = (int)(blockIdx.x / p.shares) * kTokenTile;
  const int width = p.latent + p.rope;
  for (int i = tid; i < kTokenTile; i += 256) {
    const int t = t0 + i;
    int row = -1;
    if (t < p.start + p.count) {
      const uint32_t pi = (uint32_t)t / (uint32_t)p.page_size;
      if (pi < (uint32_t)p.table_len) {
        const uint32_t page = (uint32_t)p.table[pi];
        if ((int64_t)page < min(p.arena_pages, (int64_t)INT32_MAX))
          row = (int)(page * (uint32_t)p.page_size + (t - pi * p.page_size));
      }
    }
    s_row[i] = row;
    if (share == 0) {
      const uint64_t have = __ballot(row >= 0);
      if ((tid & 63) == 0 && t < p.span) p.seen[t / 64] = have;
    }
  }
  __syncthreads();
  // The group's blocks of 32 projected dims (a head's nope dims, then its value
  // dims, each to a whole block), shared out evenly.
  const int nope_blocks = (p.nope + 31) / 32, each_head = nope_blocks + (p.value + 31) / 32;
  const int64_t every = (int64_t)p.heads * each_head;
  const int b0 = uniform((int)(every * share / p.shares));
  const int b1 = uniform((int)(every * (share + 1) / p.shares));

  // Copies: an instruction moves 128 bytes of 8 projection rows, the wave's. Past
  // the latent's end they repeat its last piece (the tokens are zeros there),
  // past a head's part its last row (not used).
  const int my_row = 8 * w + (lane >> 3);
  const int piece = (lane & 7) ^ swizzle(my_row);
  const int last_piece = p.latent / 8 - 1;
  const uint32_t lds = uniform(lds_address(&s_w[0][0]));
  struct Block {
    int h, part;
  };
  auto after = [&](Block x) {
    return x.part + 1 < each_head ? Block{x.h, x.part + 1} : Block{x.h + 1, 0};
  };
  auto is_value = [&](Block x) { return x.part >= nope_blocks; };
  auto dim_of = [&](Block x) { return 32 * (is_value(x) ? x.part - nope_blocks : x.part); };
  auto source = [&](Block x) {
    const int size = is_value(x) ? p.value : p.nope;
    return p.kv_b + ((int64_t)(p.head0 + x.h) * outs + (is_value(x) ? p.nope : 0) +
                     min(dim_of(x) + my_row, size - 1)) *
                        p.latent;
  };
  auto copy = [&](const f16* src, int to, int j) __attribute__((always_inline)) {
    copy_to_lds<0, 0>(src + 8 * min(8 * j + piece, last_piece),
                      lds + to * (2 * kPlanes * kPlane) + 1024 * w + j * (2 * kPlane));
  };
  int w_lane[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w_lane[i] = 64 * n + 8 * ((2 * i + hh) ^ swizzle(n));
  // The wave's tokens, half the planes at a time by way of its quarter of the
  // ring: as for the projections an instruction moves 128 bytes of 8 rows.
  // (Fragments straight from memory, 16 bytes of a row a lane, take the cache 4
  // times as long: 16 thousand cycles a CU at 512 dims.)
  constexpr int kHalf = kPlanes / 2;
  f16x8 tok[kChunks];
  const bool have = s_row[32 * w + n] >= 0;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 3), at = (lane & 7) ^ swizzle(r);
      const f16* src = p.arena + (int64_t)max(s_row[32 * w + r], 0) * width;
#pragma unroll
      for (int j = 0; j < kHalf; ++j)
        copy_to_lds<0, 0>(src + 8 * min(8 * (kHalf * half + j) + at, last_piece),
                          lds + (w * kHalf + j) * (2 * kPlane) + 1024 * i);
    }
    wait_vmem<0>();
    asm volatile("" ::: "memory");  // (no barrier: the wave's own copies and reads)
#pragma unroll
    for (int c = 0; c < kChunks / 2; ++c) {
      const int k = 16 * (kChunks / 2 * half + c) + 8 * hh;
      const f16x8 x = *reinterpret_cast<const f16x8*>(
          &s_w[0][0] + (w * kHalf + (c >> 2)) * kPlane + w_lane[c & 3]);
      tok[kChunks / 2 * half + c] = have && k < p.latent ? x : f16x8{};
    }
    wait_lds();
  }
  __syncthreads();
  Block now = {b0 / each_head, b0 % each_head};
  if (b0 < b1) {
    const f16* src = source(now);
#pragma unroll
    for (int j = 0; j < kPlanes; ++j) copy(src, 0, j);
  }
  if (share == 0) {
    const int pieces = p.rdim / 8;
    for (int i = tid; i < kTokenTile * pieces; i += 256) {
      const int r = i / pieces, j = i - r * pieces;
      if (t0 + r >= p.span) break;
      f16x8 x = {};
      if (s_row[r] >= 0 && 8 * j < p.rope)
        x = *reinterpret_cast<const f16x8*>(p.arena + (int64_t)s_row[r] * width + p.latent + 8 * j);
      *reinterpret_cast<f16x8*>(p.rope_keys + (int64_t)(t0 + r) * p.rdim + 8 * j) = x;
    }
  }
  // A block's results (32 dims of the wave's tokens), by rows from the wave's
  // part of LDS: 64 bytes a row. The expanded rows hold whole blocks, so every
  // dim of it is stored, also those past the head's part (keys are zeros there,
  // which the queries' zeros meet).
  f16* so = s_out[w];
  auto load_out = [&](int j) {
    return *reinterpret_cast<const f16x8*>(so + (16 * j + (lane >> 2)) * kPitch + 8 * (lane & 3));
  };
  auto store = [&](Block x, int j, const f16x8& y) __attribute__((always_inline)) {
    f16* base = is_value(x) ? p.values + (int64_t)x.h * p.span * p.vdim
                            : p.keys + (int64_t)x.h * p.span * p.kdim;
    const int pitch = is_value(x) ? p.vdim : p.kdim;
    const int64_t t = t0 + 32 * w + 16 * j + (lane >> 2);
    if (t >= p.span) return;
    *reinterpret_cast<f16x8*>(base + t * pitch + dim_of(x) + 8 * (lane & 3)) = y;
    // (Planes of the keys that no block fills.)
    if (x.part == nope_blocks - 1 && (lane & 3) == 0)
      for (int d = 32 * nope_blocks; d < p.kdim; d += 8)
        *reinterpret_cast<f16x8*>(base + t * pitch + d) = f16x8{};
  };
  Block last = now;
  for (int b = b0; b < b1; ++b, last = now, now = after(now)) {
    wait_vmem<0>();
    __syncthreads();
    const bool more = b + 1 < b1;
    const f16* src = source(more ? after(now) : now);
    const f16x8 y0 = load_out(0), y1 = load_out(1);  // (of the block before)
    const f16* wp = s_w[(b - b0) & 1];
    f32x16 acc = {};
    constexpr int kAhead = 4;
    f16x8 a[kChunks];
    auto read = [&](int c) {
      a[c] = *reinterpret_cast<const f16x8*>(wp + (c >> 2) * kPlane + w_lane[c & 3]);
    };
#pragma unroll
    for (int c = 0; c < kAhead; ++c) read(c);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      acc = mfma16<BF>(a[c], tok[c], acc);
      if (c + kAhead < kChunks) read(c + kAhead);
      if (c == 1 && b > b0) store(last, 0, y0);
      if (c == 3 && b > b0) store(last, 1, y1);
      if (c % 2 == 0 && c < 2 * kPlanes && more) copy(src, (b - b0 + 1) & 1, c / 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int left = is_value(now) ? 32 : p.nope - dim_of(now);  // keys' dims of the block
    // A token whose latent is not finite has no finite projection (an infinity or a
    // NaN times 0 is one too). Its keys become NaN, its values zeros: queries that
    // see it give NaN, and those that do not are left alone by 0 times its values.
    f16x4 y[4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int v = 0; v < 4; ++v) y[g][v] = 8 * g < left ? round16<BF>(acc[4 * g + v]) : (f16)0.0f;
    bool bad = !(fabsf(acc[0]) < INFINITY);
    if (__ballot(bad) != 0) {
#pragma unroll
      for (int v = 1; v < 16; ++v) bad &= !(fabsf(acc[v]) < INFINITY);  // (not a projection's row)
      const f16 instead = is_value(now) ? (f16)0.0f : __builtin_bit_cast(f16, (short)0x7FFF);
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int v = 0; v < 4; ++v) y[g][v] = bad && 8 * g < left ? instead : y[g][v];
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f16x4*>(so + n * kPitch + 8 * g + 4 * hh) = y[g];
  }
  if (b0 < b1) {
    store(last, 0, load_out(0));
    store(last, 1, load_out(1));
  }
}

// ---------------------------------------------------------------------------
// Attention.

// Four waves of 32 queries of one head; keys in tiles of 64 through two LDS
// buffers, straight from the expanded rows. A wave computes S^T = K Q^T (a lane
// 16 keys of one query, per 32 keys), the online softmax in the log2 domain with
// a lazy maximum, and O^T += V^T P^T from the same registers (V's rows read
// transposed in the order the scores hold the keys). Two workgroups a CU, so
// that one's products run beside the other's weights. The query tiles of a head
// are dispatched to one XCD, whose L2 then serves the head's keys and values.
// The weights are rounded to 16 bits for the second product (in bf16 1.2e-3 of the
// result's 2-norm), and the sum that divides it is of the rounded ones.
// NP, VP: planes of 64 dims of the nope part and of the values; RS: 16-dim steps
// of the rotary plane that are computed. 14 heads of 64 + 32 and 64 dims, 1531
// queries after 389 keys 24 us: 504 workgroups (168 query tiles, their keys in 3
// ranges) of up to 10 tiles, whose scores, weights and values come in turn, some
// 2.4 us a tile, and bound it.
template <int NP, int RS, int VP, bool BF>
__global__ __launch_bounds__(256, 2) void latent_prefill_kernel(const PrefillParams p) {
  constexpr int kPlane = kKeys * 64;  // halves of a 64-dim plane of a tile
  constexpr int RP = 1, KP = NP + RP;
  constexpr int kSteps = 4 * NP + RS;  // 16-dim steps of a score
  constexpr int OB = 2 * VP;          // 32-dim blocks of the output
  __shared__ __align__(1024) f16 s_k[2][KP * kPlane];
  __shared__ __align__(1024) f16 s_v[2][VP * kPlane];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int n = lane & 31, hh = lane >> 5;

  // Work items, the longest query tiles of a head first; whole rounds of 8
  // heads go one head to an XCD.
  const int per = p.tiles * p.splits;
  int item = blockIdx.x, hl;
  const int whole = p.heads / kXcds * kXcds;
  if (item < whole * per) {
    const int x = item % kXcds, j = item / kXcds;
    hl = j / per * kXcds + x;
    item = j % per;
  } else {
    item -= whole * per;
    const int rest = p.heads - whole;
    hl = whole + item % rest;
    item /= rest;
  }
  const int split = item % p.splits, tile = p.tiles - 1 - item / p.splits;
  const int h = p.head0 + hl;
  const int q0 = tile * kQueries, q1 = min(q0 + kQueries, p.count);
  const int wq0 = q0 + 32 * w, qi = wq0 + n;
  const int qpos = p.start + qi;
  const bool q_live = qi < p.count;
  const int wfirst = p.start + wq0, wlast = p.start + min(wq0 + 31, p.count - 1);

  f16x8 qf[kSteps];
  {
    const f16* qp = p.q + ((int64_t)(q_live ? qi : 0) * p.hq + h) * (p.nope + p.rope);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int d = (i < 4 * NP ? 16 * i : 16 * (i - 4 * NP)) + 8 * hh;
      const int lim = i < 4 * NP ? p.nope : p.rope;
      qf[i] = f16x8{};
      if (q_live && d < lim)
        qf[i] = *reinterpret_cast<const f16x8*>(qp + (i < 4 * NP ? 0 : p.nope) + d);
    }
  }
  const int ntile = (p.start + q1 - 1) / kKeys + 1;
  const int t_begin = (int)((int64_t)ntile * split / p.splits);
  const int t_end = (int)((int64_t)ntile * (split + 1) / p.splits);
  const int wave_end = wq0 < p.count ? min(t_end, wlast / kKeys + 1) : t_begin;

  // Copies: a wave moves 16 keys of a tile, 128 bytes of 8 rows an instruction,
  // their 16-byte pieces swizzled.
  const f16 *src_k[2], *src_r[2], *src_v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = 16 * w + 8 * i + (lane >> 3);
    const int piece = 8 * ((lane & 7) ^ swizzle(key));
    src_k[i] = p.keys + ((int64_t)hl * p.span + key) * (64 * NP) + piece;
    src_r[i] = p.rope_keys + (int64_t)key * (64 * RP) + piece;
    src_v[i] = p.values + ((int64_t)hl * p.span + key) * (64 * VP) + piece;
  }
  const uint32_t k_dst = uniform(lds_address(&s_k[0][0]) + 2048 * w);
  const uint32_t v_dst = uniform(lds_address(&s_v[0][0]) + 2048 * w);
  auto copy = [&](int t, int buf) {
    const int64_t k0 = (int64_t)t * kKeys;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f16* sk = src_k[i] + k0 * (64 * NP);
      const f16* sv = src_v[i] + k0 * (64 * VP);
      const f16* sr = src_r[i] + k0 * (64 * RP);
      const uint32_t kd = k_dst + buf * (2 * KP * kPlane) + 1024 * i;
      const uint32_t vd = v_dst + buf * (2 * VP * kPlane) + 1024 * i;
      auto nope = [&](auto j) { copy_to_lds<128 * j.value, (2 * kPlane - 128) * j.value>(sk, kd); };
      auto rope = [&](auto j) {
        copy_to_lds<128 * j.value, (2 * kPlane - 128) * j.value + 2 * NP * kPlane>(sr, kd);
      };
      auto vals = [&](auto j) { copy_to_lds<128 * j.value, (2 * kPlane - 128) * j.value>(sv, vd); };
      each(nope, std::make_integer_sequence<int, NP>{});
      each(rope, std::make_integer_sequence<int, RP>{});
      each(vals, std::make_integer_sequence<int, VP>{});
    }
  };
  int k_lane[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) k_lane[i] = 64 * n + 8 * ((2 * i + hh) ^ swizzle(n));
  const int g16 = lane >> 4, s16 = lane & 15;
  int v_lane[2][2];  // [rows 8 on][odd 32 dims of a plane]
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 8 * i + 4 * hh + (s16 >> 2);
      v_lane[i][j] = 64 * r + 4 * (s16 & 1) +
                     8 * ((4 * j + 2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ swizzle(r));
    }
  // A positive scale is applied with the maximum's subtraction, another one to
  // the scores.
  const bool direct = p.scale_log2 > 0.0f;
  const float c = direct ? p.scale_log2 : 1.0f;

  f32x16 o[OB];
#pragma unroll
  for (int i = 0; i < OB; ++i) o[i] = f32x16{};
  float m = -INFINITY, l = 0.0f;
  uint64_t ok_next = 0;
  if (t_begin < t_end) {
    copy(t_begin, 0);
    ok_next = p.seen[t_begin];
  }
  for (int t = t_begin; t < t_end; ++t) {
    const int buf = (t - t_begin) & 1;
    wait_vmem<0>();
    __syncthreads();
    const uint64_t okm = ok_next;
    if (t + 1 < t_end) {
      copy(t + 1, buf ^ 1);
      ok_next = p.seen[t + 1];
    }
    if (t >= wave_end) continue;
    const f16* kt = s_k[buf];
    const f16* vt = s_v[buf];
    const int k0 = t * kKeys;
    f32x16 s[2] = {};
#pragma unroll
    for (int cc = 0; cc < kSteps; ++cc) {
      const f16* kp = kt + k_lane[cc & 3] + kPlane * (cc >> 2);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        s[i] = mfma16<BF>(*reinterpret_cast<const f16x8*>(kp + 2048 * i), qf[cc], s[i]);
    }
    if (!direct) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[i][v] *= p.scale_log2;
    }
    if (k0 + kKeys - 1 > wfirst || okm != ~0ull) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int hi = qpos - k0 - 32 * i;  // the last visible key of the block
        uint32_t see = hi >= 31 ? 0xFFFFFFFFu : hi < 0 ? 0u : (2u << hi) - 1u;
        see = (see & (uint32_t)(okm >> (32 * i))) >> (4 * hh);
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (!(see >> (8 * (v / 4) + v % 4) & 1)) s[i][v] = -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(top, s[i][v]);
    top = fmaxf(top, __shfl_xor(top, 32)) * c;
    if (__ballot(top > m + kSlack)) {
      if (top > m + kSlack) {
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= f;
#pragma unroll
        for (int i = 0; i < OB; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[i][v] *= f;
      }
    }
    const float mu = m == -INFINITY ? 0.0f : m;
    f16x8 pb[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int v = 0; v < 16; ++v)
        pb[i][v / 8][v % 8] = round16<BF>(__builtin_amdgcn_exp2f(fmaf(s[i][v], c, -mu)));
#pragma unroll
      for (int v = 0; v < 16; v += 2)
        l = add_pair<BF>(pb[i][v / 8][v % 8], pb[i][v / 8][v % 8 + 1], l);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int b = 0; b < OB; ++b) {
          const f16* vp = vt + kPlane * (b / 2) + 2048 * i + 1024 * ks;
          const f16x4 lo = read_tr(vp + v_lane[0][b & 1]), hi = read_tr(vp + v_lane[1][b & 1]);
          o[b] = mfma16<BF>(f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]},
                            pb[i][ks], o[b]);
        }
  }
  wait_vmem<0>();
  if (!q_live) return;
  l += __shfl_xor(l, 32);
  const int64_t at = (int64_t)qi * p.hq + h;
  if (p.splits > 1) {
    const int64_t pair = (int64_t)split * p.count * p.hq + at;
    float* dst = p.part_o + pair * p.value + 4 * hh;
#pragma unroll
    for (int b = 0; b < OB; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * b + 8 * g < p.value)
          *reinterpret_cast<float4*>(dst + 32 * b + 8 * g) =
              make_float4(o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]);
    if (hh == 0) p.part_ml[pair] = make_float2(m, l);
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  f16* dst = p.out + at * p.value + 4 * hh;
#pragma unroll
  for (int b = 0; b < OB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (32 * b + 8 * g >= p.value) continue;
      f16x4 y;
#pragma unroll
      for (int v = 0; v < 4; ++v) y[v] = round16<BF>(o[b][4 * g + v] * inv);
      *reinterpret_cast<f16x4*>(dst + 32 * b + 8 * g) = y;
    }
}

// The same attention with two blocks of 32 queries a wave (256 queries a
// workgroup, one workgroup a CU), for rows of two nope planes, a rotary plane and
// two value planes. A fragment read from LDS serves both blocks, which halves the
// LDS reads that bound the kernel above, and with one wave a SIMD the weights are
// taken beside the products by a schedule: while the scores of one 32-key block
// are summed up and the values of another are weighed in, alternating, the weights
// of the block between them are formed, a few instructions after each product. A
// tile's V is used an iteration after its K. The outputs (2 x 32 x 128, 128
// registers a lane) and the queries live in accumulator registers.
// What takes the running maximum past 2^8 is found from the weights' sum after
// the fact and weighed again (settle). Rounded as above. 128 heads, 4096 tokens 684
// to 936 us for 687 GFLOP (0.73 to 1.0 PFLOP/s), by the clock that its load leaves
// from dispatch to dispatch; 16 heads, 512 at 7777 55 us for 42 GFLOP; the matrix
// cores bound it.
template <bool BF>
__global__ __launch_bounds__(256, 1) void latent_prefill_wide_kernel(const PrefillParams p) {
  constexpr int NP = 2, RP = 1, VP = 2, KP = NP + RP, OB = 2 * VP, QB = 2;
  constexpr int kPlane = kKeys * 64;
  constexpr int kSteps = 4 * KP;  // 16-dim steps of a score
  constexpr int kWide = 128 * QB; // queries of a workgroup
  __shared__ __align__(1024) f16 s_k[2][KP * kPlane];
  __shared__ __align__(1024) f16 s_v[2][VP * kPlane];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int n = lane & 31, hh = lane >> 5;

  const int units = p.paired ? (p.tiles + 1) / 2 : p.tiles;
  const int per = units * p.splits;
  int item = blockIdx.x, hl;
  const int whole = p.heads / kXcds * kXcds;
  if (item < whole * per) {
    const int x = item % kXcds, j = item / kXcds;
    hl = j / per * kXcds + x;
    item = j % per;
  } else {
    item -= whole * per;
    const int rest = p.heads - whole;
    hl = whole + item % rest;
    item /= rest;
  }
  const int split = item % p.splits, unit = item / p.splits;
  const int h = p.head0 + hl;
  // Paired: the longest query tile left and then the shortest, so that every
  // workgroup has the same number of keys to go over.
  const int last_tile = p.paired ? unit : p.tiles - 1 - unit;
#pragma unroll 1
  for (int tile = p.tiles - 1 - unit; tile >= last_tile;
       tile = tile > last_tile ? last_tile : last_tile - 1) {
  const int q0 = tile * kWide, q1 = min(q0 + kWide, p.count);
  const int wq0 = q0 + 32 * QB * w, qi = wq0 + n;
  const int qpos = p.start + qi;
  const int wfirst = p.start + wq0, wlast = p.start + min(wq0 + 32 * QB - 1, p.count - 1);
  const int ntile = (p.start + q1 - 1) / kKeys + 1;
  const int t_begin = (int)((int64_t)ntile * split / p.splits);
  const int t_end = (int)((int64_t)ntile * (split + 1) / p.splits);
  // The tiles that this wave's queries see.
  const int wb = uniform(wq0 < p.count ? min(t_end, wlast / kKeys + 1) : t_begin);

  // Copies, as above.
  const f16 *src_k[2], *src_r[2], *src_v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = 16 * w + 8 * i + (lane >> 3);
    const int piece = 8 * ((lane & 7) ^ swizzle(key));
    const int64_t at = (int64_t)t_begin * kKeys + key;
    src_k[i] = p.keys + ((int64_t)hl * p.span + at) * (64 * NP) + piece;
    src_r[i] = p.rope_keys + at * (64 * RP) + piece;
    src_v[i] = p.values + ((int64_t)hl * p.span + at) * (64 * VP) + piece;
  }
  const uint32_t k_dst = uniform(lds_address(&s_k[0][0]) + 2048 * w);
  const uint32_t v_dst = uniform(lds_address(&s_v[0][0]) + 2048 * w);
  // Copy i of a tile's K (two rows' parts, NP nope planes and the rotary ones
  // each) and of its V, whose sources move on a tile at a time.
  auto copy_k = [&](auto i, int buf) __attribute__((always_inline)) {
    constexpr int half = i.value / KP, j = i.value % KP;
    const uint32_t kd = k_dst + buf * (2 * KP * kPlane) + 1024 * half;
    if constexpr (j < NP)
      copy_to_lds<128 * j, (2 * kPlane - 128) * j>(src_k[half], kd);
    else
      copy_to_lds<128 * (j - NP), (2 * kPlane - 128) * (j - NP) + 2 * NP * kPlane>(src_r[half], kd);
  };
  auto copy_v = [&](auto i, int buf) __attribute__((always_inline)) {
    constexpr int half = i.value / VP, j = i.value % VP;
    copy_to_lds<128 * j, (2 * kPlane - 128) * j>(src_v[half],
                                                 v_dst + buf * (2 * VP * kPlane) + 1024 * half);
  };
  auto next_k = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      src_k[i] += kKeys * 64 * NP;
      src_r[i] += kKeys * 64 * RP;
    }
  };
  auto next_v = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) src_v[i] += kKeys * 64 * VP;
  };
  auto all_k = [&](int buf) {
    auto one = [&](auto i) { copy_k(i, buf); };
    each(one, std::make_integer_sequence<int, 2 * KP>{});
  };
  auto all_v = [&](int buf) {
    auto one = [&](auto i) { copy_v(i, buf); };
    each(one, std::make_integer_sequence<int, 2 * VP>{});
    next_v();
  };
  uint64_t ok_now = t_begin < t_end ? p.seen[t_begin] : 0;
  if (t_begin < t_end) all_k(0);
  if (t_begin + 1 < t_end) next_k();

  f16x8 qf[QB][kSteps];
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    const bool live = qi + 32 * j < p.count;
    const f16* qp = p.q + ((int64_t)(live ? qi + 32 * j : 0) * p.hq + h) * (p.nope + p.rope);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int d = (i < 4 * NP ? 16 * i : 16 * (i - 4 * NP)) + 8 * hh;
      const int lim = i < 4 * NP ? p.nope : p.rope;
      const f16x8 x = *reinterpret_cast<const f16x8*>(qp + (d < lim ? (i < 4 * NP ? 0 : p.nope) + d : 0));
      qf[j][i] = live && d < lim ? x : f16x8{};
    }
  }
#pragma unroll
  for (int j = 0; j < QB; ++j)
#pragma unroll
    for (int i = 0; i < kSteps; ++i) asm volatile("" : "+a"(qf[j][i]));

  const int g16 = lane >> 4, s16 = lane & 15;
  const int k_place = 64 * n + 8 * (hh ^ swizzle(n));
  const int v_row = 4 * hh + (s16 >> 2);
  const int v_place =
      64 * v_row + 4 * (s16 & 1) + 8 * ((2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ swizzle(v_row));
  const bool direct = p.scale_log2 > 0.0f;
  const float c = direct ? p.scale_log2 : 1.0f;

  f32x16 o[QB * OB];
#pragma unroll
  for (int i = 0; i < QB * OB; ++i) o[i] = f32x16{};
  outputs_settle(o);
  float m[QB], l[QB], lb[QB];
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.0f;
  }
  f32x16 s0[QB] = {}, s1[QB] = {};        // scores of the even and the odd 32-key block
  f16x8 p0[2 * QB] = {}, p1[2 * QB] = {};  // and their weights

  auto read_k = [&](const f16* kt, int i) {
    return *reinterpret_cast<const f16x8*>(kt + (k_place ^ 16 * (i & 3)) + kPlane * (i >> 2));
  };
  auto read_v = [&](const f16* vt, int i) {  // product i: dims 32 (i % OB), keys 16 (i / OB)
    const f16* vp = vt + kPlane * (i % OB / 2) + 1024 * (i / OB);
    const f16x4 lo = read_tr(vp + (v_place ^ 32 * (i & 1)));
    const f16x4 hi = read_tr(vp + (v_place ^ (16 + 32 * (i & 1))) + 512);
    return f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  // Scores of a block in place: a scale that is not positive, and the masks
  // where the block has any.
  auto shape = [&](f32x16 (&x)[QB], int k0, uint32_t okm) __attribute__((always_inline)) {
    if (!direct) {
#pragma unroll
      for (int j = 0; j < QB; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) x[j][v] *= p.scale_log2;
    }
    if (k0 + 31 <= wfirst && okm == 0xFFFFFFFFu) return;
#pragma unroll
    for (int j = 0; j < QB; ++j) {
      const int hi = qpos + 32 * j - k0;  // the last visible key of the block
      uint32_t see = hi >= 31 ? 0xFFFFFFFFu : hi < 0 ? 0u : (2u << hi) - 1u;
      see = (see & okm) >> (4 * hh);
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (!(see >> (8 * (v / 4) + v % 4) & 1)) x[j][v] = -INFINITY;
    }
  };
  auto plain = [&](int k0, uint32_t okm) {
    return direct && k0 + 31 <= wfirst && okm == 0xFFFFFFFFu;
  };
  auto put_pair = [&](f16x8 (&pb)[2 * QB], int j, int i, float e0, float e1) __attribute__((always_inline)) {
    pb[2 * j + i / 4][2 * (i % 4)] = round16<BF>(e0);
    pb[2 * j + i / 4][2 * (i % 4) + 1] = round16<BF>(e1);
  };
  auto total = [&](const f16x8 (&pb)[2 * QB], int j, float start) __attribute__((always_inline)) {
    float sum[2] = {start, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      sum[i & 1] = add_pair<BF>(pb[2 * j + i / 4][2 * (i % 4)], pb[2 * j + i / 4][2 * (i % 4) + 1],
                                sum[i & 1]);
    return sum[0] + sum[1];
  };
  auto scores = [&](f32x16 (&x)[QB], const f16* kt) __attribute__((always_inline)) {
    f16x8 a[kSteps];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = read_k(kt, i);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int j = 0; j < QB; ++j) x[j] = mfma16<BF>(a[i], qf[j][i], i == 0 ? f32x16{} : x[j]);
      if (i + 4 < kSteps) a[i + 4] = read_k(kt, i + 4);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto accumulate = [&](const f16x8 (&pb)[2 * QB], const f16* vt) __attribute__((always_inline)) {
    f16x8 a[2 * OB];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = read_v(vt, i);
#pragma unroll
    for (int i = 0; i < 2 * OB; ++i) {
#pragma unroll
      for (int j = 0; j < QB; ++j) mfma_acc<BF>(a[i], pb[2 * j + i / OB], o[j * OB + i % OB]);
      if (i + 4 < 2 * OB) a[i + 4] = read_v(vt, i + 4);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The weights of a block were taken against the running maximum and summed in
  // lb. A weight past 2^8 makes lb pass it; only then, or while no key was
  // visible (lb then is infinite), the maximum is taken and the block weighed
  // again.
  auto settle = [&](const f32x16 (&x)[QB], f16x8 (&pb)[2 * QB]) __attribute__((always_inline)) {
    bool again = false;
#pragma unroll
    for (int j = 0; j < QB; ++j) again |= !(lb[j] <= 256.0f);
    if (__ballot(again) != 0) {
      bool seen = false;
      float f[QB];
#pragma unroll
      for (int j = 0; j < QB; ++j) {
        float top = x[j][0];
#pragma unroll
        for (int v = 1; v < 16; ++v) top = fmaxf(top, x[j][v]);
        top = max_halves(top) * c;
        const bool grow = top > m[j] + kSlack;
        seen |= grow && m[j] != -INFINITY;
        f[j] = grow ? __builtin_amdgcn_exp2f(m[j] - top) : 1.0f;
        m[j] = grow ? top : m[j];
        l[j] *= f[j];
        const float mu = m[j] == -INFINITY ? 0.0f : m[j];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          put_pair(pb, j, i, __builtin_amdgcn_exp2f(fmaf(x[j][2 * i], c, -mu)),
                   __builtin_amdgcn_exp2f(fmaf(x[j][2 * i + 1], c, -mu)));
        lb[j] = total(pb, j, 0.0f);
      }
      // (Sums of a lane that has seen no key are zeros.)
      if (__ballot(seen) != 0) {
        outputs_settle(o);
#pragma unroll
        for (int i = 0; i < QB * OB; ++i) {
#pragma unroll
          for (int v = 0; v < 16; ++v) o[i][v] *= f[i / OB];
          asm volatile("" : "+a"(o[i]));
        }
      }
      operands_settle(pb);
    }
#pragma unroll
    for (int j = 0; j < QB; ++j) l[j] += lb[j];
  };
  // One step: of every five fragments three are K's (scores of a later block, xn)
  // and two V's (weights pv), each for both query blocks; beside them the
  // weights of the block between (x, into pb, summed into lb).
  auto step = [&](const f32x16 (&x)[QB], f16x8 (&pb)[2 * QB], const f16x8 (&pv)[2 * QB],
                  f32x16 (&xn)[QB], const f16* kt, const f16* vt,
                  auto beside) __attribute__((always_inline)) {
    constexpr int kOps = kSteps + 2 * OB, kSlots = QB * kOps, kAhead = 4;
    constexpr int kScores = 16 * QB;
    static_assert(kSteps % 3 == 0 && 2 * kSteps == 3 * 2 * OB, "three K to two V");
    float mu[QB], e[kScores];
#pragma unroll
    for (int j = 0; j < QB; ++j) {
      mu[j] = m[j] == -INFINITY ? 0.0f : m[j];
      lb[j] = m[j] == -INFINITY ? INFINITY : 0.0f;
    }
    f16x8 a[kOps];
    auto read = [&](int i) {
      a[i] = i % 5 & 1 ? read_v(vt, i / 5 * 2 + i % 5 / 2) : read_k(kt, i / 5 * 3 + i % 5 / 2);
    };
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(i);
    e[0] = fmaf(x[0][0], c, -mu[0]);
    __builtin_amdgcn_sched_barrier(0);
    auto slot = [&](auto sc) __attribute__((always_inline)) {
      constexpr int i = sc.value / QB, j = sc.value % QB;
      if constexpr (i % 5 & 1) {
        constexpr int v = i / 5 * 2 + i % 5 / 2;
        mfma_acc<BF>(a[i], pv[2 * j + v / OB], o[j * OB + v % OB]);
      } else {
        constexpr int k = i / 5 * 3 + i % 5 / 2;
        xn[j] = mfma16<BF>(a[i], qf[j][k], k == 0 ? f32x16{} : xn[j]);
      }
      if constexpr (j == QB - 1 && i + kAhead < kOps) read(i + kAhead);
      if constexpr (j == 0) beside(std::integral_constant<int, i>{});
      constexpr int v0 = kScores * sc.value / (kSlots - 2);
      constexpr int v1 = kScores * (sc.value + 1) / (kSlots - 2);
#pragma unroll
      for (int v = v0 < kScores ? v0 : kScores; v < (v1 < kScores ? v1 : kScores); ++v) {
        // The argument of the next exp, this exp, the pair before.
        if (v + 1 < kScores) e[v + 1] = fmaf(x[(v + 1) / 16][(v + 1) % 16], c, -mu[(v + 1) / 16]);
        e[v] = __builtin_amdgcn_exp2f(e[v]);
        if ((v & 1) && v >= 3) put_pair(pb, (v - 3) / 16, (v - 3) % 16 / 2, e[v - 3], e[v - 2]);
      }
      if constexpr (sc.value == kSlots - 2)
        put_pair(pb, QB - 1, 7, e[kScores - 2], e[kScores - 1]);
      __builtin_amdgcn_sched_barrier(0);
    };
    each(slot, std::make_integer_sequence<int, kSlots>{});
#pragma unroll
    for (int j = 0; j < QB; ++j) lb[j] = total(pb, j, lb[j]);
    // Keeps the step's products in it (they would sink past settle's branch).
#pragma unroll
    for (int j = 0; j < QB; ++j)
      asm volatile("" : "+v"(xn[j]), "+v"(pb[2 * j]), "+v"(pb[2 * j + 1]), "+v"(lb[j]));
  };
  // Iteration t: V of tile t and K of the next (of the last one again) are copied
  // beside the wave's math, and published by the barrier at its end. (The phases in
  // a row, each with a loop of its own: where paths met in one loop the outputs
  // were copied.
  // In the steps a copy goes out every other fragment: issued together they
  // waited for each other, 600 of 4900 cycles a tile.)
  uint64_t ok_prev = 0;
  auto open = [&](int t) {
    const int buf = (t - t_begin) & 1;
    all_v(buf);
    all_k(buf ^ 1);
    if (t + 2 < t_end) next_k();
  };
  auto close = [&](int t) {
    ok_prev = ok_now;
    if (t + 1 < t_end) ok_now = p.seen[t + 1];
    wait_vmem<0>();
    __syncthreads();
  };
  wait_vmem<0>();
  __syncthreads();
  int t = t_begin;
  if (t < wb) {
    // First tile: scores of both blocks, weights of the first.
    open(t);
    scores(s0, s_k[0]);
    shape(s0, t * kKeys, (uint32_t)ok_now);
    scores(s1, s_k[0] + 2048);
#pragma unroll
    for (int j = 0; j < QB; ++j) lb[j] = INFINITY;
    settle(s0, p0);
    close(t);
    for (++t; t < wb; ++t) {
      const int buf = (t - t_begin) & 1;
      const int k0 = t * kKeys;
      const f16* kt = s_k[buf];
      const f16* vt = s_v[buf ^ 1];
      const uint32_t odd = (uint32_t)(ok_prev >> 32), even = (uint32_t)ok_now;
      if (!plain(k0 - 32, odd)) shape(s1, k0 - 32, odd);
      step(s1, p1, p0, s0, kt, vt, [&](auto i) __attribute__((always_inline)) {
        if constexpr (i.value % 2 == 0) {
          constexpr int c = i.value / 2;
          if constexpr (c < 2 * VP) {
            copy_v(std::integral_constant<int, c>{}, buf);
          } else if constexpr (c < 2 * VP + 2 * KP) {
            copy_k(std::integral_constant<int, c - 2 * VP>{}, buf ^ 1);
          }
        }
      });
      next_v();
      if (t + 2 < t_end) next_k();
      settle(s1, p1);
      if (!plain(k0, even)) shape(s0, k0, even);
      step(s0, p0, p1, s1, kt + 2048, vt + 2048, [](auto) {});
      settle(s0, p0);
      close(t);
    }
    // The products of the wave's last tile.
    if (t < t_end) open(t);
    const f16* vt = s_v[(t - 1 - t_begin) & 1];
    shape(s1, (t - 1) * kKeys + 32, (uint32_t)(ok_prev >> 32));
    accumulate(p0, vt);
#pragma unroll
    for (int j = 0; j < QB; ++j) lb[j] = INFINITY;
    settle(s1, p1);
    accumulate(p1, vt + 2048);
    outputs_settle(o);
    if (t < t_end) {
      close(t);
      ++t;
    }
  }
  for (; t < t_end; ++t) {
    open(t);
    close(t);
  }
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    if (qi + 32 * j >= p.count) continue;
    const float all = l[j] + __shfl_xor(l[j], 32);
    const int64_t at = (int64_t)(qi + 32 * j) * p.hq + h;
    if (p.splits > 1) {
      const int64_t pair = (int64_t)split * p.count * p.hq + at;
      float* dst = p.part_o + pair * p.value + 4 * hh;
#pragma unroll
      for (int b = 0; b < OB; ++b) {
        const f32x16& x = o[j * OB + b];
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (32 * b + 8 * g < p.value)
            *reinterpret_cast<float4*>(dst + 32 * b + 8 * g) =
                make_float4(x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]);
      }
      if (hh == 0) p.part_ml[pair] = make_float2(m[j], all);
      continue;
    }
    const float inv = all > 0.0f ? 1.0f / all : 0.0f;
    f16* dst = p.out + at * p.value + 4 * hh;
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      const f32x16& x = o[j * OB + b];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (32 * b + 8 * g >= p.value) continue;
        f16x4 y;
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = round16<BF>(x[4 * g + v] * inv);
        *reinterpret_cast<f16x4*>(dst + 32 * b + 8 * g) = y;
      }
    }
  }
  __syncthreads();  // (the tiles' LDS is the next one's)
  }
}

// Joins the key ranges of a split call: a thread has 4 value dims of one query
// and head. Reads each partial once, which bounds it (16 heads, 512 tokens in 8
// ranges: 36 MB in 10 us).
template <bool BF>
__global__ __launch_bounds__(256) void latent_join_kernel(const PrefillParams p) {
  const int64_t pairs = (int64_t)p.count * p.hq;
  const int pieces = p.value / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= pairs * pieces) return;
  const int64_t pair = i / pieces;
  const int d = 4 * (int)(i - pair * pieces);
  float top = -INFINITY;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_ml[s * pairs + pair].x);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.0f;
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.part_ml[s * pairs + pair];
    if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // no key (not one of NaN)
    const float f = __builtin_amdgcn_exp2f(ml.x - top);
    const float4 x = *reinterpret_cast<const float4*>(p.part_o + (s * pairs + pair) * p.value + d);
    acc.x = fmaf(x.x, f, acc.x);
    acc.y = fmaf(x.y, f, acc.y);
    acc.z = fmaf(x.z, f, acc.z);
    acc.w = fmaf(x.w, f, acc.w);
    sum = fmaf(ml.y, f, sum);
  }
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  const f16x4 y = {round16<BF>(acc.x * inv), round16<BF>(acc.y * inv), round16<BF>(acc.z * inv),
                   round16<BF>(acc.w * inv)};
  *reinterpret_cast<f16x4*>(p.out + pair * p.value + d) = y;
}

// ---------------------------------------------------------------------------
// Host.

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

constexpr size_t kExpandBytes = (size_t)1 << 30;  // expanded keys and values at once
// Two query blocks a wave from whole workgroups of queries and as many keys on
// that their longer start is paid for (us a call, one block / two: 16 heads of
// 128 + 64, 512 tokens at 0 30 / 37, 256 at 7777 104 / 105, 512 at 30000 338 /
// 324; 128 heads, 512 at 0 55 / 56, 1024 at 0 123 / 108, 4096 at 0 921 / 861).
constexpr int kWideQueries = 256;
constexpr int kWideKeys = 1024;

struct PrefillPlan {
  // Planes of 64 + 64 and 64 dims, else 128 + 64 and 128 (64 + 32 and 64 dims, us a
  // call with the small and the large planes: 14 heads, 1531 tokens at 389 40 and
  // 51, 32 heads, 4096 at 0 167 and 185).
  bool small;
  bool wide;    // two query blocks a wave
  bool paired;  // two query tiles a workgroup
  int kdim, vdim, rdim;
  int span, tiles, splits, heads;  // heads per group
  size_t keys, values, rope, seen, part_o, part_ml, bytes;
};

PrefillPlan plan_for(int start, int count, int q_heads, int rope, int nope, int value) {
  PrefillPlan r;
  r.small = nope <= 64 && value <= 64;
  r.kdim = r.small ? 64 : 128;
  r.vdim = r.kdim;
  r.rdim = 64;
  r.span = (start + count + kKeys - 1) / kKeys * kKeys;
  r.wide = !r.small && count >= kWideQueries && start + count >= kWideKeys;
  const int queries = r.wide ? 2 * kQueries : kQueries;
  r.tiles = (count + queries - 1) / queries;
  const size_t head_bytes = (size_t)r.span * (r.kdim + r.vdim) * 2;
  // Heads in groups whose expanded rows fit the bound, whole rounds of XCDs
  // where that many do.
  int64_t heads = std::max<int64_t>(1, (int64_t)(kExpandBytes / head_bytes));
  if (heads >= kXcds) heads = heads / kXcds * kXcds;
  r.heads = (int)std::min<int64_t>(heads, q_heads);
  // Key ranges: enough for the workgroups to fill the GPU, each of four tiles
  // of keys at least. (us a call with 2, 4 and 8: 16 heads, 512 tokens at 0 35, 33,
  // 31; one at 1000 31, 31, 35; 512 at 7777 130, 121, 128.)
  const int64_t items = (int64_t)r.tiles * r.heads;
  const int64_t most = std::min<int64_t>(kMaxSplits, std::max(1, r.span / kKeys / 4));
  r.splits = (int)std::max<int64_t>(1, std::min(most, (r.wide ? kCus : kSlots) / items));
  // Paired tiles level the causal work where workgroups come in several rounds
  // (128 heads, 4096 tokens at 0: 873 us a call, 938 unpaired).
  r.paired = r.wide && r.splits == 1 && items >= 2 * kCus;
  size_t at = 0;
  r.keys = at;
  at = up256(at + (size_t)r.heads * r.span * r.kdim * 2);
  r.values = at;
  at = up256(at + (size_t)r.heads * r.span * r.vdim * 2);
  r.rope = at;
  at = up256(at + (size_t)r.span * r.rdim * 2);
  r.seen = at;
  at = up256(at + (size_t)r.span / 64 * 8);
  r.part_o = at;
  if (r.splits > 1) at = up256(at + (size_t)r.splits * count * q_heads * value * 4);
  r.part_ml = at;
  if (r.splits > 1) at = up256(at + (size_t)r.splits * count * q_heads * 8);
  r.bytes = at;
  return r;
}

int check_prefill(int32_t start, int32_t count, int32_t q_heads, int32_t latent_dim,
                  int32_t rope_dim, int32_t nope_dim, int32_t value_dim) {
  const int rc = check_shape(q_heads, latent_dim, rope_dim, nope_dim, value_dim);
  if (rc != PDA_OK) return rc;
  if (start < 0 || count < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "start=%d count=%d", start, count);
  if ((int64_t)start + count > INT32_MAX - 512)
    return fail(PDA_ERR_TOO_LONG, "start + count next to 2^31");
  return PDA_OK;
}

template <bool BF>
const void* prefill_kernel(bool small, int rope) {
  if (!small) return (const void*)latent_prefill_kernel<2, 4, 2, BF>;
  // (32 rotary dims, us a call with 2 and 4 steps: 32 heads, 4096 tokens at 0 159 and
  // 171.)
  return rope <= 32 ? (const void*)latent_prefill_kernel<1, 2, 1, BF>
                    : (const void*)latent_prefill_kernel<1, 4, 1, BF>;
}

int latent_prefill(const void* queries, const void* arena, const void* kv_b, const int32_t* table,
                   int32_t table_len, int32_t start, int32_t count, void* out, int32_t q_heads,
                   int32_t latent_dim, int32_t rope_dim, int32_t nope_dim, int32_t value_dim,
                   int32_t page_size, int64_t arena_rows, float scale, bool bf, void* workspace,
                   size_t workspace_bytes, void* stream) {
  const int rc =
      check_prefill(start, count, q_heads, latent_dim, rope_dim, nope_dim, value_dim);
  if (rc != PDA_OK) return rc;
  if (page_size <= 0 || table_len < 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "page_size=%d table_len=%d", page_size, table_len);
  if (count == 0) return ok();
  if (table_len == 0)
    return fail(PDA_ERR_INVALID_ARGUMENT, "an empty page table holds no keys of the chunk");
  if (!queries || !arena || !kv_b || !table || !out)
    return fail(PDA_ERR_INVALID_ARGUMENT, "null buffer pointer");
  if (arena_rows < page_size || arena_rows > INT32_MAX)
    return fail(PDA_ERR_INVALID_ARGUMENT, "arena_rows %lld: a whole page at least, below 2^31",
                (long long)arena_rows);
  if (!(scale == scale) || isinf(scale))
    return fail(PDA_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (((uintptr_t)queries | (uintptr_t)arena | (uintptr_t)kv_b | (uintptr_t)out) & 15)
    return fail(PDA_ERR_ALIGNMENT, "16-bit buffers must be 16-byte aligned");
  if ((uintptr_t)table & 3) return fail(PDA_ERR_ALIGNMENT, "the table must be 4-byte aligned");
  const PrefillPlan plan = plan_for(start, count, q_heads, rope_dim, nope_dim, value_dim);
  const int64_t grid = (int64_t)plan.tiles * plan.splits * plan.heads;
  const int64_t join = ((int64_t)count * q_heads * (value_dim / 4) + 255) / 256;
  if (grid > kMaxGrid || (plan.splits > 1 && join > kMaxGrid))
    return fail(PDA_ERR_INVALID_ARGUMENT, "queries x heads beyond one launch's workgroups");
  if (!workspace || workspace_bytes < plan.bytes)
    return fail(PDA_ERR_WORKSPACE, "a workspace of %zu bytes is needed (got %zu)", plan.bytes,
                workspace ? workspace_bytes : (size_t)0);
  if ((uintptr_t)workspace & 255)
    return fail(PDA_ERR_ALIGNMENT, "the workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  PrefillParams prm;
  prm.q = static_cast<const f16*>(queries);
  prm.arena = static_cast<const f16*>(arena);
  prm.kv_b = static_cast<const f16*>(kv_b);
  prm.table = table;
  prm.out = static_cast<f16*>(out);
  prm.keys = reinterpret_cast<f16*>(ws + plan.keys);
  prm.values = reinterpret_cast<f16*>(ws + plan.values);
  prm.rope_keys = reinterpret_cast<f16*>(ws + plan.rope);
  prm.seen = reinterpret_cast<uint64_t*>(ws + plan.seen);
  prm.part_o = reinterpret_cast<float*>(ws + plan.part_o);
  prm.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
  prm.arena_pages = arena_rows / page_size;
  prm.table_len = table_len;
  prm.page_size = page_size;
  prm.start = start;
  prm.count = count;
  prm.span = plan.span;
  prm.hq = q_heads;
  prm.latent = latent_dim;
  prm.rope = rope_dim;
  prm.nope = nope_dim;
  prm.value = value_dim;
  prm.kdim = plan.kdim;
  prm.vdim = plan.vdim;
  prm.rdim = plan.rdim;
  prm.tiles = plan.tiles;
  prm.paired = plan.paired;
  prm.splits = plan.splits;
  prm.scale_log2 = scale * kLog2e;
  void* args[] = {&prm};
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  // (256 latent dims, us a call with 4 and 8 planes: 14 heads, 1531 tokens at 389 38
  // and 44, 16 heads, 512 at 8000 67 and 74.)
  const void* expand = latent_dim <= 256 ? (bf ? (const void*)latent_expand_kernel<4, true>
                                               : (const void*)latent_expand_kernel<4, false>)
                                         : (bf ? (const void*)latent_expand_kernel<8, true>
                                               : (const void*)latent_expand_kernel<8, false>);
  const int token_tiles = (plan.span + kTokenTile - 1) / kTokenTile;
  const void* attend =
      plan.wide ? (bf ? (const void*)latent_prefill_wide_kernel<true>
                      : (const void*)latent_prefill_wide_kernel<false>)
                : (bf ? prefill_kernel<true>(plan.small, rope_dim)
                      : prefill_kernel<false>(plan.small, rope_dim));
  hipError_t err = hipSuccess;
  for (int h0 = 0; h0 < q_heads && err == hipSuccess; h0 += plan.heads) {
    prm.head0 = h0;
    prm.heads = std::min(plan.heads, q_heads - h0);
    // The projected dims shared out so that the workgroups just fill the GPU.
    const int every = prm.heads * ((nope_dim + 31) / 32 + (value_dim + 31) / 32);
    int shares = std::min(every, std::max(1, kSlots / token_tiles));
    if (shares > kXcds) shares = shares / kXcds * kXcds;
    prm.shares = shares;
    err = hipLaunchKernel(expand, dim3((unsigned)(shares * token_tiles)), dim3(256), args, 0, hs);
    if (err == hipSuccess)
      err = hipLaunchKernel(
          attend,
          dim3((plan.paired ? (plan.tiles + 1) / 2 : plan.tiles) * plan.splits * prm.heads),
          dim3(256), args, 0, hs);
  }
  if (err == hipSuccess && plan.splits > 1)
    err = hipLaunchKernel(
        bf ? (const void*)latent_join_kernel<true> : (const void*)latent_join_kernel<false>,
        dim3((unsigned)join), dim3(256), args, 0, hs);
  if (err != hipSuccess)
    return fail(PDA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

}  // namespace

extern "C" {

int pda_latent_prefill_workspace_bytes(int32_t start, int32_t count, int32_t q_heads,
                                       int32_t rope_dim, int32_t nope_dim, int32_t value_dim,
                                       size_t* bytes) {
  const int rc = check_prefill(start, count, q_heads, 8, rope_dim, nope_dim, value_dim);
  if (rc != PDA_OK) return rc;
  if (!bytes) return fail(PDA_ERR_INVALID_ARGUMENT, "null result pointer");
  *bytes = count == 0 ? 0 : plan_for(start, count, q_heads, rope_dim, nope_dim, value_dim).bytes;
  return ok();
}

int pda_latent_prefill_attention(const void* queries, const void* arena, const void* kv_b,
                                 const int32_t* table, int32_t table_len, int32_t start,
                                 int32_t count, void* out, int32_t q_heads, int32_t latent_dim,
                                 int32_t rope_dim, int32_t nope_dim, int32_t value_dim,
                                 int32_t page_size, int64_t arena_rows, float scale,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  return latent_prefill(queries, arena, kv_b, table, table_len, start, count, out, q_heads,
                        latent_dim, rope_dim, nope_dim, value_dim, page_size, arena_rows, scale,
                        false, workspace, workspace_bytes, stream);
}

int pda_latent_prefill_attention_bf16(const void* queries, const void* arena, const void* kv_b,
                                      const int32_t* table, int32_t table_len, int32_t start,
                                      int32_t count, void* out, int32_t q_heads,
                                      int32_t latent_dim, int32_t rope_dim, int32_t nope_dim,
                                      int32_t value_dim, int32_t page_size, int64_t arena_rows,
                                      float scale, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  return latent_prefill(queries, arena, kv_b, table, table_len, start, count, out, q_heads,
                        latent_dim, rope_dim, nope_dim, value_dim, page_size, arena_rows, scale,
                        true, workspace, workspace_bytes, stream);
}

}  // extern "C"
