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
constexpr int kMaxSplits = 64;
constexpr float kSlack = 8.0f;
constexpr int kXcds = 8;
constexpr int kCus = 256;

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
  int32_t splits;
  float scale_log2;
};

// ---------------------------------------------------------------------------
// Expansion.

// keys[h, t] = U_h c_t, values[h, t] = D_h c_t, rounded to the element type: a
// matrix product in which the tokens stay and the projections stream. A wave
// keeps 32 TB tokens' whole latents as operands (TB x 128 registers at 512 dims,
// gathered from the pages once); the workgroup walks the projected dims of its
// heads 32 at a time through a ring of LDS blocks, each read once by every wave
// for TB products: with two token blocks the matrix cores and not the LDS bound
// it. Results are stored a block late, so that no wait for a copy waits for a
// store. Tokens without a row are zeros from the start. The workgroups of the
// group's first heads also gather the rotary keys and the mask of keys that have
// a row.
template <int TB, bool BF>
__global__ __launch_bounds__(256, TB == 2 ? 1 : 2) void latent_expand_kernel(const PrefillParams p) {
  constexpr int kRing = TB == 2 ? 4 : 2;
  constexpr int kPlane = 32 * 64;  // halves of 64 latent dims of a block
  constexpr int kPlanes = kMaxLatent / 64;
  constexpr int kChunks = 4 * kPlanes;
  constexpr int kTokens = 128 * TB;
  constexpr int kCopies = kPlanes;  // a wave's, a block
  constexpr int kPitch = 40;        // halves of a token's 32 results
  __shared__ __align__(1024) f16 s_w[kRing][kPlanes * kPlane];
  __shared__ __align__(16) f16 s_out[4][32 * TB * kPitch];
  __shared__ int s_row[kTokens];
  const int tid = threadIdx.x, w = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 31, hh = lane >> 5;
  const int outs = p.nope + p.value;
  const int t0 = blockIdx.y * kTokens;
  const int width = p.latent + p.rope;
  for (int i = tid; i < kTokens; i += 256) {
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
    if (blockIdx.x == 0) {
      const uint64_t have = __ballot(row >= 0);
      if ((tid & 63) == 0 && t < p.span) p.seen[t / 64] = have;
    }
  }
  __syncthreads();
  // The group's blocks of 32 projected dims (a head's nope dims, then its value
  // dims, each to a whole block), shared out evenly.
  const int nope_blocks = (p.nope + 31) / 32, each_head = nope_blocks + (p.value + 31) / 32;
  const int64_t every = (int64_t)p.heads * each_head;
  const int b0 = uniform((int)(every * blockIdx.x / gridDim.x));
  const int b1 = uniform((int)(every * (blockIdx.x + 1) / gridDim.x));

  // Copies: an instruction moves 128 bytes of 8 projection rows, the wave's. Past
  // the latent's end they repeat its last piece (the tokens are zeros there),
  // past a head's part its last row (not used).
  const int my_row = 8 * w + (lane >> 3);
  const int piece = (lane & 7) ^ swizzle(my_row);
  const int last_piece = p.latent / 8 - 1;
  const uint32_t lds = uniform(lds_address(&s_w[0][0]));
  auto copy = [&](int block) {
    const int h = block / each_head, part = block - h * each_head;
    const bool value = part >= nope_blocks;
    const int d0 = 32 * (value ? part - nope_blocks : part);
    const int size = value ? p.value : p.nope;
    const f16* src =
        p.kv_b + ((int64_t)(p.head0 + h) * outs + (value ? p.nope : 0) + min(d0 + my_row, size - 1)) *
                     p.latent;
    const uint32_t dst = lds + ((block - b0) % kRing) * (2 * kPlanes * kPlane) + 1024 * w;
#pragma unroll
    for (int j = 0; j < kPlanes; ++j)
      copy_to_lds<0, 0>(src + 8 * min(8 * j + piece, last_piece), dst + j * (2 * kPlane));
  };
  if (b0 < b1) copy(b0);
  if constexpr (kRing > 2) {
    if (b0 + 1 < b1) copy(b0 + 1);
    if (b0 + 2 < b1) copy(b0 + 2);
  }
  // The wave's tokens.
  f16x8 tok[TB][kChunks];
#pragma unroll
  for (int j = 0; j < TB; ++j) {
    const int row = s_row[32 * (TB * w + j) + n];
    const f16* src = p.arena + (int64_t)max(row, 0) * width;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int d = 16 * c + 8 * hh;
      const f16x8 x = *reinterpret_cast<const f16x8*>(src + min(d, p.latent - 8));
      tok[j][c] = row >= 0 && d < p.latent ? x : f16x8{};
    }
  }
  if (blockIdx.x == 0) {
    const int pieces = p.rdim / 8;
    for (int i = tid; i < kTokens * pieces; i += 256) {
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
  auto store = [&](int block) {
    const int h = block / each_head, part = block - h * each_head;
    const bool value = part >= nope_blocks;
    const int d0 = 32 * (value ? part - nope_blocks : part);
    f16* base = value ? p.values + (int64_t)h * p.span * p.vdim
                      : p.keys + (int64_t)h * p.span * p.kdim;
    const int pitch = value ? p.vdim : p.kdim;
#pragma unroll
    for (int j = 0; j < 2 * TB; ++j) {
      const int r = 16 * j + (lane >> 2);
      const int64_t t = t0 + 32 * TB * w + r;
      if (t >= p.span) continue;
      *reinterpret_cast<f16x8*>(base + t * pitch + d0 + 8 * (lane & 3)) =
          *reinterpret_cast<const f16x8*>(so + r * kPitch + 8 * (lane & 3));
      // (Planes of the keys that no block fills.)
      if (part == nope_blocks - 1 && (lane & 3) == 0)
        for (int d = 32 * nope_blocks; d < p.kdim; d += 8)
          *reinterpret_cast<f16x8*>(base + t * pitch + d) = f16x8{};
    }
  };
  int w_lane[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w_lane[i] = 64 * n + 8 * ((2 * i + hh) ^ swizzle(n));
  const int steps = (p.latent + 15) / 16;
  for (int b = b0; b < b1; ++b) {
    // (Operations end in order: of the last 2 kCopies, a block's stores may be
    // among them.)
    if (kRing > 2 && b + 2 < b1)
      wait_vmem<2 * kCopies>();
    else if (kRing > 2 && b + 1 < b1)
      wait_vmem<kCopies>();
    else
      wait_vmem<0>();
    __syncthreads();
    if (b > b0) store(b - 1);
    constexpr int kNext = kRing > 2 ? 3 : 1;
    if (b + kNext < b1) copy(b + kNext);
    const f16* wp = s_w[(b - b0) % kRing];
    f32x16 acc[TB];
#pragma unroll
    for (int j = 0; j < TB; ++j) acc[j] = f32x16{};
    constexpr int kAhead = 4;
    f16x8 a[kChunks];
    auto read = [&](int c) {
      a[c] = *reinterpret_cast<const f16x8*>(wp + (c >> 2) * kPlane + w_lane[c & 3]);
    };
    auto products = [&](auto count) {
#pragma unroll
      for (int c = 0; c < kAhead; ++c) read(c);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < count.value; ++c) {
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[j] = mfma16<BF>(a[c], tok[j][c], acc[j]);
        if (c + kAhead < count.value) read(c + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (steps <= kChunks / 2)
      products(std::integral_constant<int, kChunks / 2>{});
    else
      products(std::integral_constant<int, kChunks>{});
    const int part = b % each_head;
    const int left = part >= nope_blocks ? 32 : p.nope - 32 * part;  // keys' dims of the block
#pragma unroll
    for (int j = 0; j < TB; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f16x4 y;
#pragma unroll
        for (int v = 0; v < 4; ++v)
          y[v] = 8 * g < left ? round16<BF>(acc[j][4 * g + v]) : (f16)0.0f;
        *reinterpret_cast<f16x4*>(so + (32 * j + n) * kPitch + 8 * g + 4 * hh) = y;
      }
  }
  if (b0 < b1) store(b1 - 1);
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
// NP, RP, VP: planes of 64 dims of the nope part, the rotary part and the
// values.
template <int NP, int RP, int VP, bool BF>
__global__ __launch_bounds__(256, 2) void latent_prefill_kernel(const PrefillParams p) {
  constexpr int kPlane = kKeys * 64;  // halves of a 64-dim plane of a tile
  constexpr int KP = NP + RP;
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

  f16x8 qf[4 * KP];
  {
    const f16* qp = p.q + ((int64_t)(q_live ? qi : 0) * p.hq + h) * (p.nope + p.rope);
#pragma unroll
    for (int i = 0; i < 4 * KP; ++i) {
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
    for (int cc = 0; cc < 4 * KP; ++cc) {
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

// Joins the key ranges of a split call: a thread has 4 value dims of one query
// and head.
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
  if (top != -INFINITY) {
    for (int s = 0; s < p.splits; ++s) {
      const float2 ml = p.part_ml[s * pairs + pair];
      if (ml.x == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(ml.x - top);
      const float4 x = *reinterpret_cast<const float4*>(p.part_o + (s * pairs + pair) * p.value + d);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
      sum = fmaf(ml.y, f, sum);
    }
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
constexpr int kSlots = 512;                       // workgroups resident on an MI355X

struct PrefillPlan {
  bool small;   // planes of 64 + 64 and 64 dims, else 128 + 64 and 128
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
  r.tiles = (count + kQueries - 1) / kQueries;
  const size_t head_bytes = (size_t)r.span * (r.kdim + r.vdim) * 2;
  // Heads in groups whose expanded rows fit the bound, whole rounds of XCDs
  // where that many do.
  int64_t heads = std::max<int64_t>(1, (int64_t)(kExpandBytes / head_bytes));
  if (heads >= kXcds) heads = heads / kXcds * kXcds;
  r.heads = (int)std::min<int64_t>(heads, q_heads);
  // Key ranges: enough for the workgroups to fill the GPU, each of four tiles
  // of keys at least.
  const int64_t items = (int64_t)r.tiles * r.heads;
  const int64_t most = std::min<int64_t>(kMaxSplits, std::max(1, r.span / kKeys / 4));
  r.splits = (int)std::max<int64_t>(1, std::min(most, kSlots / items));
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
const void* prefill_kernel(bool small) {
  return small ? (const void*)latent_prefill_kernel<1, 1, 1, BF>
               : (const void*)latent_prefill_kernel<2, 1, 2, BF>;
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
  if (grid > INT32_MAX || join > INT32_MAX)
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
  prm.splits = plan.splits;
  prm.scale_log2 = scale * kLog2e;
  void* args[] = {&prm};
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  // Two token blocks a wave where that still fills the CUs (one workgroup
  // each), one where it would not (two workgroups each).
  const int64_t wide = ((int64_t)plan.span + 255) / 256 * plan.heads;
  const bool two = wide >= kCus;
  const void* expand = two ? (bf ? (const void*)latent_expand_kernel<2, true>
                                 : (const void*)latent_expand_kernel<2, false>)
                           : (bf ? (const void*)latent_expand_kernel<1, true>
                                 : (const void*)latent_expand_kernel<1, false>);
  const int tokens = two ? 256 : 128;
  const int token_tiles = (plan.span + tokens - 1) / tokens;
  const void* attend = bf ? prefill_kernel<true>(plan.small) : prefill_kernel<false>(plan.small);
  hipError_t err = hipSuccess;
  for (int h0 = 0; h0 < q_heads && err == hipSuccess; h0 += plan.heads) {
    prm.head0 = h0;
    prm.heads = std::min(plan.heads, q_heads - h0);
    // The projected dims shared out so that the workgroups just fill the GPU.
    const int every = prm.heads * ((nope_dim + 31) / 32 + (value_dim + 31) / 32);
    int shares = std::min(every, std::max(1, (two ? kCus : 2 * kCus) / token_tiles));
    if (shares > kXcds) shares = shares / kXcds * kXcds;
    err = hipLaunchKernel(expand, dim3(shares, token_tiles), dim3(256), args, 0, hs);
    if (err == hipSuccess)
      err = hipLaunchKernel(attend, dim3(plan.tiles * plan.splits * prm.heads), dim3(256), args, 0,
                            hs);
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
