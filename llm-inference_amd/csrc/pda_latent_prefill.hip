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

constexpr int kRowsM = 128;   // tokens of a workgroup
constexpr int kColsN = 128;   // projected dims of a workgroup

// keys[h, t] = U_h c_t, values[h, t] = D_h c_t, rounded to the element type: a
// matrix product of 128 tokens by 128 dims of one head over the latent, 64
// latent dims at a time through two LDS buffers, a wave 64 by 64. Tokens
// without a row become zeros. The workgroups of the group's first dims also
// gather the rotary keys and the mask of keys that have a row.
template <bool BF>
__global__ __launch_bounds__(256, 2) void latent_expand_kernel(const PrefillParams p) {
  constexpr int kPlane = 128 * 32;  // halves of a 32-dim plane of 128 rows
  __shared__ __align__(1024) f16 s_w[2][2 * kPlane];
  __shared__ __align__(1024) f16 s_c[2][2 * kPlane];
  __shared__ int s_row[kRowsM];
  const int tid = threadIdx.x, w = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 31, hh = lane >> 5;
  const int outs = p.nope + p.value;
  const int cols = (outs + kColsN - 1) / kColsN;
  const int t0 = blockIdx.x * kRowsM;
  const int hl = blockIdx.y / cols, j0 = (blockIdx.y % cols) * kColsN;
  const int width = p.latent + p.rope;
  if (tid < kRowsM) {
    const int t = t0 + tid;
    int row = -1;
    if (t < p.start + p.count) {
      const uint32_t pi = (uint32_t)t / (uint32_t)p.page_size;
      if (pi < (uint32_t)p.table_len) {
        const uint32_t page = (uint32_t)p.table[pi];
        if ((int64_t)page < min(p.arena_pages, (int64_t)INT32_MAX))
          row = (int)(page * (uint32_t)p.page_size + (t - pi * p.page_size));
      }
    }
    s_row[tid] = row;
    if (blockIdx.y == 0) {
      const uint64_t have = __ballot(row >= 0);
      if ((tid & 63) == 0 && t < p.span) p.seen[t / 64] = have;
    }
  }
  __syncthreads();
  if (blockIdx.y == 0) {
    const int pieces = p.rdim / 8;
    for (int i = tid; i < kRowsM * pieces; i += 256) {
      const int r = i / pieces, j = i - r * pieces;
      if (t0 + r >= p.span) break;
      f16x8 x = {};
      if (s_row[r] >= 0 && 8 * j < p.rope)
        x = *reinterpret_cast<const f16x8*>(p.arena + (int64_t)s_row[r] * width + p.latent + 8 * j);
      *reinterpret_cast<f16x8*>(p.rope_keys + (int64_t)(t0 + r) * p.rdim + 8 * j) = x;
    }
  }
  // Copies: a wave moves 32 rows of each operand, 16 rows and 64 bytes an
  // instruction, the 16-byte pieces swizzled by the row's group of four.
  const int piece = (lane & 3) ^ ((lane >> 4) & 3);
  const int last_piece = p.latent / 8 - 1;
  const f16* src_w[2];
  const f16* src_c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * w + 16 * i + (lane >> 2);
    src_w[i] = p.kv_b + ((int64_t)(p.head0 + hl) * outs + min(j0 + r, outs - 1)) * p.latent;
    src_c[i] = p.arena + (int64_t)max(s_row[r], 0) * width;
  }
  const uint32_t w_dst = uniform(lds_address(&s_w[0][0]) + 2048 * w);
  const uint32_t c_dst = uniform(lds_address(&s_c[0][0]) + 2048 * w);
  const int steps = (p.latent + 63) / 64;
  auto copy = [&](int k, int buf) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int at = 8 * min(8 * k + 4 * j + piece, last_piece);
        const uint32_t off = buf * (4 * kPlane) + j * (2 * kPlane) + 1024 * i;
        copy_to_lds<0, 0>(src_w[i] + at, w_dst + off);
        copy_to_lds<0, 0>(src_c[i] + at, c_dst + off);
      }
  };
  const int ksw = (n >> 2) & 3;
  const int lane0 = 32 * n + 8 * (hh ^ ksw), lane1 = 32 * n + 8 * ((2 + hh) ^ ksw);
  const int wo = w & 1, wt = w >> 1;
  f32x16 acc[2][2] = {};
  copy(0, 0);
  for (int k = 0; k < steps; ++k) {
    const int buf = k & 1;
    wait_vmem<0>();
    __syncthreads();
    if (k + 1 < steps) copy(k + 1, buf ^ 1);
    if (64 * (k + 1) > p.latent) {
      // The pieces past the latent repeat its last: zeros on one side.
      const int have = p.latent / 8 - 8 * k;
      for (int i = tid; i < 128 * 8; i += 256) {
        const int r = i >> 3, c = i & 7;
        if (c >= have)
          *reinterpret_cast<f16x8*>(&s_w[buf][(c >> 2) * kPlane + 32 * r +
                                              8 * ((c & 3) ^ ((r >> 2) & 3))]) = f16x8{};
      }
      __syncthreads();
    }
    const f16* wp = s_w[buf] + 64 * 32 * wo;
    const f16* cp = s_c[buf] + 64 * 32 * wt;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      f16x8 a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = (c >> 1) * kPlane + 1024 * i + (c & 1 ? lane1 : lane0);
        a[i] = *reinterpret_cast<const f16x8*>(wp + at);
        b[i] = *reinterpret_cast<const f16x8*>(cp + at);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<BF>(a[i], b[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 64 * wt + 32 * j + n;
    const int64_t t = t0 + r;
    if (t >= p.span) continue;
    const bool have = s_row[r] >= 0;
    f16* krow = p.keys + ((int64_t)hl * p.span + t) * p.kdim;
    f16* vrow = p.values + ((int64_t)hl * p.span + t) * p.vdim;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = j0 + 64 * wo + 32 * i + 8 * g + 4 * hh;
        if (d >= outs) continue;
        f16x4 y;
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = have ? round16<BF>(acc[i][j][4 * g + v]) : (f16)0.0f;
        *reinterpret_cast<f16x4*>(d < p.nope ? krow + d : vrow + (d - p.nope)) = y;
      }
    // (The queries are zeros past the nope dims; the keys have to be finite.)
    if (j0 == 0 && wo == 0 && hh == 0)
      for (int d = p.nope; d < p.kdim; d += 8) *reinterpret_cast<f16x8*>(krow + d) = f16x8{};
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
// NP, RP, VP: planes of 32 dims of the nope part, the rotary part and the
// values.
template <int NP, int RP, int VP, bool BF>
__global__ __launch_bounds__(256, 2) void latent_prefill_kernel(const PrefillParams p) {
  constexpr int kPlane = kKeys * 32;
  constexpr int KP = NP + RP;
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

  f16x8 qf[2 * KP];
  {
    const f16* qp = p.q + ((int64_t)(q_live ? qi : 0) * p.hq + h) * (p.nope + p.rope);
#pragma unroll
    for (int c = 0; c < 2 * KP; ++c) {
      const int d = (c < 2 * NP ? 16 * c : 16 * (c - 2 * NP)) + 8 * hh;
      const int lim = c < 2 * NP ? p.nope : p.rope;
      qf[c] = f16x8{};
      if (q_live && d < lim)
        qf[c] = *reinterpret_cast<const f16x8*>(qp + (c < 2 * NP ? 0 : p.nope) + d);
    }
  }
  const int ntile = (p.start + q1 - 1) / kKeys + 1;
  const int t_begin = (int)((int64_t)ntile * split / p.splits);
  const int t_end = (int)((int64_t)ntile * (split + 1) / p.splits);
  const int wave_end = wq0 < p.count ? min(t_end, wlast / kKeys + 1) : t_begin;

  // Copies: a wave moves 16 keys of a tile, 64 bytes of a row an instruction;
  // the keys' 16-byte pieces are swizzled.
  const int gk = 16 * w + (lane >> 2);
  const f16* src_k = p.keys + ((int64_t)hl * p.span + gk) * (32 * NP) + 8 * ((lane & 3) ^ ((lane >> 4) & 3));
  const f16* src_r = p.rope_keys + (int64_t)gk * (32 * RP) + 8 * ((lane & 3) ^ ((lane >> 4) & 3));
  const f16* src_v = p.values + ((int64_t)hl * p.span + gk) * (32 * VP) + 8 * (lane & 3);
  const uint32_t k_dst = uniform(lds_address(&s_k[0][0]) + 1024 * w);
  const uint32_t v_dst = uniform(lds_address(&s_v[0][0]) + 1024 * w);
  auto copy = [&](int t, int buf) {
    const int64_t k0 = (int64_t)t * kKeys;
    const f16* sk = src_k + k0 * (32 * NP);
    const f16* sv = src_v + k0 * (32 * VP);
    const f16* sr = src_r + k0 * (32 * RP);
    const uint32_t kd = k_dst + buf * (2 * KP * kPlane), vd = v_dst + buf * (2 * VP * kPlane);
    auto nope = [&](auto i) { copy_to_lds<64 * i.value, (2 * kPlane - 64) * i.value>(sk, kd); };
    auto rope = [&](auto i) {
      copy_to_lds<64 * i.value, (2 * kPlane - 64) * i.value + 2 * NP * kPlane>(sr, kd);
    };
    auto vals = [&](auto i) { copy_to_lds<64 * i.value, (2 * kPlane - 64) * i.value>(sv, vd); };
    each(nope, std::make_integer_sequence<int, NP>{});
    each(rope, std::make_integer_sequence<int, RP>{});
    each(vals, std::make_integer_sequence<int, VP>{});
  };
  const int ksw = (n >> 2) & 3;
  const int k_lane0 = 32 * n + 8 * (hh ^ ksw), k_lane1 = 32 * n + 8 * ((2 + hh) ^ ksw);
  const int g16 = lane >> 4, s16 = lane & 15;
  const int v_lane = (4 * (g16 >> 1) + (s16 >> 2)) * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
  // A positive scale is applied with the maximum's subtraction, another one to
  // the scores.
  const bool direct = p.scale_log2 > 0.0f;
  const float c = direct ? p.scale_log2 : 1.0f;

  f32x16 o[VP];
#pragma unroll
  for (int i = 0; i < VP; ++i) o[i] = f32x16{};
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
    for (int cc = 0; cc < 2 * KP; ++cc) {
      const f16* kp = kt + (cc & 1 ? k_lane1 : k_lane0) + kPlane * (cc >> 1);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        s[i] = mfma16<BF>(*reinterpret_cast<const f16x8*>(kp + 1024 * i), qf[cc], s[i]);
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
        for (int i = 0; i < VP; ++i)
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
        for (int b = 0; b < VP; ++b) {
          const f16* vp = vt + v_lane + kPlane * b + 1024 * i + 512 * ks;
          const f16x4 lo = read_tr(vp), hi = read_tr(vp + 256);
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
    for (int b = 0; b < VP; ++b)
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
  for (int b = 0; b < VP; ++b)
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
  bool small;   // planes of 64 + 32 and 64 dims, else 128 + 64 and 128
  int kdim, vdim, rdim;
  int span, tiles, splits, heads;  // heads per group
  size_t keys, values, rope, seen, part_o, part_ml, bytes;
};

PrefillPlan plan_for(int start, int count, int q_heads, int rope, int nope, int value) {
  PrefillPlan r;
  r.small = nope <= 64 && rope <= 32 && value <= 64;
  r.kdim = r.small ? 64 : 128;
  r.vdim = r.kdim;
  r.rdim = r.small ? 32 : 64;
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
  if ((int64_t)start + count > INT32_MAX - 2 * kRowsM)
    return fail(PDA_ERR_TOO_LONG, "start + count next to 2^31");
  return PDA_OK;
}

template <bool BF>
const void* prefill_kernel(bool small) {
  return small ? (const void*)latent_prefill_kernel<2, 1, 2, BF>
               : (const void*)latent_prefill_kernel<4, 2, 4, BF>;
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
  const int outs = nope_dim + value_dim;
  const int64_t cols = (int64_t)plan.heads * ((outs + kColsN - 1) / kColsN);
  const int64_t join = ((int64_t)count * q_heads * (value_dim / 4) + 255) / 256;
  if (grid > INT32_MAX || cols > 65535 || join > INT32_MAX)
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
  const void* expand =
      bf ? (const void*)latent_expand_kernel<true> : (const void*)latent_expand_kernel<false>;
  const void* attend = bf ? prefill_kernel<true>(plan.small) : prefill_kernel<false>(plan.small);
  hipError_t err = hipSuccess;
  for (int h0 = 0; h0 < q_heads && err == hipSuccess; h0 += plan.heads) {
    prm.head0 = h0;
    prm.heads = std::min(plan.heads, q_heads - h0);
    err = hipLaunchKernel(expand,
                          dim3((plan.span + kRowsM - 1) / kRowsM,
                               prm.heads * ((outs + kColsN - 1) / kColsN)),
                          dim3(256), args, 0, hs);
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
