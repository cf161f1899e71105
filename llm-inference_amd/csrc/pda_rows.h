// Attention of 32 query rows a wave over key tiles of 64 in LDS: what packed
// prompts (pda_prompts.hip) and drafted trees (pda_drafts.hip) have in common.
//
//   o_r = sum_k w_rk v_k / sum_k w_rk,  w_rk = exp(f(q_r . k)) over the keys that
//   row r sees; f scales and, where asked, caps: f(x) = cap tanh(scale x / cap).
//
// A wave holds 32 rows and computes S^T = K Q^T and O^T += V^T W^T on
// v_mfma_f32_32x32x16: the scores of a product come out with a lane holding 16
// keys of one row, which after the exponential are the second product's operand as
// they lie (nothing moves between lanes). Weights are taken in the log2 domain
// against a running reference that moves only when a block's weights sum past 2^8 times
// the weight its maximum was given (so that 16-bit weights stay finite), and rounded to
// the element type, to nearest; their sum is that of the rounded weights, in float32, as
// are the outputs. In fp16 that weight is 2^7: the sums stay finite up to 2^15, and keys
// down to 2^-31 of the maximum still count, of which a long sequence has many (at a
// weight of 1, 40000 keys of 2^-25 lost a quarter of their share). bf16 has float32's range.
//
// LDS: planes of 64 bytes a key (32 dims), 64 keys a plane. V as it lies, for the
// transposing reads; K with the four 16-byte chunks of a key's plane permuted by
// (key / 4) % 4, so that the 16 lanes of a read touch each bank once (no bank conflicts in
// the counters).
#ifndef PDA_ROWS_H
#define PDA_ROWS_H

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

namespace pda_rows {

typedef _Float16 f16;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kSlack = 8.0f;       // log2 of how far weights pass their maximum's
constexpr int kKeys = 64;            // keys of a tile: two blocks of 32
constexpr int kPlane = kKeys * 32;   // halves of a plane

// The kernel width that serves a head dim (zeros past it); 0: none does.
constexpr int width_for(int dim) {
  return dim <= 0 || dim % 8 ? 0 : dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128
         : dim <= 256 ? 256 : 0;
}

// How scores become weights' exponents.
struct Shape {
  float scale_log2;
  float cap_in;   // 2 log2(e) scale / softcap
  float cap_out;  // softcap log2(e); 0: no softcap
};
inline Shape shape_of(float scale, float softcap) {
  return {scale * kLog2e, softcap > 0.0f ? 2.0f * kLog2e * scale / softcap : 0.0f,
          softcap * kLog2e};
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

__device__ __forceinline__ f16x4 read_tr(const f16* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p));
}

// LDS byte address of a shared object.
__device__ __forceinline__ uint32_t lds_address(const void* at) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)at;
}

// 16 bytes per lane from global memory straight into LDS, plane `kAt` of a key's row:
// lane i's from src + 64 kAt to dst + 2 kPlane kAt + 16 i (dst: of the tile, wave-
// uniform; the instruction adds its offset to both addresses). The caller waits
// (wait_vmem) before the barrier that publishes them.
template <int kAt>
__device__ __forceinline__ void copy_plane_to_lds(const void* src, uint32_t dst) {
  asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%3" ::"s"(
                   dst),
               "v"(src), "n"((2 * kPlane - 64) * kAt), "n"(64 * kAt)
               : "memory", "m0", "scc");
}

// f(0), f(1), ... with compile-time arguments.
template <class F, int... kI>
__device__ __forceinline__ void each(F& f, std::integer_sequence<int, kI...>) {
  (f(std::integral_constant<int, kI>{}), ...);
}

// Until at most kLeft of the wave's loads and copies are under way.
template <int kLeft>
__device__ __forceinline__ void wait_vmem() {
  static_assert(kLeft < 64, "the count has six bits");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (kLeft & 15) | (kLeft >> 4) << 14);
}

template <bool BF>
__device__ __forceinline__ f32x16 mfma16(const f16x8& a, const f16x8& b, const f32x16& c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// f32 -> the 16-bit element type (to nearest even), as an fp16 bit pattern.
template <bool BF>
__device__ __forceinline__ f16 round16(float x) {
  if constexpr (BF)
    return __builtin_bit_cast(f16, (bf16)x);
  else
    return (f16)x;
}
template <bool BF>
__device__ __forceinline__ float widen16(f16 x) {
  if constexpr (BF)
    return (float)__builtin_bit_cast(bf16, x);
  else
    return (float)x;
}

// Whether one of eight elements is an infinity or a NaN: all ones in the exponent.
template <bool BF>
__device__ __forceinline__ bool not_finite(const f16x8& x) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 y = __builtin_bit_cast(u32x4, x);
  constexpr uint32_t kExp = BF ? 0x7F80u : 0x7C00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bad |= (y[i] & kExp) == kExp || ((y[i] >> 16) & kExp) == kExp;
  return bad;
}

template <bool BF>
__device__ __forceinline__ float4 widen4(const f16* p) {
  const f16x4 x = *reinterpret_cast<const f16x4*>(p);
  return make_float4(widen16<BF>(x[0]), widen16<BF>(x[1]), widen16<BF>(x[2]), widen16<BF>(x[3]));
}

// Zeros in the place of elements that are not finite.
template <bool BF>
__device__ __forceinline__ f16x8 finite_only(f16x8 x) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (!(fabsf(widen16<BF>(x[j])) < INFINITY)) x[j] = (f16)0.0f;
  return x;
}

// One bit a key from a ballot with four lanes a key.
__device__ __forceinline__ uint32_t keys_of(uint64_t lanes) {
  if (lanes == 0) return 0;
  if (lanes == ~0ull) return 0xFFFFu;
  lanes |= lanes >> 1;
  lanes |= lanes >> 2;
  uint32_t keys = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) keys |= (uint32_t)(lanes >> (4 * i) & 1) << i;
  return keys;
}

// Bits 0 .. n - 1 (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int n) {
  const uint32_t ones = n >= 32 ? 32u : n > 0 ? (uint32_t)n : 0u;
  return (uint32_t)((1ull << ones) - 1);
}

// 32 rows of one wave: lane l holds row l % 32, half l / 32 of its keys and dims
// (of every 8 the first or the last four).
// BF: queries, keys and outputs are bf16 (else fp16); VBF: values and weights are.
template <int D, bool BF, bool VBF = BF>
struct Rows {
  static constexpr float kTop = VBF ? 0.0f : 7.0f;  // log2 of a maximum's weight
  static constexpr float kMost = VBF ? 256.0f : 32768.0f;  // 2^(kTop + kSlack)

  f16x8 q[D / 16];
  f32x16 o[D / 32];
  float m, l;  // running reference (log2 units), sum of this lane's weights
  float c;     // what a shaped score is multiplied by
  int n, hh;
  int k_lane0, k_lane1, v_lane;

  __device__ __forceinline__ void init(const Shape& f) {
    const int lane = threadIdx.x & 63;
    n = lane & 31;
    hh = lane >> 5;
    const int ksw = (n >> 2) & 3;
    k_lane0 = 32 * n + 8 * (hh ^ ksw);
    k_lane1 = 32 * n + 8 * ((2 + hh) ^ ksw);
    const int g16 = lane >> 4, s16 = lane & 15;
    v_lane = (4 * (g16 >> 1) + (s16 >> 2)) * 32 + 16 * (g16 & 1) + 4 * (s16 & 3);
    c = f.cap_out <= 0.0f && f.scale_log2 > 0.0f ? f.scale_log2 : 1.0f;
    clear();
  }

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int b = 0; b < D / 32; ++b) o[b] = f32x16{};
  }

  // This lane's row of queries; `dim` elements of it, zeros past them.
  __device__ __forceinline__ void load(const f16* row, int dim, bool live) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int d = 16 * i + 8 * hh;
      const bool in = live && d < dim;
      const f16x8 x = *reinterpret_cast<const f16x8*>(row + (in ? d : 0));
      q[i] = in ? x : f16x8{};
    }
  }
  // Before their first use. Only matrix-core operands: where the outputs take half the
  // vector registers, they go to accumulator registers.
  __device__ __forceinline__ void settle_queries() {
    if constexpr (D > 128) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) asm volatile("" : "+a"(q[i]));
    }
  }

  // Scores of the 32 keys from kt on.
  __device__ __forceinline__ void scores(f32x16& x, const f16* kt) const {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const f16x8 a = *reinterpret_cast<const f16x8*>(kt + (i & 1 ? k_lane1 : k_lane0) +
                                                      kPlane * (i >> 1));
      x = mfma16<BF>(a, q[i], i == 0 ? f32x16{} : x);
    }
  }

  // Caps and scales that are not one positive factor.
  __device__ __forceinline__ static void shape(f32x16& x, const Shape& f) {
    if (f.cap_out > 0.0f) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float e = __builtin_amdgcn_exp2f(x[v] * f.cap_in);
        x[v] = (1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f)) * f.cap_out;
      }
    } else if (!(f.scale_log2 > 0.0f)) {
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = x[v] * f.scale_log2;
    }
  }

  // Hides the keys of a block whose bit in `see` is not set.
  __device__ __forceinline__ static void mask(f32x16& x, uint32_t see) {
    see >>= 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int bit = __builtin_amdgcn_sbfe((int)see, 8 * (v / 4) + (v % 4), 1);
      const float y = x[v];  // (a bit cast of x[v] itself takes element 0)
      x[v] = __builtin_bit_cast(float, (__builtin_bit_cast(int, y) & bit) |
                                           (~bit & (int)0xFF800000));
    }
  }

  // Weights 2 i, 2 i + 1 of a block, rounded to 16 bits and packed.
  __device__ __forceinline__ static void put_pair(f16x8 (&w)[2], int i, float e0, float e1) {
    f16x2 ph;
    if constexpr (VBF)
      ph = __builtin_bit_cast(f16x2, bf16x2{(bf16)e0, (bf16)e1});
    else
      ph = f16x2{(f16)e0, (f16)e1};
    w[i / 4][2 * (i % 4)] = ph[0];
    w[i / 4][2 * (i % 4) + 1] = ph[1];
  }

  // Their sum.
  __device__ __forceinline__ static float total(const f16x8 (&w)[2], float sum) {
    float s2[2] = {sum, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f16x2 ph = {w[i / 4][2 * (i % 4)], w[i / 4][2 * (i % 4) + 1]};
      if constexpr (VBF)
        s2[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, ph),
                                                    bf16x2{(bf16)1.0f, (bf16)1.0f}, s2[i & 1],
                                                    false);
      else
        s2[i & 1] = __builtin_amdgcn_fdot2(ph, f16x2{(f16)1.0f, (f16)1.0f}, s2[i & 1], false);
    }
    return s2[0] + s2[1];
  }

  __device__ __forceinline__ float weigh_against(const f32x16& x, f16x8 (&w)[2], float mu) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      put_pair(w, i, __builtin_amdgcn_exp2f(fmaf(x[2 * i], c, -mu)),
               __builtin_amdgcn_exp2f(fmaf(x[2 * i + 1], c, -mu)));
    return total(w, 0.0f);
  }

  // A block's weights w, summed in lb, were taken against the running reference.
  // Only where they sum past kMost (or no key was seen before: lb is infinite; or
  // one is not a number) the maximum is taken and the block weighed again.
  __device__ __forceinline__ void settle(const f32x16& x, f16x8 (&w)[2], float lb) {
    if (__ballot(!(lb <= kMost)) != 0) {
      float top = x[0];
#pragma unroll
      for (int v = 1; v < 16; ++v) top = fmaxf(top, x[v]);
      top = fmaxf(top, __shfl_xor(top, 32)) * c - kTop;
      if (top > m + kSlack) {
        if (m != -INFINITY) {
          const float f = __builtin_amdgcn_exp2f(m - top);
          l *= f;
#pragma unroll
          for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[b][v] *= f;
        }
        m = top;
      }
      lb = weigh_against(x, w, m == -INFINITY ? 0.0f : m);
    }
    l += lb;
  }

  __device__ __forceinline__ void weigh(const f32x16& x, f16x8 (&w)[2]) {
    settle(x, w, m == -INFINITY ? INFINITY : weigh_against(x, w, m));
  }

  // O^T += V^T W^T over the 32 keys from vt on.
  __device__ __forceinline__ void accumulate(const f16x8 (&w)[2], const f16* vt) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
        const f16* vp = vt + v_lane + kPlane * b + 512 * ks;
        const f16x4 lo4 = read_tr(vp);
        const f16x4 hi4 = read_tr(vp + 256);
        const f16x8 a = {lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
        o[b] = mfma16<VBF>(a, w[ks], o[b]);
      }
    }
  }

  // The pipeline's step: the products of a 32-key block's V (weights pv, values vt)
  // alternate with the scores of a later block (xn, keys kt), and the weights of the
  // block between them (x, into w, summed in lb) are spread over those D / 8 matrix
  // instructions, so that one wave alone keeps the matrix core busy while its
  // exponentials run. Operands are read four ahead. beside(i) is called at slot i for
  // what else is to be issued there.
  template <class F>
  __device__ __forceinline__ void step(const f32x16& x, f16x8 (&w)[2], const f16x8 (&pv)[2],
                                       f32x16& xn, float& lb, const f16* kt, const f16* vt,
                                       F beside) {
    constexpr int kSlots = D / 8, kAhead = 4;
    const float mu = m == -INFINITY ? 0.0f : m;
    lb = m == -INFINITY ? INFINITY : 0.0f;
    float e[16];
    f16x8 a[kSlots];
    auto read = [&](int i) {
      if (i & 1) {
        const int c = i >> 1;
        a[i] = *reinterpret_cast<const f16x8*>(kt + (c & 1 ? k_lane1 : k_lane0) + kPlane * (c >> 1));
      } else {
        const int b = (i >> 1) % (D / 32), ks = (i >> 1) / (D / 32);
        const f16* vp = vt + v_lane + kPlane * b + 512 * ks;
        const f16x4 lo4 = read_tr(vp);
        const f16x4 hi4 = read_tr(vp + 256);
        a[i] = f16x8{lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
      }
    };
    // (Before the other wave of the SIMD while it is in a step: 16384 tokens, 28/4 heads
    // of 128, 1869 -> 1837 us; 16 prompts 239 -> 232; until the weights are packed, not
    // summed, 1843 and 237.)
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(i);
    e[0] = fmaf(x[0], c, -mu);
    __builtin_amdgcn_sched_barrier(0);
    auto slot = [&](auto sc) {
      constexpr int i = sc.value;
      if constexpr (i & 1) {
        constexpr int cc = i >> 1;
        xn = mfma16<BF>(a[i], q[cc], cc == 0 ? f32x16{} : xn);
      } else {
        constexpr int b = (i >> 1) % (D / 32), ks = (i >> 1) / (D / 32);
        o[b] = mfma16<VBF>(a[i], pv[ks], o[b]);
      }
      if constexpr (i + kAhead < kSlots) read(i + kAhead);
      beside(sc);
      // The argument of the next exponential, this one, the pair before; done two
      // slots early.
      constexpr int v0 = 16 * i / (kSlots - 2), v1 = 16 * (i + 1) / (kSlots - 2);
#pragma unroll
      for (int v = v0 < 16 ? v0 : 16; v < (v1 < 16 ? v1 : 16); ++v) {
        if (v + 1 < 16) e[v + 1] = fmaf(x[v + 1], c, -mu);
        e[v] = __builtin_amdgcn_exp2f(e[v]);
        if ((v & 1) && v >= 3) put_pair(w, (v - 3) / 2, e[v - 3], e[v - 2]);
      }
      if constexpr (i == kSlots - 2) put_pair(w, 7, e[14], e[15]);
      __builtin_amdgcn_sched_barrier(0);
    };
    each(slot, std::make_integer_sequence<int, kSlots>{});
    lb = total(w, lb);
    __builtin_amdgcn_s_setprio(0);
    // Keeps the products of the step in it (they would sink past the branch of
    // settle, away from the weights they are to overlap).
    asm volatile("" : "+v"(xn), "+v"(w[0]), "+v"(w[1]), "+v"(lb));
#pragma unroll
    for (int b = 0; b < D / 32; ++b) asm volatile("" : "+v"(o[b]));
  }

  // A key's values that are not finite were taken as zeros (0 times one is no 0): adds
  // them where the lane's row sees the key (any weight of them comes to the same).
  // value4(d): values d .. d + 3 of the key as they are.
  template <class F>
  __device__ __forceinline__ void add_not_finite(bool seen, int dim, F value4) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const int d = 8 * i + 4 * hh;
      const float4 y = value4(min(d, dim - 4));
      const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int t = 0; t < 4; ++t)
        o[i / 4][4 * (i % 4) + t] += seen && d < dim && !(fabsf(ys[t]) < INFINITY) ? ys[t] : 0.0f;
      __builtin_amdgcn_sched_barrier(0);  // (else all loads at once)
    }
  }

  // 1 / the row's sum, 0 where the row sees nothing (and NaN for NaN).
  __device__ __forceinline__ float inverse() const {
    const float sum = l + __shfl_xor(l, 32);
    return sum == 0.0f ? 0.0f : 1.0f / sum;
  }

  // The row's outputs, normalised.
  __device__ __forceinline__ void store(f16* row, int dim, float inv) const {
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * b + 8 * g + 4 * hh;
        f16x4 y;
#pragma unroll
        for (int t = 0; t < 4; ++t) y[t] = round16<BF>(o[b][4 * g + t] * inv);
        if (d < dim) *reinterpret_cast<f16x4*>(row + d) = y;
      }
    }
  }
};

// The tiles [t0, t1) of a workgroup, of which this wave's rows see [wa, wb) (the last
// one's odd block only with odd_last). `x` moves and shapes them:
//   first(t0)     K of the first tile is readable, its V and the next K under way
//   ahead(r)      once no more scores are taken: what comes after may load its queries
//   aim(t), copy<j>(t) for all j < T::kCopies: V of tile t and K of tile t + 1
//   close(t)      they are readable by all waves; all are done with V of t - 1, K of t
//   shape(s, k0)  caps and masks of the scores of the keys from k0 on, with rough(t)
//                 telling whether the odd block before tile t or its even one need it
// T::kSpread: the copies go beside a step's products, else in front of them.
// V runs one tile behind K, so that two LDS tiles of each serve the pipeline with one
// barrier a tile.
template <class R, class T>
__device__ __forceinline__ void attend(R& r, T& x, int t0, int t1, int wa, int wb, bool odd_last) {
  int t = t0;
  x.first(t);
  auto copies = [&]() {
    x.aim(t);
    auto one = [&](auto j) { x.template copy<j.value>(t); };
    each(one, std::make_integer_sequence<int, T::kCopies>{});
  };
  auto idle = [&]() {  // a tile that this wave's rows do not see
    if (t > t0) copies();
    x.close(t);
  };
  const int from = wa < wb ? wa : t1;
  for (; t < from; ++t) idle();
  if (t < t1) {
    f32x16 s0, s1 = {};
    f16x8 w0[2], w1[2] = {};
    float lb;
    // First tile: scores of both blocks, weights of the even one.
    if (t > t0) copies();
    {
      const f16* kt = x.keys(t);
      r.scores(s0, kt);
      x.shape(s0, t * kKeys);
      if (wb - wa > 1 || odd_last) r.scores(s1, kt + 1024);
      r.weigh(s0, w0);
      x.close(t);
    }
    // Scores of tile t, weights of its even block and of tile t - 1's odd one,
    // products of tile t - 1's V.
    for (++t; t < wb; ++t) {
      const int k0 = t * kKeys;
      const f16* kt = x.keys(t);
      const f16* vt = x.values(t - 1);
      if constexpr (T::kSpread)
        x.aim(t);
      else
        copies();
      const bool rough = x.rough(t);
      if (rough) x.shape(s1, k0 - 32);
      r.step(s1, w1, w0, s0, lb, kt, vt, [&](auto i) {
        // (Every other slot: a copy is two instructions and an address.)
        if constexpr (T::kSpread && i.value % 2 == 0 && i.value / 2 < T::kCopies)
          x.template copy<i.value / 2>(t);
      });
      r.settle(s1, w1, lb);
      if (rough) x.shape(s0, k0);
      r.step(s0, w0, w1, s1, lb, kt + 1024, vt + 1024, [](auto) {});
      r.settle(s0, w0, lb);
      x.close(t);
    }
    // Past the last tile: weights of its odd block, products of its V.
    if (t < t1) copies();
    x.ahead(r);
    const f16* vt = x.values(t - 1);
    r.accumulate(w0, vt);
    if (odd_last) {
      x.shape(s1, (t - 1) * kKeys + 32);
      r.weigh(s1, w1);
      r.accumulate(w1, vt + 1024);
    }
    if (t < t1) x.close(t);
    for (++t; t < t1; ++t) idle();
  } else {
    x.ahead(r);
  }
}

}  // namespace pda_rows

#endif  // PDA_ROWS_H
