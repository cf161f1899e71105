// Shared by the latent-attention sources: types, matrix-core steps, LDS copies
// and the argument checks that the append, the decode and the prefill call
// have in common.
#ifndef PDA_LATENT_H
#define PDA_LATENT_H

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "pda.h"
#include "pda_internal.h"

namespace pda_latent {

typedef _Float16 f16;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxLatent = 512;  // latent width
constexpr int kMaxRope = 64;     // rotary dims of a row
constexpr int kMaxHead = 128;    // nope dims and value dims of a head
constexpr int64_t kMaxGrid = UINT32_MAX / 256;  // workgroups of 256 threads a launch takes

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A value at a wave-uniform place, through the scalar cache (nothing in the
// launch writes it).
template <class T>
__device__ __forceinline__ T scalar_load(const T* p, int64_t i) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)(p + i);
}

// The larger of a lane's value and that of the lane 32 on.
__device__ __forceinline__ float max_halves(float x) {
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// A 16-lane group's transposed LDS read: 4 rows x 16 columns of 16-bit
// elements, lane s given the address of row s / 4, columns 4 (s % 4) ..; it
// receives the 4 rows of column s.
__device__ __forceinline__ f16x4 read_tr(const f16* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p));
}

// One 32x32x16 matrix-core step on 16-bit operands held as fp16 bit patterns.
// A: lane (row = lane % 32) holds k slots 8 (lane / 32) ..; B: the same for
// column lane % 32; C: lane holds column lane % 32, rows 8 (v / 4) +
// 4 (lane / 32) + v % 4.
template <bool BF>
__device__ __forceinline__ f32x16 mfma16(const f16x8& a, const f16x8& b, const f32x16& c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// The same product added to c in accumulator registers, from inline asm: the
// compiler would copy so many sums between the register files. It neither knows
// what such an instruction has in flight nor that its operands need two wait
// states after a VALU instruction wrote them, so operands_settle comes between
// those writes and the first product, outputs_settle before anything but
// another product reads c, and the A fragments come from LDS.
template <bool BF>
__device__ __forceinline__ void mfma_acc(const f16x8& a, const f16x8& b, f32x16& c) {
  if constexpr (BF)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <int kN>
__device__ __forceinline__ void operands_settle(f16x8 (&b)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) asm volatile("" : "+v"(b[i]));
  asm volatile("s_nop 1");
}
template <int kN>
__device__ __forceinline__ void outputs_settle(f32x16 (&c)[kN]) {
  asm volatile("s_nop 15\n\ts_nop 7");
#pragma unroll
  for (int i = 0; i < kN; ++i) asm volatile("" : "+a"(c[i]));
}

// f32 -> the 16-bit element type (to nearest even), as an fp16 bit pattern,
// and back.
template <bool BF>
__device__ __forceinline__ f16 round16(float x) {
  if constexpr (BF)
    return __builtin_bit_cast(f16, (bf16)x);
  else
    return (f16)x;
}
template <bool BF>
__device__ __forceinline__ float widen(f16 x) {
  if constexpr (BF)
    return (float)__builtin_bit_cast(bf16, x);
  else
    return (float)x;
}

// The sum of two weights already rounded to 16 bits, added to s.
template <bool BF>
__device__ __forceinline__ float add_pair(f16 a, f16 b, float s) {
  const f16x2 x = {a, b};
  if constexpr (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x),
                                           bf16x2{(bf16)1.0f, (bf16)1.0f}, s, false);
  else
    return __builtin_amdgcn_fdot2(x, f16x2{(f16)1.0f, (f16)1.0f}, s, false);
}

// Rows of 64 16-bit elements in LDS keep their 16-byte pieces at place piece ^
// swizzle(row): 16 lanes that read one piece of 16 rows, and the 32 that read 64
// bytes of 4 rows transposed, then fall on all 64 banks once.
__device__ __forceinline__ int swizzle(int row) { return (row & 2) * 2 + (row >> 2 & 3); }

// LDS byte address of a shared object.
__device__ __forceinline__ uint32_t lds_address(const void* at) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)at;
}

// 16 bytes per lane from global memory straight into LDS: lane i's, from src +
// kOff bytes, to dst + kOff + kPlus + 16 i (dst: wave-uniform; the
// instruction adds its offset to both addresses). The caller waits
// (wait_vmem) before the barrier that publishes them. kOnce: data that nothing
// reads again soon, which is not to displace what the caches hold.
template <int kOff, int kPlus, bool kOnce = false>
__device__ __forceinline__ void copy_to_lds(const void* src, uint32_t dst) {
  static_assert(kOff < 4096, "the instruction's offset has 12 bits");
  if constexpr (kOnce)
    asm volatile(
        "s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%3 nt" ::"s"(
            dst),
        "v"(src), "n"(kPlus), "n"(kOff)
        : "memory", "m0", "scc");
  else
    asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%3" ::"s"(
                     dst),
                 "v"(src), "n"(kPlus), "n"(kOff)
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

// Until the wave's LDS reads have returned (before a copy overwrites them).
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// Head shapes the three calls share: a row of the arena is [latent | rope],
// a query head [nope | rope], a projection head [nope + value, latent].
inline int check_shape(int32_t q_heads, int32_t latent_dim, int32_t rope_dim, int32_t nope_dim,
                       int32_t value_dim) {
  using pda_internal::fail;
  if (q_heads <= 0 || latent_dim <= 0 || rope_dim < 0 || nope_dim <= 0 || value_dim <= 0)
    return fail(PDA_ERR_INVALID_ARGUMENT,
                "q_heads=%d latent_dim=%d rope_dim=%d nope_dim=%d value_dim=%d", q_heads,
                latent_dim, rope_dim, nope_dim, value_dim);
  if (latent_dim > kMaxLatent || latent_dim % 8 || rope_dim > kMaxRope || rope_dim % 16)
    return fail(PDA_ERR_HEAD_DIM,
                "latent_dim %d, rope_dim %d: latents of 8..512 dims in eights and rotary parts "
                "of 0..64 dims in sixteens",
                latent_dim, rope_dim);
  if (nope_dim > kMaxHead || nope_dim % 8 || value_dim > kMaxHead || value_dim % 8)
    return fail(PDA_ERR_HEAD_DIM,
                "nope_dim %d, value_dim %d: head dims of 8..128 in eights", nope_dim, value_dim);
  if (q_heads > 65535)
    return fail(PDA_ERR_INVALID_ARGUMENT, "q_heads %d above 65535", q_heads);
  return PDA_OK;
}

}  // namespace pda_latent

#endif  // PDA_LATENT_H
