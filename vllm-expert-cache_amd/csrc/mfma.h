// Matrix-core fragments of the products over slots (experts.h, adapters.h).
//
// Both use v_mfma_f32_16x16x32 with the weights as the first operand: 16 weight rows against
// 16 columns of tokens, so a weight is read once for up to 16 tokens. A lane holds of the
// weights row (lane & 15) and of the tokens column (lane & 15), eight values of the 32 along k
// each, at its quarter of the wave (lane >> 4). Which eight is free as long as both operands
// agree: every lane takes 16 bytes of its row as they lie, and where these are 16 one-byte
// weights the two halves feed two instructions. Of the product it holds column (lane & 15),
// rows 4 * (lane >> 4) + 0..3.
//
// One-byte weights become the tokens' type, which holds every int8 and e4m3 value exactly, and
// products are summed in 32 bits. Values that were computed in 32 bits (hidden values of an
// expert, a token's low-rank values) go in as two bfloat16, the value rounded and what that
// leaves, 16 bits of mantissa together: rounding them to one would add as much error as the
// result's own type does. The matrix cores are idle most of the time here, since 16 columns
// take 128 weights a clock and CU and memory delivers about nine bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ec {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using u32x2 = __attribute__((ext_vector_type(2))) unsigned;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;

struct E4m3 {
  unsigned char v;
};
struct Bf16 {
  unsigned short v;
};
struct F16 {
  unsigned short v;
};

template <class A, class B>
__device__ __forceinline__ A bits_as(B b) {
  static_assert(sizeof(A) == sizeof(B));
  return __builtin_bit_cast(A, b);
}

// ---- scalars ------------------------------------------------------------------------------

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return bits_as<float>((unsigned)v.v << 16); }
__device__ __forceinline__ float to_f32(F16 v) { return (float)bits_as<_Float16>(v.v); }

template <class T>
__device__ __forceinline__ T from_f32(float f);  // to nearest, ties to even
template <>
__device__ __forceinline__ Bf16 from_f32<Bf16>(float f) {
  return Bf16{bits_as<unsigned short>((__bf16)f)};
}
template <>
__device__ __forceinline__ F16 from_f32<F16>(float f) {
  return F16{bits_as<unsigned short>((_Float16)f)};
}

// f as the sum of two bfloat16, exact to 2^-17 of f. An f that rounds to infinity, or is NaN,
// leaves nothing.
__device__ __forceinline__ void split_f32(float f, Bf16& hi, Bf16& lo) {
  hi = from_f32<Bf16>(f);
  const float rest = f - to_f32(hi);
  lo = from_f32<Bf16>((hi.v & 0x7F80) == 0x7F80 ? 0.f : rest);
}

// ---- eight weights as an operand ----------------------------------------------------------

template <class X>
struct Frag;
template <>
struct Frag<Bf16> {
  using V = bf16x8;
  static __device__ __forceinline__ f32x4 mfma(u32x4 w, u32x4 x, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits_as<V>(w), bits_as<V>(x), c, 0, 0, 0);
  }
};
template <>
struct Frag<F16> {
  using V = f16x8;
  static __device__ __forceinline__ f32x4 mfma(u32x4 w, u32x4 x, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(bits_as<V>(w), bits_as<V>(x), c, 0, 0, 0);
  }
};

// The upper halves of two floats whose lower halves are zero: two bfloat16.
__device__ __forceinline__ unsigned pack_high(float lo, float hi) {
  return __builtin_amdgcn_perm(bits_as<unsigned>(hi), bits_as<unsigned>(lo), 0x07060302u);
}

// Four int8 or e4m3 as four values of X.
template <class X, class W>
struct Widen;
template <>
struct Widen<Bf16, int8_t> {
  static __device__ __forceinline__ u32x2 four(unsigned w) {
    const float f0 = (float)(int8_t)(w), f1 = (float)(int8_t)(w >> 8);
    const float f2 = (float)(int8_t)(w >> 16), f3 = (float)((int)w >> 24);
    return u32x2{pack_high(f0, f1), pack_high(f2, f3)};
  }
};
template <>
struct Widen<F16, int8_t> {
  // 0x6400 | u is 1024 + u, with u = value + 128
  static __device__ __forceinline__ u32x2 four(unsigned w) {
    const unsigned u = w ^ 0x80808080u;
    const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    const unsigned a = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    const unsigned b = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    return u32x2{bits_as<unsigned>(bits_as<f16x2>(a) - bias),
                 bits_as<unsigned>(bits_as<f16x2>(b) - bias)};
  }
};
template <>
struct Widen<Bf16, E4m3> {
  static __device__ __forceinline__ u32x2 four(unsigned w) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true);
    return u32x2{bits_as<unsigned>(a), bits_as<unsigned>(b)};
  }
};
template <>
struct Widen<F16, E4m3> {
  static __device__ __forceinline__ u32x2 four(unsigned w) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    return u32x2{bits_as<unsigned>(a), bits_as<unsigned>(b)};
  }
};

// Operand `part` of the 16 bytes of weights a lane holds: eight values of X.
template <class X, class W>
__device__ __forceinline__ u32x4 operand(u32x4 w, int part) {
  if constexpr (sizeof(W) == 2) {
    return w;
  } else {
    const u32x2 a = Widen<X, W>::four(part ? w[2] : w[0]);
    const u32x2 b = Widen<X, W>::four(part ? w[3] : w[1]);
    return u32x4{a[0], a[1], b[0], b[1]};
  }
}

// Eight float16 as two operands of bfloat16 whose sum they are: bfloat16 has eight of
// float16's eleven bits, and the rest has at most four. The clamp turns what an infinity
// leaves (NaN) into something that adds nothing to it.
__device__ __forceinline__ void split_f16(u32x4 w, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 p = bits_as<f16x2>(w[i]);
    const float f0 = (float)p[0], f1 = (float)p[1];
    const float h0 = bits_as<float>(bits_as<unsigned>(f0) & 0xFFFF0000u);
    const float h1 = bits_as<float>(bits_as<unsigned>(f1) & 0xFFFF0000u);
    hi[i] = pack_high(f0, f1);
    lo[i] = pack_high(__builtin_amdgcn_fmed3f(f0 - h0, -512.f, 512.f),
                      __builtin_amdgcn_fmed3f(f1 - h1, -512.f, 512.f));
  }
}

// acc += weights (16 bytes of type W a lane) times values given as two bfloat16 operands.
template <class W>
__device__ __forceinline__ f32x4 mfma_split(u32x4 w, int part, u32x4 hi, u32x4 lo, f32x4 acc) {
  using B = Frag<Bf16>;
  if constexpr (sizeof(W) == 2 && !__is_same(W, Bf16)) {
    u32x4 wh, wl;
    split_f16(w, wh, wl);
    // wl * lo is up to 2^-15 of the product, more than what lo itself is off by
    acc = B::mfma(wl, lo, acc);
    acc = B::mfma(wl, hi, acc);
    acc = B::mfma(wh, lo, acc);
    return B::mfma(wh, hi, acc);
  } else {
    const u32x4 v = operand<Bf16, W>(w, part);
    acc = B::mfma(v, lo, acc);
    return B::mfma(v, hi, acc);
  }
}

// A product's result is in its registers eight wait states after it and nothing holds an earlier
// read back: the compiler counts them, but (clang 22 of ROCm 7.2) not for the first instruction of
// a block that two others lead to, and moves what reads a result behind a branch if one follows.
// So where a branch does: settled() keeps what was made of a result in its product's block, and
// products_done() stands before sums are read that products were added to up to a branch.
__device__ __forceinline__ void settled(f32x4& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void products_done() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 7");
  __builtin_amdgcn_sched_barrier(0);
}

// ---- memory -------------------------------------------------------------------------------

__device__ __forceinline__ u32x4 load16(const void* p) {
  return *static_cast<const u32x4*>(p);
}

// The same for what is read once: it need not stay in the caches.
template <bool ONCE>
__device__ __forceinline__ u32x4 load16_of(const void* p) {
  if constexpr (ONCE)
    return __builtin_nontemporal_load(static_cast<const u32x4*>(p));
  else
    return load16(p);
}

// What a kernel reads at an address that is the same in all lanes and that nothing writes while
// it runs: a scalar load, beside the vector loads and not in line with them.
template <class T>
__device__ __forceinline__ T load_uniform(const T* p) {
  using Constant = const __attribute__((address_space(4))) T;
  return *(Constant*)(reinterpret_cast<uintptr_t>(p));
}

// A routing or slot id of 4 or 8 bytes; out of [0, n) becomes -1. Both widths take the same two
// loads, so that nothing waits in a branch.
struct RawId {
  unsigned low, high;
};
__device__ __forceinline__ RawId raw_id(const void* ids, long long i, bool wide) {
  const unsigned* p = static_cast<const unsigned*>(ids) + (i << wide);
  return RawId{p[0], p[wide]};
}
__device__ __forceinline__ int id_of(RawId r, bool wide, int n) {
  const bool in = (r.low < (unsigned)n) & (!wide | (r.high == 0));
  return in ? (int)r.low : -1;
}
__device__ __forceinline__ int load_id(const void* ids, long long i, bool wide, int n) {
  return id_of(raw_id(ids, i, wide), wide, n);
}

// Two ids and a weight that were loaded before this point, all under way at once: without it
// the compiler moves a load to its first use, behind another one's wait.
__device__ __forceinline__ void together(RawId& a, RawId& b, float& w) {
  asm volatile("" : "+v"(a.low), "+v"(a.high), "+v"(b.low), "+v"(b.high), "+v"(w));
}

}  // namespace ec
