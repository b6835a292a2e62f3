// plstm_ops.cuh — shared device code of the training and streaming operators
// (plstm_scan.cu, plstm_norm.cu, plstm_dropout.cu).
#pragma once

#include <type_traits>

#include "plstm_common.cuh"

namespace plstm {
namespace ops {

constexpr int kSMs = 148;  // B200

// N bytes moved by one load or store.
template <int N>
struct Word;
template <>
struct Word<2> {
  using type = unsigned short;
};
template <>
struct Word<4> {
  using type = uint32_t;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<16> {
  using type = uint4;
};

// V consecutive elements as they lie in memory, moved by one instruction (V * sizeof(T) <= 16).
template <typename T, int V>
struct Vec {
  union {
    typename Word<V * sizeof(T)>::type word;
    uint32_t w[V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1];
  };
  __device__ __forceinline__ float get(int k) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[k]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      // bf16 is the upper half of an f32.
      if constexpr (V == 1) return __uint_as_float((uint32_t)word << 16);
      return __uint_as_float(k & 1 ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
    } else {
      if constexpr (V == 1) return __half2float(__ushort_as_half(word));
      return __half2float(__ushort_as_half((unsigned short)(k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xffffu)));
    }
  }
  // Rounds all V values to nearest even.
  __device__ __forceinline__ void set(const float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < V; ++k) w[k] = __float_as_uint(f[k]);
    } else if constexpr (V == 1) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>)
        word = __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
      else
        word = __half_as_ushort(__float2half_rn(f[0]));
    } else {
#pragma unroll
      for (int k = 0; k < V; k += 2) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(f[k], f[k + 1]);
          w[k >> 1] = *reinterpret_cast<const uint32_t*>(&p);
        } else {
          const __half2 p = __floats2half2_rn(f[k], f[k + 1]);
          w[k >> 1] = *reinterpret_cast<const uint32_t*>(&p);
        }
      }
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  Vec<T, V> v;
  v.word = *reinterpret_cast<const typename Word<V * sizeof(T)>::type*>(p);
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& v) {
  *reinterpret_cast<typename Word<V * sizeof(T)>::type*>(p) = v.word;
}

// 1 / sqrt(a): the hardware's approximation and one Newton step.  a r comes first: half of a subnormal a is
// rounded, of the smallest to zero.
__device__ __forceinline__ float rsqrt_rn(float a) {
  const float r = rsqrtf(a);
  return a > 0.0f && a < INFINITY ? r * fmaf(-0.5f * (a * r), r, 1.5f) : r;
}

inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
inline bool dtype_ok(int32_t dt) { return dt == PLSTM_F32 || dt == PLSTM_F16 || dt == PLSTM_BF16; }

// ---- packed arithmetic -------------------------------------------------------------------------
// V neighbouring f32 values.  Two of them go through the f32x2 instructions, which do
// two operations for one issue slot; the special-function unit takes them one by one.
template <int V>
struct F;
template <>
struct F<1> {
  float x;
  __device__ __forceinline__ float get(int) const { return x; }
  static __device__ __forceinline__ F of(float a) { return {a}; }
  static __device__ __forceinline__ F of(const float (&a)[1]) { return {a[0]}; }
};
template <>
struct F<2> {
  float x, y;
  __device__ __forceinline__ float get(int k) const { return k ? y : x; }
  static __device__ __forceinline__ F of(float lo, float hi) { return {lo, hi}; }
  static __device__ __forceinline__ F of(float a) { return {a, a}; }
  static __device__ __forceinline__ F of(const float (&a)[2]) { return {a[0], a[1]}; }
};
__device__ __forceinline__ F<1> fma(F<1> a, F<1> b, F<1> c) { return {fmaf(a.x, b.x, c.x)}; }
__device__ __forceinline__ F<1> operator*(F<1> a, F<1> b) { return {a.x * b.x}; }
__device__ __forceinline__ F<1> operator+(F<1> a, F<1> b) { return {a.x + b.x}; }
__device__ __forceinline__ F<2> fma(F<2> a, F<2> b, F<2> c) {
  F<2> r;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ F<2> operator*(F<2> a, F<2> b) {
  F<2> r;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\n"
      "mov.b64 {%0, %1}, d;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ F<2> operator+(F<2> a, F<2> b) {
  F<2> r;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\n"
      "mov.b64 {%0, %1}, d;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
template <int V, typename Fn>
__device__ __forceinline__ F<V> each(F<V> a, Fn fn) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = fn(a.get(k));
  return F<V>::of(r);
}
// a * b + 1 and the like with a constant in every lane.
template <int V>
__device__ __forceinline__ F<V> fma(F<V> a, F<V> b, float c) { return fma(a, b, F<V>::of(c)); }
template <int V>
__device__ __forceinline__ F<V> one_plus(F<V> a) { return a + F<V>::of(1.0f); }
template <int V>
__device__ __forceinline__ F<V> one_minus(F<V> a) { return fma(a, F<V>::of(-1.0f), F<V>::of(1.0f)); }

// ---- Philox4x32-10 ------------------------------------------------------------------------
// Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3" (SC 2011): ten
// rounds of two 32 x 32 -> 64-bit products and key additions (Weyl sequence) on a 128-bit
// counter.  One call gives the words of four consecutive elements.
// `seed` comes as a warp-uniform value (uniform_seed), so the round keys cost no vector operations.
// The products are asked for as one widening instruction each: from a 64-bit product in C the compiler
// makes two (65 instructions a call against 47, 36 us against 27 us for 8.4 M calls).  Where the
// block's upper word is warp-uniform too, two of the 20 products are hoisted out of the caller's loop.
__device__ __forceinline__ void mul_wide(uint32_t a, uint32_t b, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .u64 t;\nmul.wide.u32 t, %2, %3;\nmov.b64 {%0, %1}, t;\n}" : "=r"(lo), "=r"(hi) : "r"(a), "r"(b));
}
__device__ __forceinline__ uint4 philox(uint32_t block_lo, uint32_t block_hi, uint64_t offset, uint64_t seed) {
  uint32_t c0 = block_lo, c1 = block_hi, c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    uint32_t a_lo, a_hi, b_lo, b_hi;
    mul_wide(c0, 0xD2511F53u, a_lo, a_hi);
    mul_wide(c2, 0xCD9E8D57u, b_lo, b_hi);
    c0 = b_hi ^ c1 ^ k0;
    c1 = b_lo;
    c2 = a_hi ^ c3 ^ k1;
    c3 = a_lo;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// A dropout call as the kernels take it.
struct Drop {
  uint64_t seed, offset;
  const uint64_t* seed_ptr;
  uint32_t threshold;  // keep where word >= threshold
  float scale;
  int mode;            // 0: keep everything, 1: draw, 2: drop everything (p = 1)
};

// The seed, from the descriptor or from the GPU's memory.  Every lane holds the same value; the
// reductions tell the compiler so.  All lanes of the warp have to call this.
__device__ __forceinline__ uint64_t uniform_seed(const Drop& d) {
  const uint64_t s = d.seed_ptr != nullptr ? *d.seed_ptr : d.seed;
  const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)s), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(s >> 32));
  return (uint64_t)hi << 32 | lo;
}

// Applies the dropout to the eight elements of the Philox blocks (lo, hi) and (lo + 1, hi), lo even:
// x / (1 - p) where the word keeps the element, else 0 (whatever x is).  The products are instructions of
// their own (f32x2, each rounded), never contracted with a later sum, so that the fused and the separate
// calls give the same bits.
__device__ __forceinline__ void drop_eight(const Drop& d, uint64_t seed, uint32_t lo, uint32_t hi, float (&x)[8]) {
  if (d.mode == 0) return;
  if (d.mode == 2) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.0f;
    return;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint4 w = philox(lo + q, hi, d.offset, seed);
    const F<2> a = F<2>::of(x[4 * q], x[4 * q + 1]) * F<2>::of(d.scale);
    const F<2> b = F<2>::of(x[4 * q + 2], x[4 * q + 3]) * F<2>::of(d.scale);
    x[4 * q] = w.x >= d.threshold ? a.x : 0.0f;
    x[4 * q + 1] = w.y >= d.threshold ? a.y : 0.0f;
    x[4 * q + 2] = w.z >= d.threshold ? b.x : 0.0f;
    x[4 * q + 3] = w.w >= d.threshold ? b.y : 0.0f;
  }
}

// Checks a descriptor and fills the kernel's form of it (NULL: no dropout).
inline int32_t make_drop(const plstm_dropout_desc* d, Drop* out) {
  *out = Drop{0, 0, nullptr, 0, 1.0f, 0};
  if (d == nullptr) return PLSTM_OK;
  PLSTM_CHECK_ARG(d->p >= 0.0 && d->p <= 1.0, "dropout: p must be in [0, 1]");
  out->seed = d->seed;
  out->offset = d->offset;
  out->seed_ptr = d->seed_ptr;
  PLSTM_CHECK_ARG(aligned_to(d->seed_ptr, 8), "dropout: seed_ptr must be 8-byte aligned");
  if (d->p == 0.0) return PLSTM_OK;
  if (d->p == 1.0) {
    out->mode = 2;
    return PLSTM_OK;
  }
  out->mode = 1;
  out->threshold = (uint32_t)(d->p * 4294967296.0);
  out->scale = (float)(1.0 / (1.0 - d->p));
  return PLSTM_OK;
}

}  // namespace ops
}  // namespace plstm
