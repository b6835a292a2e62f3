// plstm_dropout.cu — dropout from a counter-based generator, with an optional residual.
//
// y[e] = [residual[e] +] (word(e) >= floor(p 2^32) ? x[e] / (1 - p) : 0).  The mask is a
// function of (seed, offset, e), so nothing is stored for the backward, which is the same
// kernel over dy.  One Philox call serves four consecutive elements, which is why a thread
// always takes whole groups of four.
#include <algorithm>

#include "plstm_ops.cuh"

namespace plstm {
namespace ops {
namespace {

constexpr int kThreads = 256;

// A thread takes kUnroll groups of eight elements a turn, a CTA's apart, and issues all their loads
// before it draws: with one 16-byte load in flight a thread the kernel waited on memory (68 to 69 us
// for 65.5 M f16 elements against 64 us; two groups take 65 to 69 us).  64 us is 63 % of the measured
// bandwidth: 20 widening products a Philox call keep the multiplier 62 % busy, issue is 57 %.  In f32 as many take
// 110 us, 73 %, and with a residual 154 us, 78 % (its four groups do not fit 64 registers: 168 bytes spill); f16 with
// a residual 73 us, 82 %.
constexpr int kUnroll = 4;

template <typename T>
struct Eight {
  static constexpr int P = 16 / (int)sizeof(T);
  Vec<T, P> p[8 / P];
  __device__ __forceinline__ void load(const T* from) {
#pragma unroll
    for (int q = 0; q < 8 / P; ++q) p[q] = load_vec<T, P>(from + q * P);
  }
  __device__ __forceinline__ float get(int k) const { return p[k / P].get(k % P); }
  __device__ __forceinline__ void store(T* to, const float (&f)[8]) {
#pragma unroll
    for (int q = 0; q < 8 / P; ++q) {
      float part[P];
#pragma unroll
      for (int k = 0; k < P; ++k) part[k] = f[q * P + k];
      p[q].set(part);
      store_vec<T, P>(to + q * P, p[q]);
    }
  }
};

// ALIGNED: all pointers are 16-byte aligned; else, and in the last n % 8 elements, one by one.
template <typename TX, typename TY, bool RESIDUAL, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 4) dropout_kernel(Drop d, int64_t n, const TX* __restrict__ x,
                                                              const TY* __restrict__ residual, TY* __restrict__ y) {
  const uint64_t seed = uniform_seed(d);
  const int64_t groups = (n + 7) / 8, whole = ALIGNED ? n / 8 : 0;
  for (int64_t first = blockIdx.x * (int64_t)(kThreads * kUnroll); first < groups;
       first += (int64_t)gridDim.x * (kThreads * kUnroll)) {
    // `first` and with it the upper word of its Philox block is the CTA's own; its lowest 10 bits are
    // zero, so the thread's place never carries into that word.
    const int64_t base = first + threadIdx.x;
    const uint32_t block = (uint32_t)(2 * first), block_hi = (uint32_t)(2 * first >> 32);
    Eight<TX> in[kUnroll];
    Eight<TY> res[RESIDUAL ? kUnroll : 1];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t g = base + u * kThreads;
      if (g < whole) {
        in[u].load(x + g * 8);
        if constexpr (RESIDUAL) res[u].load(residual + g * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t g = base + u * kThreads, e = g * 8;
      float v[8];
      if (g < whole) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = in[u].get(k);
        drop_eight(d, seed, block + 2 * (u * kThreads + threadIdx.x), block_hi, v);
        if constexpr (RESIDUAL) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(res[u].get(k), v[k]);
        }
        Eight<TY> out;
        out.store(y + e, v);
      } else if (g < groups) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = e + k < n ? to_f32(x[e + k]) : 0.0f;
        drop_eight(d, seed, block + 2 * (u * kThreads + threadIdx.x), block_hi, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (e + k < n) y[e + k] = from_f32<TY>(RESIDUAL ? __fadd_rn(to_f32(residual[e + k]), v[k]) : v[k]);
        }
      }
    }
  }
}

template <typename TX, typename TY>
int32_t launch(const Drop& d, int64_t n, const void* x, const void* residual, void* y, cudaStream_t s) {
  const int64_t turns = ((n + 7) / 8 + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  const int grid = (int)std::min<int64_t>(turns, kSMs * 4);
  const bool aligned = aligned16(x) && aligned16(y) && aligned16(residual);
  const auto kernel = residual != nullptr ? (aligned ? dropout_kernel<TX, TY, true, true> : dropout_kernel<TX, TY, true, false>)
                                          : (aligned ? dropout_kernel<TX, TY, false, true> : dropout_kernel<TX, TY, false, false>);
  kernel<<<grid, kThreads, 0, s>>>(d, n, static_cast<const TX*>(x), static_cast<const TY*>(residual),
                                   static_cast<TY*>(y));
  PLSTM_TRY_CUDA(cudaGetLastError());
  note_launches(1);
  return PLSTM_OK;
}

}  // namespace
}  // namespace ops
}  // namespace plstm

using namespace plstm;
using namespace plstm::ops;

extern "C" int32_t plstm_dropout(const plstm_dropout_desc* drop, int64_t n, const void* x, int32_t x_dtype,
                                 const void* residual, void* y, int32_t y_dtype, int32_t device, void* stream) {
  clear_error();
  PLSTM_CHECK_ARG(drop != nullptr, "plstm_dropout: the dropout descriptor is NULL");
  PLSTM_CHECK_ARG(n >= 0, "plstm_dropout: n must be >= 0");
  PLSTM_CHECK_ARG(dtype_ok(x_dtype) && dtype_ok(y_dtype), "plstm_dropout: bad dtype");
  PLSTM_CHECK_ARG(x_dtype == y_dtype || x_dtype == PLSTM_F32 || y_dtype == PLSTM_F32,
                  "plstm_dropout: x and y must have one type, or one of them f32");
  Drop d;
  if (const int32_t rc = make_drop(drop, &d)) return rc;
  if (n == 0) return PLSTM_OK;
  PLSTM_CHECK_ARG(x != nullptr && y != nullptr, "plstm_dropout: x and y must not be NULL");
  PLSTM_CHECK_ARG(aligned_to(x, dtype_size(x_dtype)) && aligned_to(y, dtype_size(y_dtype)) &&
                      aligned_to(residual, dtype_size(y_dtype)),
                  "plstm_dropout: a pointer is not aligned to its element");
  DeviceGuard guard;
  if (const int32_t rc = guard.enter(device)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == PLSTM_F32 && y_dtype == PLSTM_F32) return launch<float, float>(d, n, x, residual, y, s);
  if (x_dtype == PLSTM_F16 && y_dtype == PLSTM_F16) return launch<__half, __half>(d, n, x, residual, y, s);
  if (x_dtype == PLSTM_BF16 && y_dtype == PLSTM_BF16)
    return launch<__nv_bfloat16, __nv_bfloat16>(d, n, x, residual, y, s);
  if (x_dtype == PLSTM_F16) return launch<__half, float>(d, n, x, residual, y, s);
  if (x_dtype == PLSTM_BF16) return launch<__nv_bfloat16, float>(d, n, x, residual, y, s);
  if (y_dtype == PLSTM_F16) return launch<float, __half>(d, n, x, residual, y, s);
  return launch<float, __nv_bfloat16>(d, n, x, residual, y, s);
}
