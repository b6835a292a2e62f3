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

// E elements per thread and step (4 or 8), whole vectors; the last n % E elements one by one.
template <typename TX, typename TY, int E, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) dropout_kernel(Drop d, int64_t n, const TX* __restrict__ x,
                                                           const TY* __restrict__ residual, TY* __restrict__ y) {
  const uint64_t seed = drop_seed(d);
  const int64_t groups = (n + E - 1) / E;
  for (int64_t g = blockIdx.x * (int64_t)kThreads + threadIdx.x; g < groups; g += (int64_t)gridDim.x * kThreads) {
    const int64_t e = g * E;
    float v[E], r[E];
    const bool whole = ALIGNED && e + E <= n;
    if (whole) {
      constexpr int VX = 16 / sizeof(TX) < E ? 16 / sizeof(TX) : E, VY = 16 / sizeof(TY) < E ? 16 / sizeof(TY) : E;
#pragma unroll
      for (int k = 0; k < E; k += VX) {
        const Vec<TX, VX> in = load_vec<TX, VX>(x + e + k);
#pragma unroll
        for (int j = 0; j < VX; ++j) v[k + j] = in.get(j);
      }
      if (residual != nullptr) {
#pragma unroll
        for (int k = 0; k < E; k += VY) {
          const Vec<TY, VY> in = load_vec<TY, VY>(residual + e + k);
#pragma unroll
          for (int j = 0; j < VY; ++j) r[k + j] = in.get(j);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const bool in = e + k < n;
        v[k] = in ? to_f32(x[e + k]) : 0.0f;
        r[k] = in && residual != nullptr ? to_f32(residual[e + k]) : 0.0f;
      }
    }
    drop_vec<E>(d, seed, e, v);
    if (residual != nullptr) {
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = __fadd_rn(r[k], v[k]);
    }
    if (whole) {
      constexpr int VY = 16 / sizeof(TY) < E ? 16 / sizeof(TY) : E;
#pragma unroll
      for (int k = 0; k < E; k += VY) {
        float part[VY];
#pragma unroll
        for (int j = 0; j < VY; ++j) part[j] = v[k + j];
        Vec<TY, VY> out;
        out.set(part);
        store_vec<TY, VY>(y + e + k, out);
      }
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (e + k < n) y[e + k] = from_f32<TY>(v[k]);
    }
  }
}

template <typename TX, typename TY>
int32_t launch(const Drop& d, int64_t n, const void* x, const void* residual, void* y, cudaStream_t s) {
  constexpr int E = sizeof(TX) == 2 || sizeof(TY) == 2 ? 8 : 4;
  const int64_t groups = (n + E - 1) / E;
  const int grid = (int)std::min<int64_t>((groups + kThreads - 1) / kThreads, kSMs * 8);
  if (aligned16(x) && aligned16(y) && aligned16(residual))
    dropout_kernel<TX, TY, E, true><<<grid, kThreads, 0, s>>>(
        d, n, static_cast<const TX*>(x), static_cast<const TY*>(residual), static_cast<TY*>(y));
  else
    dropout_kernel<TX, TY, E, false><<<grid, kThreads, 0, s>>>(
        d, n, static_cast<const TX*>(x), static_cast<const TY*>(residual), static_cast<TY*>(y));
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
