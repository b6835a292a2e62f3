// plstm_norm.cu — layer norm over the last axis, forward and backward, plain or fused with
// the residual step z = residual + dropout(x) in front of it.
//
// Forward, per row: mean, then the centred sum of squares (two passes over registers, so no
// cancellation for rows far from zero), then y = (v - mean) rstd w + b.
// Backward, with xh = (v - mean) rstd and g = dy w:
//   dv = rstd (g - mean(g) - xh mean(g xh)) [+ dz],  dw = sum over rows of dy xh,  db = sum of dy.
// The weight gradients are summed per thread over the rows its CTA visits, then over the
// CTA's row groups, then over the CTAs by a second kernel: a fixed order, no atomics.
#include <algorithm>

#include "plstm_ops.cuh"

namespace plstm {
namespace ops {
namespace {

constexpr int kGroupThreads = 256;  // CTA size when a row takes at most one warp

// The widest CTA make_split gives a variant: 16384 columns in chunks of 8 x 4 or of 4 x 4 and less.
constexpr int max_threads(int v) { return v == 8 ? 512 : 1024; }

// How a row of N elements is spread over threads: `tpr` threads take chunks of V elements,
// chunk c of thread t starting at column (c * tpr + t) * V; a thread has CH chunks.
struct Split {
  int v, ch, tpr, block;
};

struct NormArgs {
  int64_t rows;
  int cols, tpr;
  float eps;
  int64_t x_stride, res_stride, dy_stride, dz_stride;
  const void *x, *residual, *dy, *dz, *v, *weight, *bias;
  void *z, *y, *dx, *dres;
  float* mean;
  float* rstd;
  float* partial;
  int w_dtype;
  Drop drop;
};

// Sum over the `tpr` threads of a row (a power of two up to 32, or the whole CTA).
template <int NV>
__device__ __forceinline__ void row_sum(float (&a)[NV], int tpr, float* scratch) {
  for (int o = min(tpr, 32) >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k) a[k] += __shfl_xor_sync(0xffffffffu, a[k], o);
  }
  if (tpr <= 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = tpr >> 5;
  __syncthreads();  // the scratch of the previous sum has been read
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) scratch[k * 32 + warp] = a[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    a[k] = lane < warps ? scratch[k * 32 + lane] : 0.0f;
    for (int o = 16; o > 0; o >>= 1) a[k] += __shfl_xor_sync(0xffffffffu, a[k], o);
  }
}

// V elements of a weight that has x's type or f32 (NULL: `none`).  V > 1 needs 16-byte aligned weights.
template <typename TX, int V>
__device__ __forceinline__ void load_weight(const void* w, int dtype, int col, float none, float (&out)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = none;
  } else if (sizeof(TX) == 4 || dtype == PLSTM_F32) {
    constexpr int VW = V < 4 ? V : 4;
#pragma unroll
    for (int q = 0; q < V; q += VW) {
      const Vec<float, VW> in = load_vec<float, VW>(static_cast<const float*>(w) + col + q);
#pragma unroll
      for (int k = 0; k < VW; ++k) out[q + k] = in.get(k);
    }
  } else {
    const Vec<TX, V> in = load_vec<TX, V>(static_cast<const TX*>(w) + col);
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = in.get(k);
  }
}

template <typename TX, typename TZ, int V, int CH, bool FUSED>
__global__ void __launch_bounds__(max_threads(V)) norm_forward_kernel(NormArgs a) {
  __shared__ float scratch[64];
  const int tpr = a.tpr, lane = threadIdx.x % tpr;
  const int rows_per_cta = blockDim.x / tpr;
  const uint64_t seed = FUSED ? drop_seed(a.drop) : 0;
  const float inv_n = 1.0f / (float)a.cols;
  // Every thread of a warp takes every turn (the sums shuffle over the whole warp).
  for (int64_t row0 = (int64_t)blockIdx.x * rows_per_cta; row0 < a.rows; row0 += (int64_t)gridDim.x * rows_per_cta) {
    const int64_t row = row0 + threadIdx.x / tpr;
    const bool live = row < a.rows;
    float v[CH][V];
    float sum[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * tpr + lane) * V;
      if (live && col < a.cols) {
        const Vec<TX, V> in = load_vec<TX, V>(static_cast<const TX*>(a.x) + row * a.x_stride + col);
#pragma unroll
        for (int k = 0; k < V; ++k) v[c][k] = in.get(k);
        if constexpr (FUSED) {
          const int64_t e = row * a.cols + col;
          drop_vec<V>(a.drop, seed, e, v[c]);
          const TZ* res = static_cast<const TZ*>(a.residual) + row * a.res_stride + col;
          constexpr int VZ = 16 / sizeof(TZ) < V ? 16 / sizeof(TZ) : V;
#pragma unroll
          for (int q = 0; q < V; q += VZ) {
            const Vec<TZ, VZ> r = load_vec<TZ, VZ>(res + q);
            float part[VZ];
#pragma unroll
            for (int k = 0; k < VZ; ++k) part[k] = __fadd_rn(r.get(k), v[c][q + k]);
            Vec<TZ, VZ> z;
            z.set(part);
#pragma unroll
            for (int k = 0; k < VZ; ++k) v[c][q + k] = z.get(k);  // the norm is of z as stored
            store_vec<TZ, VZ>(static_cast<TZ*>(a.z) + e + q, z);
          }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) sum[0] += v[c][k];
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[c][k] = 0.0f;
      }
    }
    row_sum<1>(sum, tpr, scratch);
    const float mean = sum[0] * inv_n;
    float sq[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if ((c * tpr + lane) * V < a.cols) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          v[c][k] -= mean;
          sq[0] += v[c][k] * v[c][k];
        }
      }
    }
    row_sum<1>(sq, tpr, scratch);
    const float rstd = 1.0f / sqrtf(sq[0] * inv_n + a.eps);
    if (!live) continue;
    if (a.mean != nullptr && lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * tpr + lane) * V;
      if (col < a.cols) {
        float w[V], b[V];
        load_weight<TX, V>(a.weight, a.w_dtype, col, 1.0f, w);
        load_weight<TX, V>(a.bias, a.w_dtype, col, 0.0f, b);
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] = v[c][k] * rstd * w[k] + b[k];
        Vec<TX, V> out;
        out.set(w);
        store_vec<TX, V>(static_cast<TX*>(a.y) + row * a.cols + col, out);
      }
    }
  }
}

// TV: the normalised tensor's type (x or z).  partial [gridDim.x][2][cols], or NULL.
template <typename TX, typename TV, int V, int CH, bool FUSED>
__global__ void __launch_bounds__(max_threads(V)) norm_backward_kernel(NormArgs a) {
  extern __shared__ float acc[];  // [2][cols] when a CTA holds several row groups
  __shared__ float scratch[64];
  const int tpr = a.tpr, lane = threadIdx.x % tpr;
  const int rows_per_cta = blockDim.x / tpr;
  const uint64_t seed = FUSED ? drop_seed(a.drop) : 0;
  const float inv_n = 1.0f / (float)a.cols;
  const int64_t v_stride = FUSED ? (int64_t)a.cols : a.x_stride;
  constexpr int VV = 16 / sizeof(TV) < V ? 16 / sizeof(TV) : V;
  float dw[CH][V], db[CH][V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int k = 0; k < V; ++k) dw[c][k] = db[c][k] = 0.0f;
  }
  for (int64_t row0 = (int64_t)blockIdx.x * rows_per_cta; row0 < a.rows; row0 += (int64_t)gridDim.x * rows_per_cta) {
    const int64_t row = row0 + threadIdx.x / tpr;
    const bool live = row < a.rows;
    float xh[CH][V], g[CH][V];
    float s[2] = {0.0f, 0.0f};
    const float mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * tpr + lane) * V;
      if (live && col < a.cols) {
        const Vec<TX, V> dy = load_vec<TX, V>(static_cast<const TX*>(a.dy) + row * a.dy_stride + col);
#pragma unroll
        for (int q = 0; q < V; q += VV) {
          const Vec<TV, VV> in = load_vec<TV, VV>(static_cast<const TV*>(a.v) + row * v_stride + col + q);
#pragma unroll
          for (int k = 0; k < VV; ++k) xh[c][q + k] = (in.get(k) - mean) * rstd;
        }
        float w[V];
        load_weight<TX, V>(a.weight, a.w_dtype, col, 1.0f, w);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = dy.get(k);
          dw[c][k] += d * xh[c][k];
          db[c][k] += d;
          g[c][k] = d * w[k];
          s[0] += g[c][k];
          s[1] += g[c][k] * xh[c][k];
        }
      }
    }
    row_sum<2>(s, tpr, scratch);
    if (!live) continue;
    const float m1 = s[0] * inv_n, m2 = s[1] * inv_n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * tpr + lane) * V;
      if (col < a.cols) {
        const int64_t e = row * a.cols + col;
        float dv[V];
#pragma unroll
        for (int k = 0; k < V; ++k) dv[k] = rstd * (g[c][k] - m1 - xh[c][k] * m2);
        if constexpr (FUSED) {
          if (a.dz != nullptr) {
#pragma unroll
            for (int q = 0; q < V; q += VV) {
              const Vec<TV, VV> dz = load_vec<TV, VV>(static_cast<const TV*>(a.dz) + row * a.dz_stride + col + q);
#pragma unroll
              for (int k = 0; k < VV; ++k) dv[q + k] += dz.get(k);
            }
          }
          if (a.dres != nullptr) {
#pragma unroll
            for (int q = 0; q < V; q += VV) {
              float part[VV];
#pragma unroll
              for (int k = 0; k < VV; ++k) part[k] = dv[q + k];
              Vec<TV, VV> out;
              out.set(part);
              store_vec<TV, VV>(static_cast<TV*>(a.dres) + e + q, out);
            }
          }
          if (a.dx == nullptr) continue;
          drop_vec<V>(a.drop, seed, e, dv);
        }
        if (a.dx != nullptr) {
          Vec<TX, V> out;
          out.set(dv);
          store_vec<TX, V>(static_cast<TX*>(a.dx) + e, out);
        }
      }
    }
  }
  if (a.partial == nullptr) return;
  float* to = a.partial + (int64_t)blockIdx.x * 2 * a.cols;
  if (tpr >= 32 && rows_per_cta == 1) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * tpr + lane) * V;
      if (col < a.cols) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          to[col + k] = dw[c][k];
          to[a.cols + col + k] = db[c][k];
        }
      }
    }
    return;
  }
  // Row groups within a warp, then the warps one after the other.
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      for (int o = tpr; o < 32; o <<= 1) {
        dw[c][k] += __shfl_xor_sync(0xffffffffu, dw[c][k], o);
        db[c][k] += __shfl_xor_sync(0xffffffffu, db[c][k], o);
      }
    }
  }
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int w = 0; w < warps; ++w) {
    if (warp == w && (int)(threadIdx.x & 31) < tpr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (c * tpr + lane) * V;
        if (col < a.cols) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            acc[col + k] = (w > 0 ? acc[col + k] : 0.0f) + dw[c][k];
            acc[a.cols + col + k] = (w > 0 ? acc[a.cols + col + k] : 0.0f) + db[c][k];
          }
        }
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) to[i] = acc[i];
}

// dweight / dbias from the CTAs' partial sums [parts][2][cols]: 32 columns per CTA, 32 threads
// deep over the parts, then a fixed tree.
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* __restrict__ partial, int parts, int cols,
                                                                void* dweight, void* dbias, int w_dtype) {
  __shared__ float sums[32][33];
  const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (col < cols)
    for (int p = threadIdx.y; p < parts; p += 32) s += partial[((int64_t)p * 2 + which) * cols + col];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sums[threadIdx.x][threadIdx.y];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  void* out = which == 0 ? dweight : dbias;
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < cols && out != nullptr) store_any(out, w_dtype, c, s);
}

// Vectors of 16 bytes of x where every row allows them, else single elements.
Split make_split(const plstm_norm_desc& d, bool vec_ok) {
  Split s;
  s.v = vec_ok ? 16 / (int)dtype_size(d.x_dtype) : 1;
  const int chunks = (d.cols + s.v - 1) / s.v;
  s.tpr = 1;
  while (s.tpr < 32 && s.tpr < chunks) s.tpr *= 2;
  s.ch = 1;
  while (s.ch < 4 && s.ch * s.tpr < chunks) s.ch *= 2;
  while (s.tpr < 1024 && s.ch * s.tpr < chunks) s.tpr *= 2;
  if (s.ch * s.tpr < chunks) s.ch = 16;  // single elements, more than 4096 columns
  s.block = s.tpr <= 32 ? kGroupThreads : s.tpr;
  return s;
}

int64_t row_ctas(const plstm_norm_desc& d, const Split& s, int per_sm) {
  const int64_t per_cta = s.block / s.tpr;
  return std::min<int64_t>((d.rows + per_cta - 1) / per_cta, (int64_t)kSMs * per_sm);
}

int backward_per_sm(const Split& s) { return s.block >= 1024 ? 1 : s.block >= 512 ? 2 : s.block == 256 ? 2 : 4; }

template <typename TX, typename TZ, int V, int CH>
void launch_forward(const NormArgs& a, const Split& s, int grid, bool fused, cudaStream_t st) {
  if (fused)
    norm_forward_kernel<TX, TZ, V, CH, true><<<grid, s.block, 0, st>>>(a);
  else if constexpr (sizeof(TX) == sizeof(TZ))
    norm_forward_kernel<TX, TZ, V, CH, false><<<grid, s.block, 0, st>>>(a);
}

template <typename TX, typename TZ, int V, int CH>
void launch_backward(const NormArgs& a, const Split& s, int grid, bool fused, cudaStream_t st) {
  const size_t smem = s.block > s.tpr ? (size_t)a.cols * 2 * sizeof(float) : 0;
  if (fused)
    norm_backward_kernel<TX, TZ, V, CH, true><<<grid, s.block, smem, st>>>(a);
  else if constexpr (sizeof(TX) == sizeof(TZ))
    norm_backward_kernel<TX, TZ, V, CH, false><<<grid, s.block, smem, st>>>(a);
}

template <typename TX, typename TZ>
void dispatch(bool backward, const NormArgs& a, const Split& s, int grid, bool fused, cudaStream_t st) {
  constexpr int VF = 16 / sizeof(TX);
#define PLSTM_NORM_CASE(V, CH)                                              \
  if (s.v == V && s.ch == CH) {                                             \
    if (backward)                                                           \
      launch_backward<TX, TZ, V, CH>(a, s, grid, fused, st);                \
    else                                                                    \
      launch_forward<TX, TZ, V, CH>(a, s, grid, fused, st);                 \
    return;                                                                 \
  }
  PLSTM_NORM_CASE(VF, 1)
  PLSTM_NORM_CASE(VF, 2)
  PLSTM_NORM_CASE(VF, 4)
  PLSTM_NORM_CASE(1, 1)
  PLSTM_NORM_CASE(1, 2)
  PLSTM_NORM_CASE(1, 4)
  PLSTM_NORM_CASE(1, 16)
#undef PLSTM_NORM_CASE
}

void dispatch_types(bool backward, const plstm_norm_desc& d, const NormArgs& a, const Split& s, int grid, bool fused,
                    cudaStream_t st) {
  if (d.x_dtype == PLSTM_F32)
    dispatch<float, float>(backward, a, s, grid, fused, st);
  else if (d.x_dtype == PLSTM_F16 && d.z_dtype == PLSTM_F16)
    dispatch<__half, __half>(backward, a, s, grid, fused, st);
  else if (d.x_dtype == PLSTM_F16)
    dispatch<__half, float>(backward, a, s, grid, fused, st);
  else if (d.z_dtype == PLSTM_BF16)
    dispatch<__nv_bfloat16, __nv_bfloat16>(backward, a, s, grid, fused, st);
  else
    dispatch<__nv_bfloat16, float>(backward, a, s, grid, fused, st);
}

int32_t check_desc(const plstm_norm_desc* d, bool fused) {
  PLSTM_CHECK_ARG(d != nullptr, "layer norm: the descriptor is NULL");
  PLSTM_CHECK_ARG(d->rows >= 0, "layer norm: rows must be >= 0");
  PLSTM_CHECK_ARG(d->cols >= 1 && d->cols <= PLSTM_NORM_MAX_COLS, "layer norm: cols must be in [1, 16384]");
  PLSTM_CHECK_ARG(dtype_ok(d->x_dtype) && dtype_ok(d->z_dtype) && dtype_ok(d->w_dtype), "layer norm: bad dtype");
  PLSTM_CHECK_ARG(d->z_dtype == d->x_dtype || (fused && d->z_dtype == PLSTM_F32),
                  "layer norm: z_dtype must be x_dtype, or f32 with a residual");
  PLSTM_CHECK_ARG(d->w_dtype == d->x_dtype || d->w_dtype == PLSTM_F32, "layer norm: w_dtype must be x_dtype or f32");
  PLSTM_CHECK_ARG(d->eps >= 0.0f, "layer norm: eps must be >= 0");
  PLSTM_CHECK_ARG(d->x_stride >= 0 && d->residual_stride >= 0 && d->dy_stride >= 0 && d->dz_stride >= 0,
                  "layer norm: strides must be >= 0");
  return PLSTM_OK;
}

// Every row of the tensor starts on a 16-byte boundary.
bool rows16(const void* p, int64_t stride, int32_t dtype) {
  return p == nullptr || (aligned16(p) && stride * (int64_t)dtype_size(dtype) % 16 == 0);
}

}  // namespace
}  // namespace ops
}  // namespace plstm

using namespace plstm;
using namespace plstm::ops;

extern "C" {

int32_t plstm_layer_norm_forward(const plstm_norm_desc* d, const plstm_dropout_desc* drop, const void* x,
                                 const void* residual, const void* weight, const void* bias, void* z, void* y,
                                 float* stats, void* stream) {
  clear_error();
  const bool fused = residual != nullptr;
  if (const int32_t rc = check_desc(d, fused)) return rc;
  PLSTM_CHECK_ARG(fused || drop == nullptr, "layer norm: dropout needs a residual");
  NormArgs a{};
  if (const int32_t rc = make_drop(drop, &a.drop)) return rc;
  if (d->rows == 0) return PLSTM_OK;
  PLSTM_CHECK_ARG(x != nullptr && y != nullptr && (!fused || z != nullptr), "layer norm: x, y and z must not be NULL");
  const size_t xs = dtype_size(d->x_dtype), zs = dtype_size(d->z_dtype), wsz = dtype_size(d->w_dtype);
  PLSTM_CHECK_ARG(aligned_to(x, xs) && aligned_to(y, xs) && aligned_to(residual, zs) && aligned_to(z, zs) &&
                      aligned_to(weight, wsz) && aligned_to(bias, wsz) && aligned_to(stats, 4),
                  "layer norm: a pointer is not aligned to its element");
  DeviceGuard guard;
  if (const int32_t rc = guard.enter(d->device)) return rc;
  const bool vec = d->cols % (16 / xs) == 0 && rows16(x, d->x_stride, d->x_dtype) && aligned16(y) &&
                   rows16(residual, d->residual_stride, d->z_dtype) && aligned16(z) && aligned16(weight) &&
                   aligned16(bias);
  const Split s = make_split(*d, vec);
  a.rows = d->rows;
  a.cols = d->cols;
  a.tpr = s.tpr;
  a.eps = d->eps;
  a.x_stride = d->x_stride;
  a.res_stride = d->residual_stride;
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.bias = bias;
  a.z = z;
  a.y = y;
  a.mean = stats;
  a.rstd = stats != nullptr ? stats + d->rows : nullptr;
  a.w_dtype = d->w_dtype;
  dispatch_types(false, *d, a, s, (int)row_ctas(*d, s, 2048 / s.block), fused, static_cast<cudaStream_t>(stream));
  PLSTM_TRY_CUDA(cudaGetLastError());
  note_launches(1);
  return PLSTM_OK;
}

int32_t plstm_layer_norm_backward_workspace_size(const plstm_norm_desc* d, size_t* bytes) {
  clear_error();
  PLSTM_CHECK_ARG(bytes != nullptr, "bytes is NULL");
  if (const int32_t rc = check_desc(d, true)) return rc;
  // The larger of the two splits that alignment chooses between.
  const Split s0 = make_split(*d, false), s1 = make_split(*d, true);
  const int64_t parts = std::max(row_ctas(*d, s0, backward_per_sm(s0)), row_ctas(*d, s1, backward_per_sm(s1)));
  *bytes = (size_t)parts * 2 * (size_t)d->cols * sizeof(float);
  return PLSTM_OK;
}

int32_t plstm_layer_norm_backward(const plstm_norm_desc* d, const plstm_dropout_desc* drop, int32_t fused,
                                  const void* dy, const void* dz, const void* v, const void* weight,
                                  const float* stats, void* dx, void* dresidual, void* dweight, void* dbias,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int32_t rc = check_desc(d, fused != 0)) return rc;
  PLSTM_CHECK_ARG(fused || (drop == nullptr && dz == nullptr && dresidual == nullptr),
                  "layer norm backward: dropout, dz and dresidual need `fused`");
  NormArgs a{};
  if (const int32_t rc = make_drop(drop, &a.drop)) return rc;
  const bool grads = dweight != nullptr || dbias != nullptr;
  if (d->rows > 0) {
    PLSTM_CHECK_ARG(dy != nullptr && v != nullptr && stats != nullptr,
                    "layer norm backward: dy, v and stats must not be NULL");
    if (grads) {
      size_t need = 0;
      if (const int32_t rc = plstm_layer_norm_backward_workspace_size(d, &need)) return rc;
      PLSTM_CHECK_ARG(workspace != nullptr && aligned16(workspace),
                      "layer norm backward: workspace must not be NULL and must be 16-byte aligned");
      if (workspace_bytes < need) {
        set_error("layer norm backward: workspace smaller than plstm_layer_norm_backward_workspace_size");
        return PLSTM_EWORKSPACE;
      }
    }
  }
  const size_t xs = dtype_size(d->x_dtype), zs = dtype_size(d->z_dtype), wsz = dtype_size(d->w_dtype);
  PLSTM_CHECK_ARG(aligned_to(dy, xs) && aligned_to(dx, xs) && aligned_to(dz, zs) && aligned_to(v, zs) &&
                      aligned_to(dresidual, zs) && aligned_to(weight, wsz) && aligned_to(dweight, wsz) &&
                      aligned_to(dbias, wsz) && aligned_to(stats, 4),
                  "layer norm backward: a pointer is not aligned to its element");
  DeviceGuard guard;
  if (const int32_t rc = guard.enter(d->device)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int parts = 0;
  if (d->rows > 0 && (grads || dx != nullptr || dresidual != nullptr)) {
    const bool vec = d->cols % (16 / xs) == 0 && rows16(dy, d->dy_stride, d->x_dtype) &&
                     rows16(v, fused ? d->cols : d->x_stride, d->z_dtype) && rows16(dz, d->dz_stride, d->z_dtype) &&
                     aligned16(dx) && aligned16(dresidual) && aligned16(weight);
    const Split s = make_split(*d, vec);
    parts = (int)row_ctas(*d, s, backward_per_sm(s));
    a.rows = d->rows;
    a.cols = d->cols;
    a.tpr = s.tpr;
    a.x_stride = d->x_stride;
    a.dy_stride = d->dy_stride;
    a.dz_stride = d->dz_stride;
    a.dy = dy;
    a.dz = dz;
    a.v = v;
    a.weight = weight;
    a.dx = dx;
    a.dres = dresidual;
    a.mean = const_cast<float*>(stats);
    a.rstd = const_cast<float*>(stats) + d->rows;
    a.partial = grads ? static_cast<float*>(workspace) : nullptr;
    a.w_dtype = d->w_dtype;
    dispatch_types(true, *d, a, s, parts, fused != 0, st);
    PLSTM_TRY_CUDA(cudaGetLastError());
    note_launches(1);
  }
  if (grads) {
    norm_weight_grad_kernel<<<dim3((d->cols + 31) / 32, 2), dim3(32, 32), 0, st>>>(
        static_cast<const float*>(workspace), parts, d->cols, dweight, dbias, d->w_dtype);
    PLSTM_TRY_CUDA(cudaGetLastError());
    note_launches(1);
  }
  return PLSTM_OK;
}

}  // extern "C"
