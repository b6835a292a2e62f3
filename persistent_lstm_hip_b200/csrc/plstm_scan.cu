// plstm_scan.cu — the gated scan: the recurrence of an LSTM layer whose gates do not look
// back, forward and backward.
//
//   c_t = f_t c_{t-1} + u_t,   f = sigmoid(f~), u = sigmoid(i~) tanh(g~)
//   h_t = sigmoid(o~_t) tanh(c_t)
//
// is linear in c, so a run of steps acts on the state entering it as c -> A c + b with
// A = prod f and b its end state from zero, and runs compose: (A2, b2) after (A1, b1) is
// (A1 A2, A2 b1 + b2).  Time is split three ways: a thread takes kSeg consecutive steps of V
// channels in registers, the `seg` threads of a CTA that share a channel take consecutive
// segments, and the CTAs of a cluster take consecutive CTA tiles.  Per turn a thread reads its
// segment once, reduces it to (A, b), learns the state entering it from the (A, b) of the
// segments before it (shared memory within the CTA, distributed shared memory across the
// cluster, always folded in time order, so results do not depend on timing), and runs its
// steps again out of registers to write h.  The input is read once and the waits are the
// hardware's barriers.
//
// Backward, with e_t = dh_t o_t (1 - tanh(c_t)^2): dc_t = e_t + G_t, G_{t-1} = f_t dc_t, where
// G enters the last step as dc_n and leaves the first as dc0: the same composition in reversed
// time.  c is rebuilt from the state that the forward kept for every segment.
#include <algorithm>
#include <cooperative_groups.h>

#include "plstm_ops.cuh"

namespace cg = cooperative_groups;

namespace plstm {
namespace ops {
namespace {

constexpr int kSeg = PLSTM_SCAN_SEGMENT;
constexpr int kMaxThreads = 256;
constexpr int kMaxCluster = 8;

struct ScanArgs {
  int B, T, H;
  int cl, seg;        // channel lanes and time segments of a CTA (cl * seg threads)
  int ch_blocks;      // CTAs (or clusters) along the channels of a row
  int64_t g_sb, g_st, h_sb, h_st, d_sb, d_st;
  const void* gates;
  const int32_t* lengths;
  const float* c0;
  void* h;
  float* c_n;
  float* ckpt;        // [B][ceil(T / kSeg)][H]
  const void* dh;
  const float* dc_n;
  void* dgates;
  float* dc0;
};

// f32 inputs use CUDA's accurate functions; for 16-bit inputs the exponential's and the
// division's fast forms (a few units in 2^-23 for the arguments gates take) are far below the
// inputs' own 2^-9 or 2^-12, and tanh takes its odd series below 0.3, where 1 - 2 / (1 + e^2x)
// would cancel.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float x) {
  if constexpr (sizeof(T) == 4) return sigmoid_acc(x);
  return __fdividef(1.0f, 1.0f + __expf(-x));
}
template <typename T>
__device__ __forceinline__ float tanh_of(float x) {
  if constexpr (sizeof(T) == 4) return tanh_acc(x);
  const float s = x * x;
  const float small = x * (1.0f + s * (-1.0f / 3 + s * (2.0f / 15 + s * (-17.0f / 315 + s * (62.0f / 2835)))));
  const float large = 1.0f - __fdividef(2.0f, 1.0f + __expf(2.0f * x));
  return fabsf(x) < 0.3f ? small : large;
}

template <int V>
struct alignas(8 * V) Run {  // the action (A, b) of a run of steps on V channels
  float a[V], b[V];
};

// Where a thread stands.
template <int V>
struct Place {
  int b, ch, cl, seg, rank, ranks, len;
  bool live;  // its channels exist
  __device__ __forceinline__ Place(const ScanArgs& p, int cluster) {
    ranks = cluster;
    rank = blockIdx.x % cluster;
    const int group = blockIdx.x / cluster;
    cl = threadIdx.x % p.cl;
    seg = threadIdx.x / p.cl;
    b = group / p.ch_blocks;
    ch = ((group % p.ch_blocks) * p.cl + cl) * V;
    live = ch < p.H;
    len = p.T;
    if (p.lengths != nullptr) len = min(max(p.lengths[b], 0), p.T);
  }
};

// The exchange between the threads that share a channel.  `own` is this thread's run; on return
// `state` (the value entering the tile) has become the value entering this thread's run and
// `carry` the value leaving the whole tile.  ORDER(s): the s-th segment or rank in running order.
template <int V, bool REVERSE>
struct Exchange {
  Run<V>* segs;   // [2][seg][cl]
  Run<V>* ranks;  // [2][kMaxCluster][cl]

  __device__ __forceinline__ void operator()(const ScanArgs& p, const Place<V>& at, int turn, const Run<V>& own,
                                             float (&state)[V], float (&carry)[V]) const {
    const int parity = turn & 1;
    Run<V>* mine = segs + parity * p.seg * p.cl;
    const int order = REVERSE ? p.seg - 1 - at.seg : at.seg;
    mine[order * p.cl + at.cl] = own;
    __syncthreads();
    // The run of the CTA's segments before this thread's.
    Run<V> pre;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      pre.a[k] = 1.0f;
      pre.b[k] = 0.0f;
    }
    Run<V> all = pre;
    for (int s = 0; s < p.seg; ++s) {
      if (s == order) pre = all;
      const Run<V> r = mine[s * p.cl + at.cl];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        all.b[k] = r.a[k] * all.b[k] + r.b[k];
        all.a[k] *= r.a[k];
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) carry[k] = state[k];
    if (at.ranks > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      Run<V>* slots = ranks + parity * kMaxCluster * p.cl;
      const int rank_order = REVERSE ? at.ranks - 1 - at.rank : at.rank;
      for (int r = at.seg; r < at.ranks; r += p.seg)  // the segments share the remote stores
        cluster.map_shared_rank(slots, r)[rank_order * p.cl + at.cl] = all;
      cluster.sync();
      for (int r = 0; r < at.ranks; ++r) {
        if (r == rank_order) {
#pragma unroll
          for (int k = 0; k < V; ++k) state[k] = carry[k];
        }
        const Run<V> q = slots[r * p.cl + at.cl];
#pragma unroll
        for (int k = 0; k < V; ++k) carry[k] = q.a[k] * carry[k] + q.b[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) carry[k] = all.a[k] * carry[k] + all.b[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) state[k] = pre.a[k] * state[k] + pre.b[k];
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) scan_forward_kernel(const __grid_constant__ ScanArgs p, int cluster) {
  extern __shared__ __align__(16) float smem[];
  const Place<V> at(p, cluster);
  Exchange<V, false> exchange{reinterpret_cast<Run<V>*>(smem),
                              reinterpret_cast<Run<V>*>(smem) + 2 * p.seg * p.cl};
  // Distributed shared memory may be written once every CTA of the cluster has started.
  if (cluster > 1) cg::this_cluster().sync();
  const int tile = kSeg * p.seg * cluster;
  const int turns = (at.len + tile - 1) / tile;
  const int segments = (p.T + kSeg - 1) / kSeg;
  const T* gates = static_cast<const T*>(p.gates) + at.b * p.g_sb + at.ch;
  T* h = static_cast<T*>(p.h) + at.b * p.h_sb + at.ch;
  float carry[V];
#pragma unroll
  for (int k = 0; k < V; ++k)
    carry[k] = at.live && p.c0 != nullptr ? p.c0[(int64_t)at.b * p.H + at.ch + k] : 0.0f;
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = turn * tile + (at.rank * p.seg + at.seg) * kSeg;
    Vec<T, V> raw[4][kSeg];
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      if (at.live && t0 + j < at.len) {
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[q][j] = load_vec<T, V>(gates + (t0 + j) * p.g_st + (int64_t)q * p.H);
      }
    }
    float f[kSeg][V], u[kSeg][V];
    Run<V> own;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      own.a[k] = 1.0f;
      own.b[k] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      const bool in = at.live && t0 + j < at.len;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        f[j][k] = in ? sigmoid_of<T>(to_f32(raw[1][j].v[k])) : 1.0f;
        u[j][k] = in ? sigmoid_of<T>(to_f32(raw[0][j].v[k])) * tanh_of<T>(to_f32(raw[2][j].v[k])) : 0.0f;
        own.b[k] = f[j][k] * own.b[k] + u[j][k];
        own.a[k] *= f[j][k];
      }
    }
    float c[V];
#pragma unroll
    for (int k = 0; k < V; ++k) c[k] = carry[k];
    exchange(p, at, turn, own, c, carry);
    if (at.live && p.ckpt != nullptr && t0 < at.len) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        p.ckpt[((int64_t)at.b * segments + t0 / kSeg) * p.H + at.ch + k] = c[k];
    }
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      if (at.live && t0 + j < p.T) {
        Vec<T, V> out;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          c[k] = f[j][k] * c[k] + u[j][k];
          const float o = t0 + j < at.len ? sigmoid_of<T>(to_f32(raw[3][j].v[k])) * tanh_of<T>(c[k]) : 0.0f;
          out.v[k] = from_f32<T>(o);
        }
        store_vec<T, V>(h + (t0 + j) * p.h_st, out);
      }
    }
  }
  if (!at.live) return;
  Vec<T, V> zero;
#pragma unroll
  for (int k = 0; k < V; ++k) zero.v[k] = from_f32<T>(0.0f);
  for (int64_t t = (int64_t)turns * tile + at.rank * p.seg + at.seg; t < p.T; t += p.seg * cluster)
    store_vec<T, V>(h + t * p.h_st, zero);
  if (at.rank == 0 && at.seg == 0) {
#pragma unroll
    for (int k = 0; k < V; ++k) p.c_n[(int64_t)at.b * p.H + at.ch + k] = carry[k];
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) scan_backward_kernel(const __grid_constant__ ScanArgs p, int cluster) {
  extern __shared__ __align__(16) float smem[];
  const Place<V> at(p, cluster);
  Exchange<V, true> exchange{reinterpret_cast<Run<V>*>(smem),
                             reinterpret_cast<Run<V>*>(smem) + 2 * p.seg * p.cl};
  // Distributed shared memory may be written once every CTA of the cluster has started.
  if (cluster > 1) cg::this_cluster().sync();
  const int tile = kSeg * p.seg * cluster;
  const int turns = (at.len + tile - 1) / tile;
  const int segments = (p.T + kSeg - 1) / kSeg;
  const T* gates = static_cast<const T*>(p.gates) + at.b * p.g_sb + at.ch;
  const T* dh = p.dh != nullptr ? static_cast<const T*>(p.dh) + at.b * p.h_sb + at.ch : nullptr;
  T* dg = static_cast<T*>(p.dgates) + at.b * p.d_sb + at.ch;
  Vec<T, V> zero;
#pragma unroll
  for (int k = 0; k < V; ++k) zero.v[k] = from_f32<T>(0.0f);
  float carry[V];
#pragma unroll
  for (int k = 0; k < V; ++k)
    carry[k] = at.live && p.dc_n != nullptr ? p.dc_n[(int64_t)at.b * p.H + at.ch + k] : 0.0f;
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = (turns - 1 - turn) * tile + (at.rank * p.seg + at.seg) * kSeg;
    Vec<T, V> raw[4][kSeg], rdh[kSeg];
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      if (at.live && t0 + j < at.len) {
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[q][j] = load_vec<T, V>(gates + (t0 + j) * p.g_st + (int64_t)q * p.H);
        rdh[j] = dh != nullptr ? load_vec<T, V>(dh + (t0 + j) * p.h_st) : zero;
      }
    }
    float c[V];
#pragma unroll
    for (int k = 0; k < V; ++k)
      c[k] = at.live && t0 < at.len ? p.ckpt[((int64_t)at.b * segments + t0 / kSeg) * p.H + at.ch + k] : 0.0f;
    // Per step: f, e and what dc is multiplied with in the gradients of i, f and g.
    float f[kSeg][V], e[kSeg][V], wi[kSeg][V], wf[kSeg][V], wg[kSeg][V];
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      const bool in = at.live && t0 + j < at.len;
      Vec<T, V> d_o = zero;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        f[j][k] = 1.0f;
        e[j][k] = 0.0f;
        if (in) {
          const float si = sigmoid_of<T>(to_f32(raw[0][j].v[k])), sf = sigmoid_of<T>(to_f32(raw[1][j].v[k]));
          const float g = tanh_of<T>(to_f32(raw[2][j].v[k])), so = sigmoid_of<T>(to_f32(raw[3][j].v[k]));
          const float d = to_f32(rdh[j].v[k]);
          f[j][k] = sf;
          wf[j][k] = c[k] * sf * (1.0f - sf);
          wi[j][k] = g * si * (1.0f - si);
          wg[j][k] = si * (1.0f - g * g);
          c[k] = sf * c[k] + si * g;
          const float tc = tanh_of<T>(c[k]);
          e[j][k] = d * so * (1.0f - tc * tc);
          d_o.v[k] = from_f32<T>(d * tc * so * (1.0f - so));
        }
      }
      if (at.live && t0 + j < p.T) store_vec<T, V>(dg + (t0 + j) * p.d_st + 3 * (int64_t)p.H, d_o);
    }
    Run<V> own;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      own.a[k] = 1.0f;
      own.b[k] = 0.0f;
    }
#pragma unroll
    for (int j = kSeg - 1; j >= 0; --j) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        own.b[k] = f[j][k] * (e[j][k] + own.b[k]);
        own.a[k] *= f[j][k];
      }
    }
    float G[V];
#pragma unroll
    for (int k = 0; k < V; ++k) G[k] = carry[k];
    exchange(p, at, turn, own, G, carry);
#pragma unroll
    for (int j = kSeg - 1; j >= 0; --j) {
      if (at.live && t0 + j < p.T) {
        const bool in = t0 + j < at.len;
        Vec<T, V> di = zero, df = zero, dgg = zero;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if (in) {
            const float dc = e[j][k] + G[k];
            G[k] = f[j][k] * dc;
            di.v[k] = from_f32<T>(dc * wi[j][k]);
            df.v[k] = from_f32<T>(dc * wf[j][k]);
            dgg.v[k] = from_f32<T>(dc * wg[j][k]);
          }
        }
        T* to = dg + (t0 + j) * p.d_st;
        store_vec<T, V>(to, di);
        store_vec<T, V>(to + p.H, df);
        store_vec<T, V>(to + 2 * (int64_t)p.H, dgg);
      }
    }
  }
  if (!at.live) return;
  for (int64_t t = (int64_t)turns * tile + at.rank * p.seg + at.seg; t < p.T; t += p.seg * cluster) {
#pragma unroll
    for (int q = 0; q < 4; ++q) store_vec<T, V>(dg + t * p.d_st + (int64_t)q * p.H, zero);
  }
  if (p.dc0 != nullptr && at.rank == 0 && at.seg == 0) {
#pragma unroll
    for (int k = 0; k < V; ++k) p.dc0[(int64_t)at.b * p.H + at.ch + k] = carry[k];
  }
}

// How the work is split: channel lanes to fill a warp where H allows, then time segments up to
// the CTA's threads, then a cluster where the CTAs would not fill the GPU; never more segments
// than the sequence has.
struct Plan {
  int cl, seg, cluster, ch_blocks;
};

Plan make_plan(int B, int T, int H, int V) {
  Plan p;
  const int lanes = (H + V - 1) / V;
  p.cl = 1;
  while (p.cl < 32 && p.cl < lanes) p.cl *= 2;
  p.ch_blocks = (lanes + p.cl - 1) / p.cl;
  const int segments = std::max(1, (T + kSeg - 1) / kSeg);
  p.seg = 1;
  while (p.seg * p.cl < kMaxThreads && p.seg < segments) p.seg *= 2;
  p.cluster = 1;
  const int64_t groups = (int64_t)B * p.ch_blocks;
  while (p.cluster < kMaxCluster && groups * p.cluster < 2 * kSMs && p.seg * p.cluster < segments) p.cluster *= 2;
  return p;
}

template <typename T, int V>
int32_t launch(bool backward, ScanArgs a, cudaStream_t s) {
  const Plan plan = make_plan(a.B, a.T, a.H, V);
  a.cl = plan.cl;
  a.seg = plan.seg;
  a.ch_blocks = plan.ch_blocks;
  const int64_t ctas = (int64_t)a.B * plan.ch_blocks * plan.cluster;
  if (ctas > 0x7fffffff) {
    set_error("gated scan: batch * hidden is too large for one launch");
    return PLSTM_ENOTSUP;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(plan.cl * plan.seg);
  cfg.dynamicSmemBytes = (size_t)2 * (plan.seg + kMaxCluster) * plan.cl * sizeof(Run<V>);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (backward)
    PLSTM_TRY_CUDA(cudaLaunchKernelEx(&cfg, scan_backward_kernel<T, V>, a, plan.cluster));
  else
    PLSTM_TRY_CUDA(cudaLaunchKernelEx(&cfg, scan_forward_kernel<T, V>, a, plan.cluster));
  note_launches(1);
  return PLSTM_OK;
}

// Two channels per thread where every access is aligned to the pair, else one.
int32_t dispatch(bool backward, int dtype, const ScanArgs& a, cudaStream_t s) {
  const size_t pair = 2 * dtype_size(dtype);
  const bool even = a.H % 2 == 0 && a.g_sb % 2 == 0 && a.g_st % 2 == 0 && a.h_sb % 2 == 0 && a.h_st % 2 == 0 &&
                    a.d_sb % 2 == 0 && a.d_st % 2 == 0 && aligned_to(a.gates, pair) && aligned_to(a.h, pair) &&
                    aligned_to(a.dh, pair) && aligned_to(a.dgates, pair);
  if (dtype == PLSTM_F32) return even ? launch<float, 2>(backward, a, s) : launch<float, 1>(backward, a, s);
  if (dtype == PLSTM_F16) return even ? launch<__half, 2>(backward, a, s) : launch<__half, 1>(backward, a, s);
  return even ? launch<__nv_bfloat16, 2>(backward, a, s) : launch<__nv_bfloat16, 1>(backward, a, s);
}

int32_t check_desc(const plstm_scan_desc* d) {
  PLSTM_CHECK_ARG(d != nullptr, "gated scan: the descriptor is NULL");
  PLSTM_CHECK_ARG(d->batch >= 0 && d->seq_len >= 0, "gated scan: batch and seq_len must be >= 0");
  PLSTM_CHECK_ARG(d->seq_len <= 0x7fffffff - 65536, "gated scan: seq_len is too large");
  PLSTM_CHECK_ARG(d->hidden >= 1 && d->hidden <= (1 << 28), "gated scan: hidden must be in [1, 2^28]");
  PLSTM_CHECK_ARG(dtype_ok(d->dtype), "gated scan: bad dtype");
  PLSTM_CHECK_ARG(d->reserved == 0, "gated scan: reserved must be 0");
  PLSTM_CHECK_ARG(d->gates_batch_stride >= 0 && d->gates_time_stride >= 0 && d->h_batch_stride >= 0 &&
                      d->h_time_stride >= 0 && d->dgates_batch_stride >= 0 && d->dgates_time_stride >= 0,
                  "gated scan: strides must be >= 0");
  return PLSTM_OK;
}

}  // namespace
}  // namespace ops
}  // namespace plstm

using namespace plstm;
using namespace plstm::ops;

extern "C" {

int32_t plstm_gated_scan_checkpoint_size(const plstm_scan_desc* d, size_t* bytes) {
  clear_error();
  PLSTM_CHECK_ARG(bytes != nullptr, "bytes is NULL");
  if (const int32_t rc = ops::check_desc(d)) return rc;
  *bytes = (size_t)d->batch * ((d->seq_len + kSeg - 1) / kSeg) * d->hidden * sizeof(float);
  return PLSTM_OK;
}

int32_t plstm_gated_scan_forward(const plstm_scan_desc* d, const void* gates, const int32_t* lengths, const float* c0,
                                 void* h, float* c_n, float* checkpoints, void* stream) {
  clear_error();
  if (const int32_t rc = ops::check_desc(d)) return rc;
  if (d->batch == 0) return PLSTM_OK;
  PLSTM_CHECK_ARG(c_n != nullptr, "gated scan: c_n must not be NULL");
  PLSTM_CHECK_ARG(d->seq_len == 0 || (gates != nullptr && h != nullptr), "gated scan: gates and h must not be NULL");
  const size_t e = dtype_size(d->dtype);
  PLSTM_CHECK_ARG(aligned_to(gates, e) && aligned_to(h, e) && aligned_to(c0, 4) && aligned_to(c_n, 4) &&
                      aligned_to(checkpoints, 4) && aligned_to(lengths, 4),
                  "gated scan: a pointer is not aligned to its element");
  DeviceGuard guard;
  if (const int32_t rc = guard.enter(d->device)) return rc;
  ScanArgs a{};
  a.B = d->batch;
  a.T = d->seq_len;
  a.H = d->hidden;
  a.g_sb = d->gates_batch_stride;
  a.g_st = d->gates_time_stride;
  a.h_sb = d->h_batch_stride;
  a.h_st = d->h_time_stride;
  a.gates = gates;
  a.lengths = lengths;
  a.c0 = c0;
  a.h = h;
  a.c_n = c_n;
  a.ckpt = checkpoints;
  return dispatch(false, d->dtype, a, static_cast<cudaStream_t>(stream));
}

int32_t plstm_gated_scan_backward(const plstm_scan_desc* d, const void* gates, const int32_t* lengths,
                                  const float* checkpoints, const void* dh, const float* dc_n, void* dgates,
                                  float* dc0, void* stream) {
  clear_error();
  if (const int32_t rc = ops::check_desc(d)) return rc;
  if (d->batch == 0) return PLSTM_OK;
  PLSTM_CHECK_ARG(d->seq_len == 0 || (gates != nullptr && checkpoints != nullptr && dgates != nullptr),
                  "gated scan backward: gates, checkpoints and dgates must not be NULL");
  const size_t e = dtype_size(d->dtype);
  PLSTM_CHECK_ARG(aligned_to(gates, e) && aligned_to(dh, e) && aligned_to(dgates, e) && aligned_to(dc_n, 4) &&
                      aligned_to(checkpoints, 4) && aligned_to(lengths, 4) && aligned_to(dc0, 4),
                  "gated scan backward: a pointer is not aligned to its element");
  DeviceGuard guard;
  if (const int32_t rc = guard.enter(d->device)) return rc;
  ScanArgs a{};
  a.B = d->batch;
  a.T = d->seq_len;
  a.H = d->hidden;
  a.g_sb = d->gates_batch_stride;
  a.g_st = d->gates_time_stride;
  a.h_sb = d->h_batch_stride;
  a.h_st = d->h_time_stride;
  a.d_sb = d->dgates_batch_stride;
  a.d_st = d->dgates_time_stride;
  a.gates = gates;
  a.lengths = lengths;
  a.ckpt = const_cast<float*>(checkpoints);
  a.dh = dh;
  a.dc_n = dc_n;
  a.dgates = dgates;
  a.dc0 = dc0;
  return dispatch(true, d->dtype, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
