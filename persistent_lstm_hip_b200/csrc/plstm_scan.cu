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

// One special-function instruction each; results below 2^-126 come out as 0, 1 / inf as 0.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// max and min that keep a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- gate functions ----------------------------------------------------------------------------
// exp(s x) for s = -1 or -2.  exp = 2^(s log2(e) x) by the special-function unit is good to two
// units in 2^-23 plus the rounding of the product, |x| units in 2^-24: far below 16-bit inputs' own
// rounding.  For f32 (PRECISE) the product's rounding error is carried along: with t = fl(a x),
// a = hi + lo, the error r = a x - t enters as 2^(t + r) = 2^t (1 + r ln 2).
template <bool PRECISE, int V>
__device__ __forceinline__ F<V> exp_of(F<V> x, float s) {
  constexpr float kHi = 1.44269502162933349609375f;      // log2(e) to 24 bits
  constexpr float kLo = 1.925963033500011079e-8f;        // log2(e) - kHi
  constexpr float kLn2 = 0.693147180559945309f;
  if constexpr (PRECISE) {
    // Neither 2^t nor r overflows in here, and sigmoid(-87.6) is already below 2^-126.
    x = each(x, [](float v) { return min_nan(max_nan(v, -87.6f), 87.6f); });
    const F<V> t = x * F<V>::of(s * kHi);
    const F<V> r = fma(x, F<V>::of(s * kLo), fma(x, F<V>::of(s * kHi), t * F<V>::of(-1.0f)));
    const F<V> e = each(t, ex2);
    return fma(e, r * F<V>::of(kLn2), e);
  } else {
    return each(x * F<V>::of(s * kHi), ex2);
  }
}
template <bool PRECISE, int V>
__device__ __forceinline__ F<V> sigmoid_f(F<V> x) {
  return each(one_plus(exp_of<PRECISE>(x, -1.0f)), rcp);
}
// tanh(x) = num / den.  From 0.3 on (1 - e^-2x) / (1 + e^-2x), of x >= -9.1, where tanh rounds to
// -1 and the exponential is still small enough to be multiplied with another; below 0.3, where
// the difference would cancel, the odd series to x^9 (the next term is 4e-8 of the value).
template <bool PRECISE, int V>
__device__ __forceinline__ void tanh_parts(F<V> x, F<V>& num, F<V>& den) {
  const F<V> e = exp_of<PRECISE>(each(x, [](float v) { return max_nan(v, -9.1f); }), -2.0f);
  const F<V> s = x * x;
  F<V> p = fma(s, F<V>::of(62.0f / 2835), -17.0f / 315);
  p = fma(s, p, 2.0f / 15);
  p = fma(s, p, -1.0f / 3);
  p = fma(x * s, p, x);
  const F<V> n = one_minus(e), d = one_plus(e);
  float rn[V], rd[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const bool small = fabsf(x.get(k)) < 0.3f;
    rn[k] = small ? p.get(k) : n.get(k);
    rd[k] = small ? 1.0f : d.get(k);
  }
  num = F<V>::of(rn);
  den = F<V>::of(rd);
}
template <bool PRECISE, int V>
__device__ __forceinline__ F<V> tanh_f(F<V> x) {
  F<V> num, den;
  tanh_parts<PRECISE>(x, num, den);
  return num * each(den, rcp);
}
// sigmoid(a) tanh(x) with one reciprocal.
template <bool PRECISE, int V>
__device__ __forceinline__ F<V> sigmoid_tanh(F<V> a, F<V> x) {
  F<V> num, den;
  tanh_parts<PRECISE>(x, num, den);
  return num * each(one_plus(exp_of<PRECISE>(a, -1.0f)) * den, rcp);
}

template <int V>
struct alignas(8 * V) Run {  // the action c -> a c + b of a run of steps
  F<V> a, b;
};

// Reads V elements; those past the length are given as the step that changes nothing.
template <typename T>
__device__ __forceinline__ uint32_t infinity_bits() {
  return sizeof(T) == 4 ? 0x7f800000u : std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> constant_vec(uint32_t bits) {
  Vec<T, V> v;
  if constexpr (V * sizeof(T) == 2) {
    v.word = (unsigned short)bits;
  } else {
#pragma unroll
    for (int k = 0; k < (int)(V * sizeof(T) / 4); ++k) v.w[k] = bits;
  }
  return v;
}
template <typename T, int V>
__device__ __forceinline__ F<V> widen(const Vec<T, V>& v) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = v.get(k);
  return F<V>::of(r);
}
// Rounds to T; zero where the step is past the length.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(F<V> f, bool in) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = f.get(k);
  Vec<T, V> v;
  v.set(r);
  if constexpr (V * sizeof(T) == 2) {
    if (!in) v.word = 0;
  } else {
#pragma unroll
    for (int k = 0; k < (int)(V * sizeof(T) / 4); ++k) v.w[k] = in ? v.w[k] : 0u;
  }
  return v;
}
template <int V>
__device__ __forceinline__ F<V> load_state(const float* p, int64_t at, bool live) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = live && p != nullptr ? p[at + k] : 0.0f;
  return F<V>::of(r);
}
template <int V>
__device__ __forceinline__ void store_state(float* p, int64_t at, F<V> f) {
#pragma unroll
  for (int k = 0; k < V; ++k) p[at + k] = f.get(k);
}

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

// The exchange between the threads that share a channel.  `own` is this thread's run; `carry`, the
// state entering the tile, becomes the one leaving it.  Returns the state entering this thread's
// run.  Runs are folded in running order (backward: from the last segment and rank to the first).
template <int V, bool REVERSE>
struct Exchange {
  Run<V>* segs;   // [2][seg][cl]
  Run<V>* ranks;  // [2][kMaxCluster][cl]

  __device__ __forceinline__ F<V> operator()(const ScanArgs& p, const Place<V>& at, int turn, const Run<V>& own,
                                             F<V>& carry) const {
    const int parity = turn & 1;
    Run<V>* mine = segs + parity * p.seg * p.cl;
    const int order = REVERSE ? p.seg - 1 - at.seg : at.seg;
    F<V> state = carry;
    if (at.ranks == 1) {
      if (p.seg == 1) {
        carry = fma(own.a, carry, own.b);
        return state;
      }
      mine[order * p.cl + at.cl] = own;
      __syncthreads();
      for (int s = 0; s < p.seg; ++s) {
        if (s == order) state = carry;
        const Run<V> r = mine[s * p.cl + at.cl];
        carry = fma(r.a, carry, r.b);
      }
      return state;
    }
    mine[order * p.cl + at.cl] = own;
    __syncthreads();
    // The run of the CTA's segments before this thread's, and of all of them.
    Run<V> all{F<V>::of(1.0f), F<V>::of(0.0f)}, pre = all;
    for (int s = 0; s < p.seg; ++s) {
      if (s == order) pre = all;
      const Run<V> r = mine[s * p.cl + at.cl];
      all.b = fma(r.a, all.b, r.b);
      all.a = r.a * all.a;
    }
    cg::cluster_group cluster = cg::this_cluster();
    Run<V>* slots = ranks + parity * kMaxCluster * p.cl;
    const int rank_order = REVERSE ? at.ranks - 1 - at.rank : at.rank;
    for (int r = at.seg; r < at.ranks; r += p.seg)  // the segments share the remote stores
      cluster.map_shared_rank(slots, r)[rank_order * p.cl + at.cl] = all;
    cluster.sync();
    for (int r = 0; r < at.ranks; ++r) {
      if (r == rank_order) state = carry;
      const Run<V> q = slots[r * p.cl + at.cl];
      carry = fma(q.a, carry, q.b);
    }
    return fma(pre.a, state, pre.b);
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads, 3) scan_forward_kernel(const __grid_constant__ ScanArgs p, int cluster) {
  constexpr bool PRECISE = sizeof(T) == 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const Place<V> at(p, cluster);
  const Exchange<V, false> exchange{reinterpret_cast<Run<V>*>(smem),
                                    reinterpret_cast<Run<V>*>(smem) + 2 * p.seg * p.cl};
  // Distributed shared memory may be written once every CTA of the cluster has started.
  if (cluster > 1) cg::this_cluster().sync();
  const int tile = kSeg * p.seg * cluster;
  const int turns = (at.len + tile - 1) / tile;
  const int segments = (p.T + kSeg - 1) / kSeg;
  const T* gates = static_cast<const T*>(p.gates) + at.b * p.g_sb + at.ch;
  T* h = static_cast<T*>(p.h) + at.b * p.h_sb + at.ch;
  const int64_t state_at = (int64_t)at.b * p.H + at.ch;
  F<V> carry = load_state<V>(p.c0, state_at, at.live);
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = turn * tile + (at.rank * p.seg + at.seg) * kSeg;
    Vec<T, V> raw[4][kSeg];
    const T* from = gates + t0 * p.g_st;
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      const bool in = at.live && t0 + j < at.len;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // f = 1, u = 0: an infinite forget gate over a zero candidate.
        raw[q][j] = in ? load_vec<T, V>(from + (int64_t)q * p.H) : constant_vec<T, V>(q == 1 ? infinity_bits<T>() : 0);
      }
      from += p.g_st;
    }
    F<V> f[kSeg], u[kSeg];
    Run<V> own{F<V>::of(1.0f), F<V>::of(0.0f)};
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      f[j] = sigmoid_f<PRECISE>(widen(raw[1][j]));
      u[j] = sigmoid_tanh<PRECISE>(widen(raw[0][j]), widen(raw[2][j]));
      own.b = fma(f[j], own.b, u[j]);
      own.a = own.a * f[j];
    }
    F<V> c = exchange(p, at, turn, own, carry);
    if (at.live && p.ckpt != nullptr && t0 < at.len)
      store_state<V>(p.ckpt, ((int64_t)at.b * segments + t0 / kSeg) * p.H + at.ch, c);
    T* to = h + t0 * p.h_st;
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      c = fma(f[j], c, u[j]);
      const Vec<T, V> out = narrow<T, V>(sigmoid_tanh<PRECISE>(widen(raw[3][j]), c), t0 + j < at.len);
      if (at.live && t0 + j < p.T) store_vec<T, V>(to, out);
      to += p.h_st;
    }
  }
  if (!at.live) return;
  for (int64_t t = (int64_t)turns * tile + at.rank * p.seg + at.seg; t < p.T; t += p.seg * cluster)
    store_vec<T, V>(h + t * p.h_st, constant_vec<T, V>(0));
  if (at.rank == 0 && at.seg == 0) store_state<V>(p.c_n, state_at, carry);
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads, 2) scan_backward_kernel(const __grid_constant__ ScanArgs p, int cluster) {
  constexpr bool PRECISE = sizeof(T) == 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const Place<V> at(p, cluster);
  const Exchange<V, true> exchange{reinterpret_cast<Run<V>*>(smem),
                                   reinterpret_cast<Run<V>*>(smem) + 2 * p.seg * p.cl};
  if (cluster > 1) cg::this_cluster().sync();
  const int tile = kSeg * p.seg * cluster;
  const int turns = (at.len + tile - 1) / tile;
  const int segments = (p.T + kSeg - 1) / kSeg;
  const T* gates = static_cast<const T*>(p.gates) + at.b * p.g_sb + at.ch;
  const T* dh = p.dh != nullptr ? static_cast<const T*>(p.dh) + at.b * p.h_sb + at.ch : nullptr;
  T* dg = static_cast<T*>(p.dgates) + at.b * p.d_sb + at.ch;
  const int64_t state_at = (int64_t)at.b * p.H + at.ch;
  F<V> carry = load_state<V>(p.dc_n, state_at, at.live);
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = (turns - 1 - turn) * tile + (at.rank * p.seg + at.seg) * kSeg;
    Vec<T, V> raw[4][kSeg], rdh[kSeg];
    const T* from = gates + t0 * p.g_st;
    const T* dfrom = dh + t0 * p.h_st;
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      const bool in = at.live && t0 + j < at.len;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        raw[q][j] = in ? load_vec<T, V>(from + (int64_t)q * p.H) : constant_vec<T, V>(q == 1 ? infinity_bits<T>() : 0);
      }
      rdh[j] = in && dh != nullptr ? load_vec<T, V>(dfrom) : constant_vec<T, V>(0);
      from += p.g_st;
      dfrom += p.h_st;
    }
    F<V> c = load_state<V>(p.ckpt, ((int64_t)at.b * segments + t0 / kSeg) * p.H + at.ch, at.live && t0 < at.len);
    // Per step: f, e and what dc is multiplied with in the gradients of i, f and g.
    F<V> f[kSeg], e[kSeg], wi[kSeg], wf[kSeg], wg[kSeg];
    T* to = dg + t0 * p.d_st;
#pragma unroll
    for (int j = 0; j < kSeg; ++j) {
      const F<V> si = sigmoid_f<PRECISE>(widen(raw[0][j])), sf = sigmoid_f<PRECISE>(widen(raw[1][j]));
      const F<V> g = tanh_f<PRECISE>(widen(raw[2][j])), so = sigmoid_f<PRECISE>(widen(raw[3][j]));
      const F<V> d = widen(rdh[j]);
      f[j] = sf;
      wf[j] = c * (sf * one_minus(sf));
      wi[j] = g * (si * one_minus(si));
      wg[j] = si * one_minus(g * g);
      c = fma(sf, c, si * g);
      const F<V> tc = tanh_f<PRECISE>(c), dso = d * so;
      e[j] = t0 + j < at.len ? dso * one_minus(tc * tc) : F<V>::of(0.0f);
      const Vec<T, V> d_o = narrow<T, V>(dso * tc * one_minus(so), t0 + j < at.len);
      if (at.live && t0 + j < p.T) store_vec<T, V>(to + 3 * (int64_t)p.H, d_o);
      to += p.d_st;
    }
    Run<V> own{F<V>::of(1.0f), F<V>::of(0.0f)};
#pragma unroll
    for (int j = kSeg - 1; j >= 0; --j) {
      own.b = f[j] * (e[j] + own.b);
      own.a = own.a * f[j];
    }
    F<V> G = exchange(p, at, turn, own, carry);
#pragma unroll
    for (int j = kSeg - 1; j >= 0; --j) {
      to -= p.d_st;
      const bool in = t0 + j < at.len;
      const F<V> dc = e[j] + G;
      G = f[j] * dc;
      const Vec<T, V> di = narrow<T, V>(dc * wi[j], in), df = narrow<T, V>(dc * wf[j], in),
                      dgg = narrow<T, V>(dc * wg[j], in);
      if (at.live && t0 + j < p.T) {
        store_vec<T, V>(to, di);
        store_vec<T, V>(to + p.H, df);
        store_vec<T, V>(to + 2 * (int64_t)p.H, dgg);
      }
    }
  }
  if (!at.live) return;
  for (int64_t t = (int64_t)turns * tile + at.rank * p.seg + at.seg; t < p.T; t += p.seg * cluster) {
#pragma unroll
    for (int q = 0; q < 4; ++q) store_vec<T, V>(dg + t * p.d_st + (int64_t)q * p.H, constant_vec<T, V>(0));
  }
  if (p.dc0 != nullptr && at.rank == 0 && at.seg == 0) store_state<V>(p.dc0, state_at, carry);
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
