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
// Measured (GPU time, of the measured 6.54 TB/s): forward 168 us for B = 512, T = 1000, H = 128, f16, 60 % (the
// special-function unit is 69 % busy with its eight instructions an element, the issue slots 59 %; 1024 CTAs are 1.73
// waves of the 592 that fit), in f32 250 us, 80 %; 183 us for one row of 65,536 steps of H = 512, bf16, 28 % (32 turns,
// each with a cluster barrier under which only the next turn's copies run); 231 us for 1024 rows of 200 to 1000 steps,
// 60 %; 31 us for 4096 rows of three steps of H = 512, bf16, 31 %.
//
// Backward, with e_t = dh_t o_t (1 - tanh(c_t)^2): dc_t = e_t + G_t, G_{t-1} = f_t dc_t, where
// G enters the last step as dc_n and leaves the first as dc0: the same composition in reversed
// time.  c is rebuilt from the state that the forward kept for every segment.  294 us for the first shape
// above, 61 %: ten special-function instructions an element and 16 warps on an SM, since a step leaves
// five values for the second pass; in f32 481 us, 75 %.  The long row takes 290 us, 32 %, the short ones 47 us, 37 %
// (64 registers, of which up to 132 bytes spill).
#include <algorithm>
#include <cooperative_groups.h>
#include <initializer_list>

#include "plstm_ops.cuh"

namespace cg = cooperative_groups;

namespace plstm {
namespace ops {
namespace {

constexpr int kSeg = PLSTM_SCAN_SEGMENT;
constexpr int kMaxThreads = 128;
constexpr int kMaxCluster = 16;
constexpr int kWanted = 384;       // CTAs that keep the GPU busy (make_plan)
constexpr int kAlone = 16 * kSMs;  // warps that do without splitting time

struct ScanArgs {
  int B, T, H;
  int cl, seg, groups;  // channel lanes, time segments and channel groups of a CTA (their product: threads)
  int ch_blocks;        // groups along the channels of a row
  int stage_at;         // where shared memory past the exchange begins
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
// tanh(x) = num / den with den = 1 + e^-2x, of x >= -9.1, where tanh rounds to -1 and the exponential
// is still small enough to be multiplied with another.  num is 1 - e^-2x from 0.3 on; below, where
// that difference would cancel, den times the odd series to x^9 (the next term is 4e-8 of the value).
template <bool PRECISE, int V>
__device__ __forceinline__ void tanh_parts(F<V> x, F<V>& num, F<V>& den) {
  const F<V> e = exp_of<PRECISE>(each(x, [](float v) { return max_nan(v, -9.1f); }), -2.0f);
  const F<V> s = x * x;
  F<V> p = fma(s, F<V>::of(62.0f / 2835), -17.0f / 315);
  p = fma(s, p, 2.0f / 15);
  p = fma(s, p, -1.0f / 3);
  p = fma(x * s, p, x);
  den = one_plus(e);
  const F<V> n = one_minus(e), q = p * den;
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = fabsf(x.get(k)) < 0.3f ? q.get(k) : n.get(k);
  num = F<V>::of(r);
}
template <bool PRECISE, int V>
__device__ __forceinline__ F<V> tanh_f(F<V> x) {
  F<V> num, den;
  tanh_parts<PRECISE>(x, num, den);
  return num * each(den, rcp);
}
// sigmoid(a) tanh(x) with one reciprocal.  The product of the two denominators, up to 2^128 and 2^26.3, is taken
// 2^-27 times, so that it passes f32's range only where the result is below 2^-126; undoing that afterwards is
// exact (and after the product with num, which may be as small as x).
template <bool PRECISE, int V>
__device__ __forceinline__ F<V> sigmoid_tanh(F<V> a, F<V> x) {
  F<V> num, den;
  tanh_parts<PRECISE>(x, num, den);
  constexpr float kDown = 1.0f / (1 << 27);
  return num * each(fma(exp_of<PRECISE>(a, -1.0f), F<V>::of(kDown), kDown) * den, rcp) * F<V>::of(kDown);
}

template <int V>
struct alignas(8 * V) Run {  // the action c -> a c + b of a run of steps
  F<V> a, b;
};

// The type's infinity, for 16 bits twice: with the other gates zero it is the forget gate of a step that changes nothing.
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
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(F<V> f) {
  float r[V];
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = f.get(k);
  Vec<T, V> v;
  v.set(r);
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

// Where a thread stands.  The groups of channels that share a CTA with an exchange (and so its barriers)
// walk the whole sequence together; a group on its own stops at its length.
template <int V>
struct Place {
  int b, ch, cl, seg, rank, ranks, len;
  int warp_seg, warp_ch;  // the warp's first segment and channel
  int local, span;        // the group's place in the CTA, the steps it walks
  bool live;              // its channels exist
  __device__ __forceinline__ Place(const ScanArgs& p, int cluster) {
    ranks = cluster;
    rank = blockIdx.x % cluster;
    cl = threadIdx.x % p.cl;
    const int part = threadIdx.x / p.cl;
    seg = part % p.seg;
    local = part / p.seg;
    const int group = blockIdx.x / cluster * p.groups + local;
    b = group / p.ch_blocks;
    ch = ((group - b * p.ch_blocks) * p.cl + cl) * V;
    warp_seg = seg - (int)(threadIdx.x & 31) / p.cl;
    warp_ch = ch - cl * V;
    live = b < p.B && ch < p.H;
    len = p.T;
    if (b >= p.B)
      len = 0;
    else if (p.lengths != nullptr)
      len = min(max(p.lengths[b], 0), p.T);
    span = p.groups > 1 && p.seg > 1 ? p.T : len;
  }
};

// The exchange between the threads that share a channel, one barrier a turn (two in a cluster).  `own`
// is this thread's run; `carry`, the state entering the tile, becomes the one leaving it.  Returns the
// state entering this thread's run.  Runs are folded in running order (backward: from the last segment
// and rank to the first).  The buffers alternate from turn to turn, so a turn's barrier also frees the
// turn before's.
template <int V, bool REVERSE>
struct Exchange {
  Run<V>* segs;   // [2][seg][cl] of the group
  Run<V>* ranks;  // [2][kMaxCluster][cl]

  __device__ __forceinline__ F<V> operator()(const ScanArgs& p, const Place<V>& at, int turn, const Run<V>& own,
                                             F<V>& carry) const {
    const int parity = turn & 1;
    Run<V>* const mine = segs + parity * p.seg * p.cl + at.cl;
    const int order = REVERSE ? p.seg - 1 - at.seg : at.seg;
    F<V> state = carry;
    if (at.ranks == 1) {
      if (p.seg == 1) {
        carry = fma(own.a, carry, own.b);
        return state;
      }
      mine[order * p.cl] = own;
      __syncthreads();
      int s = 0;
#pragma unroll 4
      for (; s < order; ++s) carry = fma(mine[s * p.cl].a, carry, mine[s * p.cl].b);
      state = carry;
#pragma unroll 4
      for (; s < p.seg; ++s) carry = fma(mine[s * p.cl].a, carry, mine[s * p.cl].b);
      return state;
    }
    mine[order * p.cl] = own;
    __syncthreads();
    // The run of the CTA's segments before this thread's, and of all of them.
    Run<V> all{F<V>::of(1.0f), F<V>::of(0.0f)};
    const auto fold = [&](const Run<V>& r) {
      all.b = fma(r.a, all.b, r.b);
      all.a = r.a * all.a;
    };
    int s = 0;
#pragma unroll 4
    for (; s < order; ++s) fold(mine[s * p.cl]);
    const Run<V> pre = all;
#pragma unroll 4
    for (; s < p.seg; ++s) fold(mine[s * p.cl]);
    cg::cluster_group cluster = cg::this_cluster();
    Run<V>* const slots = ranks + parity * kMaxCluster * p.cl + at.cl;
    const int rank_order = REVERSE ? at.ranks - 1 - at.rank : at.rank;
    for (int r = at.seg; r < at.ranks; r += p.seg)  // the segments share the remote stores
      cluster.map_shared_rank(slots, r)[rank_order * p.cl] = all;
    cluster.sync();
    int r = 0;
    for (; r < rank_order; ++r) carry = fma(slots[r * p.cl].a, carry, slots[r * p.cl].b);
    state = carry;
    for (; r < at.ranks; ++r) carry = fma(slots[r * p.cl].a, carry, slots[r * p.cl].b);
    return fma(pre.a, state, pre.b);
  }
};

// K consecutive steps of the four gates of V channels, `left` of them within the length.  Those past it
// are given as the step that changes nothing: an infinite forget gate over zeros.
template <typename T, int V, int K>
__device__ __forceinline__ void load_steps(const T* from, int64_t stride, int H, bool live, int left,
                                           Vec<T, V> (&raw)[4][K]) {
  if (live && left >= K) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q) raw[q][j] = load_vec<T, V>(from + j * stride + (int64_t)q * H);
    }
  } else {
#pragma unroll
    for (int j = 0; j < K; ++j) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        raw[q][j] = live && j < left ? load_vec<T, V>(from + j * stride + (int64_t)q * H)
                                     : constant_vec<T, V>(q == 1 ? infinity_bits<T>() : 0);
    }
  }
}

// The gates of a warp's segments on their way into shared memory, 16 bytes a lane and copy (cp.async):
// word [step][gate][lane] is what `lane` will read.  A warp reads only what it copied, so no barrier is
// needed, and the copies for a turn fly while the turn before is worked on without holding registers.
// Steps past the length and channels past H arrive as zeros.  The forward stages in clusters, where a turn
// is long and the warps are few (one row of 65,536 steps, H = 512, bf16: a fifth less time than with the next
// turn in registers); elsewhere the detour costs more than it hides (B = 512, T = 1000, H = 128, f16: 185 us
// against 168 us), and so it does in the backward.
template <typename T, int V, int K>
struct Staged {
  enum : int {
    kWord = V * (int)sizeof(T),
    kPieces = 32 * kWord / 16,  // 16-byte pieces of one [lane] row
    kCopies = K * 4 * kPieces / 32,
    kBytes = K * 4 * 32 * kWord,
  };
  unsigned char* smem;  // this warp's
  // `t`: first step of the warp's first segment; `from`: its row's first channel at step 0.
  __device__ __forceinline__ void issue(const T* from, int64_t stride, int H, int cl, int ch0, int t, int len) const {
    const int lane = threadIdx.x & 31, r = lane % kPieces, per_seg = cl * kWord / 16;
    const int segment = r / per_seg, ch = (r - segment * per_seg) * (16 / (int)sizeof(T));
    const bool live = ch0 + ch < H;
    t += segment * K;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(smem) + lane * 16;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const int row = c * (32 / kPieces) + lane / kPieces, j = row / 4, q = row % 4;
      const bool in = live && t + j < len;
      const T* src = in ? from + (t + j) * stride + (int64_t)q * H + ch : from;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + c * 512), "l"(src), "r"(in ? 16 : 0)
                   : "memory");
    }
  }
  __device__ __forceinline__ Vec<T, V> get(int j, int q) const {
    return load_vec<T, V>(reinterpret_cast<const T*>(smem + ((j * 4 + q) * 32 + (threadIdx.x & 31)) * kWord));
  }
};
__device__ __forceinline__ void staged_wait() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
}

// K: steps of a segment, kSeg, or fewer where the whole sequence is no longer.  The state entering
// every segment is kept for the backward.
template <typename T, int V, int K, bool STAGED>
__global__ void __launch_bounds__(kMaxThreads, K < kSeg ? 8 : STAGED ? 5 : 4) scan_forward_kernel(const __grid_constant__ ScanArgs p, int cluster) {
  constexpr bool PRECISE = sizeof(T) == 4, ONE = K < kSeg;  // ONE: one segment is the whole sequence
  extern __shared__ __align__(16) unsigned char smem[];
  const Place<V> at(p, cluster);
  const Exchange<V, false> exchange{reinterpret_cast<Run<V>*>(smem) + at.local * 2 * p.seg * p.cl,
                                    reinterpret_cast<Run<V>*>(smem) + 2 * p.groups * p.seg * p.cl};
  // Distributed shared memory may be written once every CTA of the cluster has started.
  if (!ONE && cluster > 1) cg::this_cluster().sync();
  const int tile = K * p.seg * cluster;
  const int turns = (at.span + tile - 1) / tile;
  const int kept = (p.T + kSeg - 1) / kSeg;
  const T* gates = static_cast<const T*>(p.gates) + at.b * p.g_sb + at.ch;
  T* h = static_cast<T*>(p.h) + at.b * p.h_sb + at.ch;
  const int64_t state_at = (int64_t)at.b * p.H + at.ch;
  F<V> carry = load_state<V>(p.c0, state_at, at.live);
  const int mine = (at.rank * p.seg + at.seg) * K;
  // The next turn's gates are on their way during the exchange and the second pass: into shared
  // memory, or into registers where those hold them.
  constexpr bool AHEAD = !STAGED && K == kSeg && V * sizeof(T) <= 4;
  const Staged<T, V, K> staged{smem + p.stage_at + threadIdx.x / 32 * Staged<T, V, K>::kBytes};
  const int warp_t = (at.rank * p.seg + at.warp_seg) * K;
  const T* const row = gates - at.ch + at.warp_ch;
  Vec<T, V> raw[4][K];
  if (STAGED && turns > 0) staged.issue(row, p.g_st, p.H, p.cl, at.warp_ch, warp_t, at.len);
  if (AHEAD) load_steps<T, V, K>(gates + mine * p.g_st, p.g_st, p.H, at.live, at.len - mine, raw);
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = turn * tile + mine;
    if (STAGED) {
      staged_wait();
#pragma unroll
      for (int j = 0; j < K; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[q][j] = staged.get(j, q);
        if (t0 + j >= at.len) {
          raw[1][j] = constant_vec<T, V>(infinity_bits<T>());
        }
      }
    } else if (!AHEAD) {
      load_steps<T, V, K>(gates + t0 * p.g_st, p.g_st, p.H, at.live, at.len - t0, raw);
    }
    F<V> f[K], u[K];
    Run<V> own{F<V>::of(1.0f), F<V>::of(0.0f)};
#pragma unroll
    for (int j = 0; j < K; ++j) {
      f[j] = sigmoid_f<PRECISE>(widen<T, V>(raw[1][j]));
      u[j] = sigmoid_tanh<PRECISE>(widen<T, V>(raw[0][j]), widen<T, V>(raw[2][j]));
      own.b = j == 0 ? u[0] : fma(f[j], own.b, u[j]);
      own.a = j == 0 ? f[0] : own.a * f[j];
    }
    Vec<T, V> out_gate[K];
#pragma unroll
    for (int j = 0; j < K; ++j) out_gate[j] = raw[3][j];
    if (STAGED && turn + 1 < turns) {
      __syncwarp();
      staged.issue(row, p.g_st, p.H, p.cl, at.warp_ch, warp_t + (turn + 1) * tile, at.len);
    }
    if (AHEAD && turn + 1 < turns)
      load_steps<T, V, K>(gates + (t0 + tile) * p.g_st, p.g_st, p.H, at.live, at.len - t0 - tile, raw);
    F<V> c = ONE ? carry : exchange(p, at, turn, own, carry);
    if (ONE) carry = fma(own.a, carry, own.b);
    if (!at.live) continue;
    if (p.ckpt != nullptr && t0 < at.len)
      store_state<V>(p.ckpt, ((int64_t)at.b * kept + t0 / kSeg) * p.H + at.ch, c);
    T* const to = h + t0 * p.h_st;
    if (t0 + K <= at.len) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        c = fma(f[j], c, u[j]);
        store_vec<T, V>(to + j * p.h_st, narrow<T, V>(sigmoid_tanh<PRECISE>(widen<T, V>(out_gate[j]), c)));
      }
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        c = fma(f[j], c, u[j]);
        const Vec<T, V> out = narrow<T, V>(sigmoid_tanh<PRECISE>(widen<T, V>(out_gate[j]), c));
        if (t0 + j < p.T) store_vec<T, V>(to + j * p.h_st, t0 + j < at.len ? out : constant_vec<T, V>(0));
      }
    }
  }
  if (!at.live) return;
  for (int64_t t = (int64_t)turns * tile + at.rank * p.seg + at.seg; t < p.T; t += p.seg * cluster)
    store_vec<T, V>(h + t * p.h_st, constant_vec<T, V>(0));
  if (at.rank == 0 && at.seg == 0) store_state<V>(p.c_n, state_at, carry);
}

// Two of the five values that a step keeps for the second pass wait in shared memory (not for pairs of f32
// channels: 64 x 2000 x 256 251 us without, 328 us with).  For pairs of 16-bit channels this frees the
// registers of four CTAs an SM from spills (512 x 1000 x 128 f16: 298 us, without 336 us), or makes room for a
// fifth, which only the long turns of a cluster repay (CTAS = 5: one row of 65,536 steps, H = 512, bf16, 287 us
// against 357 us with four; 512 x 1000 x 128 330 us).
template <typename T, int V>
constexpr bool kHeld = V * sizeof(T) <= 4;
template <typename T, int V, int K, int CTAS>
__global__ void __launch_bounds__(kMaxThreads, K < kSeg ? 8 : CTAS) scan_backward_kernel(const __grid_constant__ ScanArgs p, int cluster) {
  constexpr bool PRECISE = sizeof(T) == 4, ONE = K < kSeg, HELD = kHeld<T, V> && !ONE;  // ONE: one segment is the whole sequence
  extern __shared__ __align__(16) unsigned char smem[];
  const Place<V> at(p, cluster);
  const Exchange<V, true> exchange{reinterpret_cast<Run<V>*>(smem) + at.local * 2 * p.seg * p.cl,
                                   reinterpret_cast<Run<V>*>(smem) + 2 * p.groups * p.seg * p.cl};
  if (!ONE && cluster > 1) cg::this_cluster().sync();
  const int tile = K * p.seg * cluster;
  const int turns = (at.span + tile - 1) / tile;
  const int kept = (p.T + kSeg - 1) / kSeg;
  const T* gates = static_cast<const T*>(p.gates) + at.b * p.g_sb + at.ch;
  const T* dh = p.dh != nullptr ? static_cast<const T*>(p.dh) + at.b * p.h_sb + at.ch : nullptr;
  T* dg = static_cast<T*>(p.dgates) + at.b * p.d_sb + at.ch;
  const int64_t state_at = (int64_t)at.b * p.H + at.ch;
  F<V> carry = load_state<V>(p.dc_n, state_at, at.live);
  F<V>* const held = reinterpret_cast<F<V>*>(smem + p.stage_at) + threadIdx.x;  // [2 K][kMaxThreads]
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = (turns - 1 - turn) * tile + (at.rank * p.seg + at.seg) * K;
    const int left = at.len - t0;
    const bool whole = left >= K;
    Vec<T, V> raw[4][K], rdh[K];
    load_steps<T, V, K>(gates + t0 * p.g_st, p.g_st, p.H, at.live, left, raw);
#pragma unroll
    for (int j = 0; j < K; ++j)
      rdh[j] = at.live && j < left && dh != nullptr ? load_vec<T, V>(dh + (t0 + j) * p.h_st) : constant_vec<T, V>(0);
    F<V> c = load_state<V>(p.ckpt, ((int64_t)at.b * kept + t0 / kSeg) * p.H + at.ch, at.live && left > 0);
    // Per step: f, e and what dc is multiplied with in the gradients of i, f and g.
    F<V> f[K], e[K], wf[K], wi[HELD ? 1 : K], wg[HELD ? 1 : K];
    T* const to = dg + t0 * p.d_st;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const F<V> si = sigmoid_f<PRECISE>(widen<T, V>(raw[0][j])), sf = sigmoid_f<PRECISE>(widen<T, V>(raw[1][j]));
      const F<V> g = tanh_f<PRECISE>(widen<T, V>(raw[2][j])), so = sigmoid_f<PRECISE>(widen<T, V>(raw[3][j]));
      f[j] = sf;
      wf[j] = c * (sf * one_minus(sf));
      (HELD ? held[2 * j * kMaxThreads] : wi[HELD ? 0 : j]) = g * (si * one_minus(si));
      (HELD ? held[(2 * j + 1) * kMaxThreads] : wg[HELD ? 0 : j]) = si * one_minus(g * g);
      c = fma(sf, c, si * g);
      const F<V> tc = tanh_f<PRECISE>(c), dso = widen<T, V>(rdh[j]) * so;
      e[j] = dso * one_minus(tc * tc);
      const Vec<T, V> d_o = narrow<T, V>(dso * tc * one_minus(so));
      if (whole) {
        if (at.live) store_vec<T, V>(to + j * p.d_st + 3 * (int64_t)p.H, d_o);
      } else {
        if (j >= left) e[j] = F<V>::of(0.0f);
        if (at.live && t0 + j < p.T)
          store_vec<T, V>(to + j * p.d_st + 3 * (int64_t)p.H, j < left ? d_o : constant_vec<T, V>(0));
      }
    }
    Run<V> own{f[K - 1], f[K - 1] * e[K - 1]};
#pragma unroll
    for (int j = K - 2; j >= 0; --j) {
      own.b = f[j] * (e[j] + own.b);
      own.a = own.a * f[j];
    }
    F<V> G = ONE ? carry : exchange(p, at, turn, own, carry);
    if (ONE) carry = fma(own.a, carry, own.b);
    if (!at.live) continue;
    if (whole) {
#pragma unroll
      for (int j = K - 1; j >= 0; --j) {
        const F<V> dc = e[j] + G;
        G = f[j] * dc;
        T* const at_j = to + j * p.d_st;
        store_vec<T, V>(at_j, narrow<T, V>(dc * (HELD ? held[2 * j * kMaxThreads] : wi[HELD ? 0 : j])));
        store_vec<T, V>(at_j + p.H, narrow<T, V>(dc * wf[j]));
        store_vec<T, V>(at_j + 2 * (int64_t)p.H, narrow<T, V>(dc * (HELD ? held[(2 * j + 1) * kMaxThreads] : wg[HELD ? 0 : j])));
      }
    } else {
#pragma unroll
      for (int j = K - 1; j >= 0; --j) {
        const F<V> dc = e[j] + G;
        G = f[j] * dc;
        const Vec<T, V> none = constant_vec<T, V>(0);
        T* const at_j = to + j * p.d_st;
        if (t0 + j < p.T) {
          store_vec<T, V>(at_j, j < left ? narrow<T, V>(dc * (HELD ? held[2 * j * kMaxThreads] : wi[HELD ? 0 : j])) : none);
          store_vec<T, V>(at_j + p.H, j < left ? narrow<T, V>(dc * wf[j]) : none);
          store_vec<T, V>(at_j + 2 * (int64_t)p.H, j < left ? narrow<T, V>(dc * (HELD ? held[(2 * j + 1) * kMaxThreads] : wg[HELD ? 0 : j])) : none);
        }
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

// One step of a batch of streams: a thread takes V channels of one row, nothing is exchanged.  16 rows of
// H = 512 bf16 take 1.9 us, a launch; 4096 rows of H = 2048 24 us, 96 % of the measured bandwidth with the f32 state
// read and written (the general kernel took 53 us, most of it finding its place).
template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) scan_step_kernel(const __grid_constant__ ScanArgs p) {
  constexpr bool PRECISE = sizeof(T) == 4;
  constexpr int W = V == 1 ? 1 : 2;
  const int ch = (blockIdx.x * kMaxThreads + threadIdx.x) * V;
  if (ch >= p.H) return;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const bool in = p.lengths == nullptr || p.lengths[b] > 0;
    const T* const from = static_cast<const T*>(p.gates) + b * p.g_sb + ch;
    const int64_t at = (int64_t)b * p.H + ch;
    Vec<T, V> raw[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      raw[q] = in ? load_vec<T, V>(from + (int64_t)q * p.H) : constant_vec<T, V>(q == 1 ? infinity_bits<T>() : 0);
    float c[V], h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      c[k] = p.c0 != nullptr ? p.c0[at + k] : 0.0f;
      if (p.ckpt != nullptr) p.ckpt[at + k] = c[k];
    }
#pragma unroll
    for (int i = 0; i < V / W; ++i) {
      F<W> gate[4], state;
      if constexpr (V == 1) {
#pragma unroll
        for (int q = 0; q < 4; ++q) gate[q] = F<1>::of(raw[q].get(0));
        state = F<1>::of(c[0]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) gate[q] = F<2>::of(raw[q].get(2 * i), raw[q].get(2 * i + 1));
        state = F<2>::of(c[2 * i], c[2 * i + 1]);
      }
      const F<W> f = sigmoid_f<PRECISE>(gate[1]), u = sigmoid_tanh<PRECISE>(gate[0], gate[2]);
      state = fma(f, state, u);
      const F<W> o = sigmoid_tanh<PRECISE>(gate[3], state);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        c[W * i + k] = state.get(k);
        h[W * i + k] = o.get(k);
      }
    }
    Vec<T, V> out;
    out.set(h);
    store_vec<T, V>(static_cast<T*>(p.h) + b * p.h_sb + ch, in ? out : constant_vec<T, V>(0));
#pragma unroll
    for (int k = 0; k < V; ++k) p.c_n[at + k] = c[k];
  }
}

// How the work is split (B x T x H; GPU times).  A CTA has 128 threads of up to 128 registers, four or five
// on an SM: 32 channel lanes, 128 bytes of a 16-bit row, by four segments of time.
// - Fewer than kWanted CTAs: fewer channels and more segments each, down to rows of 32 bytes (8 x 4096 x 1024
//   bf16 forward: 111 us with rows of 32 bytes, 116 us with clusters of four), or of 64 where rows do not
//   start on sectors (16 x 2000 x 310: 50 us with 64, 63 us with 32); then the CTAs of a cluster share a
//   channel (1 x 65536 x 512: 178 us with 16, 234 us with 8), and with 16 of them still too few, rows of 16
//   bytes (1 x 40759 x 21 f16, forward and backward: 77 us, without 419 us).
// - kAlone warps or more without splitting time: every warp walks its rows alone (4096 x 64 x 128 bf16: forward
//   79 us against 93 us, backward 142 us against 156 us); with 1024 warps splitting wins (512 x 1000 x 128 f16
//   forward: 171 us with four segments, 193 us with two).
// There are never more segments than the sequence has, and a CTA that they do not fill takes several groups.
struct Plan {
  int cl, seg, groups, cluster, ch_blocks;
};

Plan make_plan(int B, int T, int H, int V, int K, int size) {
  Plan p;
  const int lanes = (H + V - 1) / V, segments = std::max(1, (T + K - 1) / K);
  p.cl = 1;
  const int narrowest = (int64_t)H * size % 32 == 0 ? 32 : 64;  // bytes of a row that cost whole sectors
  while (p.cl < 32 && p.cl < lanes) p.cl *= 2;
  const auto blocks = [&] { return (int64_t)B * ((lanes + p.cl - 1) / p.cl); };
  while (p.cl * V * size / 2 >= narrowest && blocks() < kWanted && kMaxThreads / p.cl < segments) p.cl /= 2;
  p.seg = 1;
  if (blocks() < kAlone || p.cl < 32)
    while (p.seg * p.cl < kMaxThreads && p.seg < segments) p.seg *= 2;
  p.cluster = 1;
  while (p.cluster < kMaxCluster && blocks() * p.cluster < kWanted && p.seg * p.cluster < segments) p.cluster *= 2;
  // A long sequence of few channels: sectors are wasted rather than SMs.
  while (p.cluster == kMaxCluster && p.cl > 4 && blocks() * p.cluster < kWanted && p.seg * p.cluster < segments) {
    p.cl /= 2;
    p.seg *= 2;
  }
  p.groups = p.cluster == 1 ? std::max(1, kMaxThreads / (p.cl * p.seg)) : 1;
  p.ch_blocks = (lanes + p.cl - 1) / p.cl;
  return p;
}

// STAGED: V channels of a lane that come through shared memory, 16 bytes a copy.
template <typename T, int V, int K, bool STAGED>
int32_t launch(bool backward, ScanArgs a, cudaStream_t s) {
  const Plan plan = make_plan(a.B, a.T, a.H, V, K, (int)sizeof(T));
  a.cl = plan.cl;
  a.seg = plan.seg;
  a.groups = plan.groups;
  a.ch_blocks = plan.ch_blocks;
  const int64_t ctas = ((int64_t)a.B * plan.ch_blocks + plan.groups - 1) / plan.groups * plan.cluster;
  if ((int64_t)a.B * plan.ch_blocks > 0x7fffffff - kMaxThreads || ctas > 0x7fffffff) {
    set_error("gated scan: batch * hidden is too large for one launch");
    return PLSTM_ENOTSUP;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(plan.cl * plan.seg * plan.groups);
  a.stage_at = plan.seg > 1 ? (int)((2 * plan.groups * plan.seg + 2 * kMaxCluster) * plan.cl * sizeof(Run<V>)) : 0;
  const bool staged = STAGED && !backward && plan.cluster > 1;
  cfg.dynamicSmemBytes = a.stage_at + (backward ? (kHeld<T, V> && K == kSeg ? 2 * K * kMaxThreads * sizeof(F<V>) : 0)
                                       : staged ? cfg.blockDim.x / 32 * Staged<T, V, K>::kBytes
                                                : 0);
  // 48 KB need no allowance: runs, ranks' slots (of up to 32 lanes), and what is held or staged.
  static_assert((2 * kMaxThreads + 2 * kMaxCluster * 32) * sizeof(Run<V>) +
                    std::max<size_t>(kHeld<T, V> && K == kSeg ? 2 * K * kMaxThreads * sizeof(F<V>) : 0,
                                     STAGED ? kMaxThreads / 32 * Staged<T, V, K>::kBytes : 0) <=
                48 * 1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = plan.cluster > 1 ? 1 : 0;
  const auto go = [&](auto kernel) -> int32_t {
    if (plan.cluster > 8)  // beyond the portable size: has to be allowed for the kernel
      PLSTM_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    PLSTM_TRY_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, plan.cluster));
    note_launches(1);
    return PLSTM_OK;
  };
  if (backward) {
    if constexpr (K == kSeg && V == 2 && sizeof(T) == 2) {
      if (plan.cluster > 1) return go(scan_backward_kernel<T, V, K, 5>);
    }
    return go(scan_backward_kernel<T, V, K, V == 1 ? 5 : 4>);
  }
  if constexpr (STAGED) {
    if (staged) return go(scan_forward_kernel<T, V, K, true>);
  }
  if constexpr (K > 1) return go(scan_forward_kernel<T, V, K, false>);
  return PLSTM_EINVAL;  // one step forward is launch_step's
}

// Every access of V channels is aligned to V elements.
bool aligned_lanes(int dtype, const ScanArgs& a, int V) {
  const size_t bytes = V * dtype_size(dtype);
  for (const int64_t s : {(int64_t)a.H, a.g_sb, a.g_st, a.h_sb, a.h_st, a.d_sb, a.d_st})
    if (s % V != 0) return false;
  return aligned_to(a.gates, bytes) && aligned_to(a.h, bytes) && aligned_to(a.dh, bytes) && aligned_to(a.dgates, bytes);
}

template <typename T, int V>
int32_t launch_step(const ScanArgs& a, cudaStream_t s) {
  const dim3 grid((a.H + V * kMaxThreads - 1) / (V * kMaxThreads), std::min(a.B, 65535));
  scan_step_kernel<T, V><<<grid, std::min(kMaxThreads, ((a.H + V - 1) / V + 31) / 32 * 32), 0, s>>>(a);
  PLSTM_TRY_CUDA(cudaGetLastError());
  note_launches(1);
  return PLSTM_OK;
}

// A single step, or up to four, would waste most of a segment of eight (forward and backward of
// 4096 x 3 x 512 bf16: 32 + 47 us against 51 + 75 us; backward of 4096 x 1 x 2048: 78 us against 276 us).
template <typename T, int V>
int32_t dispatch_steps(bool backward, int dtype, const ScanArgs& a, cudaStream_t s) {
  if (backward && a.T == 1) return launch<T, V, 1, false>(true, a, s);
  if (a.T <= 4) return launch<T, V, 4, false>(backward, a, s);
  if constexpr (V == 2 && sizeof(T) == 2) {
    if (aligned_lanes(dtype, a, 16 / sizeof(T)) && a.H >= 64) return launch<T, V, kSeg, true>(backward, a, s);
  }
  return launch<T, V, kSeg, false>(backward, a, s);
}

template <typename T>
int32_t dispatch_type(bool backward, int dtype, const ScanArgs& a, cudaStream_t s) {
  if (!backward && a.T == 1) return aligned_lanes(dtype, a, 4) ? launch_step<T, 4>(a, s) : launch_step<T, 1>(a, s);
  return aligned_lanes(dtype, a, 2) ? dispatch_steps<T, 2>(backward, dtype, a, s)
                                    : dispatch_steps<T, 1>(backward, dtype, a, s);
}

int32_t dispatch(bool backward, int dtype, const ScanArgs& a, cudaStream_t s) {
  if (dtype == PLSTM_F32) return dispatch_type<float>(backward, dtype, a, s);
  if (dtype == PLSTM_F16) return dispatch_type<__half>(backward, dtype, a, s);
  return dispatch_type<__nv_bfloat16>(backward, dtype, a, s);
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
