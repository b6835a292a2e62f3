// plstm_norm.cu — layer norm over the last axis, forward and backward, plain or fused with
// the residual step z = residual + dropout(x) in front of it.
//
// Forward, per row: mean, then the centred sum of squares (two passes over registers, so no
// cancellation for rows far from zero), then y = (v - mean) rstd w + b.
// Backward, with xh = (v - mean) rstd and g = dy w:
//   dv = rstd (g - mean(g) - xh mean(g xh)) [+ dz],  dw = sum over rows of dy xh,  db = sum of dy.
// The weight gradients are summed per thread over the rows its CTA visits, then over the
// CTA's row groups, then over the CTAs by a second kernel: a fixed order, no atomics.
//
// Measured at 65536 x 1024 bf16 with f32 weights: forward 53 us, 78 % of the measured 6.54 TB/s (14 instructions an
// element, issue 54 %); backward with the weight gradients 86 us, 71 % (27 an element, issue 63 %, 23 % of the warps).
// With residual and dropout at 131072 x 512: 128 and 157 us, 64 % and 65 % (Philox adds 11.5 instructions an element);
// the same elements 1024 wide: 165 and 166 us, 50 % and 62 %, where the forward's four chunks a thread spill (make_split)
// and it waits for memory (issue 46 %); with f32 throughout at 65536 x 512: 88 and 114 us, 94 % and 90 %.
// Rows 1001 wide (33000 of them, bf16) take 57 and 91 us, rows 1024 wide 31 and 50 us: the masked ends, the columns'
// places and single reads of the weights cost instructions.  Rows of 16384 (8192 of them, bf16, f32 weights): 156 and
// 366 us, 53 % and 34 %.
#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "plstm_ops.cuh"

namespace plstm {
namespace ops {
namespace {

// How the work is spread.  Memory is walked in chunks of eight elements that are aligned in the
// flattened tensor, whatever the row length: a row then starts and ends inside a chunk (its phase
// is row * cols mod 8), whose foreign elements are masked, every other access is 16 bytes wide, and a
// chunk is two whole Philox blocks.  A team of `tpr` threads (a power of two up to a warp, or whole
// warps) takes a row: chunk c of lane t is the row's (c * tpr + t)-th.  A CTA holds `teams` teams.
// The forward issues the loads of a team's next row before the sums over the current one.
//
// WHOLE: cols is a multiple of 8 and every row is aligned, so there is no phase and no mask.
struct Split {
  int ch, tpr, teams;
  int block() const { return tpr * teams; }
};
// Widest team: four chunks a thread hold 16384 columns (2049 chunks), two a thread 4096 (513).  The CTA of 544 threads
// leaves 96 registers to every four-chunk kernel, of whatever width: the plain forwards spill up to 68 bytes, the fused
// ones 24 to 556, the backwards 48 to 864.
constexpr int max_block(int ch) { return ch == 4 ? 544 : 288; }
constexpr int kTeamBlock = 128;  // CTA size up to which teams share a CTA

// A tensor as the kernels address it: element (row, col) at row * stride + col.
struct Mat {
  const void* p;
  int64_t stride;
  int64_t extent;  // elements from the first to the last, so that no vector leaves the tensor
  int vec;         // chunks are 16-byte aligned
};

struct NormArgs {
  int64_t rows;
  int cols, tpr, teams;
  float eps;
  Mat x, residual, z, y;        // forward
  Mat dy, dz, v, dx, dres;      // backward
  const void *weight, *bias;
  float* mean;
  float* rstd;
  float* partial;
  int w_dtype;
  Drop drop;
};

// Teams of several warps share a CTA only as two of 64 threads.  The barriers' numbers are constants:
// a number in a register makes the compiler claim all 16, and then three CTAs fill an SM.
__device__ __forceinline__ void team_sync(int team, int threads) {
  if (threads > kTeamBlock / 2) {
    __syncthreads();
  } else if (team == 0) {
    asm volatile("bar.sync 1, 64;" ::: "memory");
  } else {
    asm volatile("bar.sync 2, 64;" ::: "memory");
  }
}

// Sums NV values over a team.  `scratch` [teams][2][NV][32]: two turns apart, so that one barrier a
// sum is enough (`turn` alternates from sum to sum).
template <int NV>
__device__ __forceinline__ void team_sum(float (&a)[NV], int team, int tpr, float* scratch, int turn) {
  for (int o = min(tpr, 32) >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k) a[k] += __shfl_xor_sync(0xffffffffu, a[k], o);
  }
  if (tpr <= 32) return;
  const int t = threadIdx.x - team * tpr, warps = tpr >> 5;
  float* mine = scratch + (team * 2 + (turn & 1)) * NV * 32;
  if ((t & 31) == 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) mine[(t >> 5) * NV + k] = a[k];
  }
  team_sync(team, tpr);
#pragma unroll
  for (int k = 0; k < NV; ++k) a[k] = 0.0f;
#pragma unroll 4
  for (int w = 0; w < warps; ++w) {
#pragma unroll
    for (int k = 0; k < NV; ++k) a[k] += mine[w * NV + k];
  }
}

// Eight elements as they lie in memory.
template <typename T>
struct Chunk {
  static constexpr int P = 16 / (int)sizeof(T);
  Vec<T, P> p[8 / P];
  __device__ __forceinline__ float get(int k) const { return p[k / P].get(k % P); }
  __device__ __forceinline__ F<2> pair(int k) const { return F<2>::of(get(2 * k), get(2 * k + 1)); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int q = 0; q < 8 / P; ++q) {
      float part[P];
#pragma unroll
      for (int k = 0; k < P; ++k) part[k] = f[q * P + k];
      p[q].set(part);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int q = 0; q < 8 / P; ++q) {
#pragma unroll
      for (int k = 0; k < 4; ++k) p[q].w[k] = 0;
    }
  }
  // Columns col .. col + 7 of a row of `cols`, those outside it as zero.
  template <bool WHOLE>
  __device__ __forceinline__ void load(const Mat& m, int64_t row, int col, int cols) {
    const int64_t at = row * m.stride + col;
    const T* from = static_cast<const T*>(m.p) + at;
    if (WHOLE || (m.vec && at >= 0 && at + 8 <= m.extent)) {
#pragma unroll
      for (int q = 0; q < 8 / P; ++q) p[q] = load_vec<T, P>(from + q * P);
      if (!WHOLE && (col < 0 || col + 8 > cols)) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = col + k >= 0 && col + k < cols ? get(k) : 0.0f;
        set(f);
      }
    } else {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = col + k >= 0 && col + k < cols ? to_f32(from[k]) : 0.0f;
      set(f);
    }
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(const Mat& m, int64_t row, int col, int cols) const {
    T* to = static_cast<T*>(const_cast<void*>(m.p)) + row * m.stride + col;
    if (WHOLE || (m.vec && col >= 0 && col + 8 <= cols)) {
#pragma unroll
      for (int q = 0; q < 8 / P; ++q) store_vec<T, P>(to + q * P, p[q]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + k >= 0 && col + k < cols) to[k] = from_f32<T>(get(k));
    }
  }
};

// A weight of `cols` columns in shared memory as f32, so that a warp's reads of its chunks meet no
// bank twice: without phases as 16-byte halves of the chunks, else by column modulo 8.
__host__ __device__ inline int chunk_columns(int cols) { return (cols + 7) / 8 + 1; }
template <bool WHOLE>
struct Columns {
  float* s;
  int n;  // chunk_columns(cols)
  __device__ __forceinline__ int place(int col) const {
    return WHOLE ? (((col >> 2) & 1) * n + (col >> 3)) * 4 + (col & 3) : (col & 7) * n + (col >> 3);
  }
  __device__ __forceinline__ void fill(const void* w, int dtype, int cols, float none) const {
    for (int i = threadIdx.x; i < 8 * n; i += blockDim.x)
      s[place(i)] = i >= cols ? 0.0f : w != nullptr ? load_any(w, dtype, i) : none;
  }
  __device__ __forceinline__ void read(int col, F<2> (&out)[4]) const {
    if constexpr (WHOLE) {
      const float4 lo = reinterpret_cast<const float4*>(s)[col >> 3], hi = reinterpret_cast<const float4*>(s)[n + (col >> 3)];
      out[0] = F<2>::of(lo.x, lo.y);
      out[1] = F<2>::of(lo.z, lo.w);
      out[2] = F<2>::of(hi.x, hi.y);
      out[3] = F<2>::of(hi.z, hi.w);
    } else {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = s[place(max(col + k, 0))];
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k] = F<2>::of(f[2 * k], f[2 * k + 1]);
    }
  }
};

// Walks a team over its rows.
struct Team {
  int team, lane;
  int64_t first, step;  // first row of the warp's first team, rows between turns
  int within;           // this team's place in the warp
  __device__ __forceinline__ Team(const NormArgs& a) {
    team = threadIdx.x / a.tpr;
    lane = threadIdx.x - team * a.tpr;
    const int head = a.tpr < 32 ? (threadIdx.x & ~31) / a.tpr : team;
    first = (int64_t)blockIdx.x * a.teams + head;
    within = team - head;
    step = (int64_t)gridDim.x * a.teams;
  }
};
// Elements of the row's first chunk that belong to the row before.
template <bool WHOLE>
__device__ __forceinline__ int phase_of(int64_t row, int cols) {
  return WHOLE ? 0 : (int)((uint32_t)row * (uint32_t)cols & 7u);
}

template <typename TX, typename TZ, int CH, bool FUSED, bool WHOLE>
__global__ void __launch_bounds__(max_block(CH), CH == 4 ? 1 : 2) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float scratch[2 * 32 * (kTeamBlock / 32)];
  extern __shared__ __align__(16) float columns[];
  const Team at(a);
  const int tpr = a.tpr, cols = a.cols, n = chunk_columns(cols);
  const uint64_t seed = FUSED ? uniform_seed(a.drop) : 0;
  const float inv_n = 1.0f / (float)cols;
  Chunk<TX> x[CH];
  Chunk<TZ> r[FUSED ? CH : 1];
  const auto fetch = [&](int64_t row) {
    const int col0 = at.lane * 8 - phase_of<WHOLE>(row, cols);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (row < a.rows && col < cols) {
        x[c].template load<WHOLE>(a.x, row, col, cols);
        if constexpr (FUSED) r[c].template load<WHOLE>(a.residual, row, col, cols);
      }
    }
  };
  fetch(at.first + at.within);
  const Columns<WHOLE> w{columns, n}, b{columns + 8 * n, n};
  w.fill(a.weight, a.w_dtype, cols, 1.0f);
  b.fill(a.bias, a.w_dtype, cols, 0.0f);
  __syncthreads();
  for (int64_t head = at.first; head < a.rows; head += at.step) {
    const int64_t row = head + at.within;
    const bool live = row < a.rows;
    const int phase = phase_of<WHOLE>(row, cols), col0 = at.lane * 8 - phase;
    F<2> v[CH][4], sum2 = F<2>::of(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (live && col < cols) {
        if constexpr (FUSED) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = x[c].get(k);
          const uint64_t block = (uint64_t)(row * cols + col) >> 2;
          drop_eight(a.drop, seed, (uint32_t)block, (uint32_t)(block >> 32), f);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = __fadd_rn(r[c].get(k), f[k]);
          r[c].set(f);  // the norm is of z as stored
          r[c].template store<WHOLE>(a.z, row, col, cols);
          if (!WHOLE && (col < 0 || col + 8 > cols)) {
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = col + k >= 0 && col + k < cols ? r[c].get(k) : 0.0f;
            r[c].set(f);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) v[c][k] = r[c].pair(k);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[c][k] = x[c].pair(k);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[c][k] = F<2>::of(0.0f);
      }
      sum2 = sum2 + ((v[c][0] + v[c][1]) + (v[c][2] + v[c][3]));
    }
    fetch(row + at.step);
    float sum[1] = {sum2.get(0) + sum2.get(1)};
    team_sum<1>(sum, at.team, tpr, scratch, 0);
    const float mean = sum[0] * inv_n;
    F<2> sq2 = F<2>::of(0.0f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (col < cols) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[c][k] = v[c][k] + F<2>::of(-mean);
        if (!WHOLE && (col < 0 || col + 8 > cols)) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[c][k] = F<2>::of(col + 2 * k >= 0 && col + 2 * k < cols ? v[c][k].get(0) : 0.0f,
                               col + 2 * k + 1 >= 0 && col + 2 * k + 1 < cols ? v[c][k].get(1) : 0.0f);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) sq2 = fma(v[c][k], v[c][k], sq2);
      }
    }
    float sq[1] = {sq2.get(0) + sq2.get(1)};
    team_sum<1>(sq, at.team, tpr, scratch, 1);
    const float rstd = rsqrt_rn(sq[0] * inv_n + a.eps);
    if (!live) continue;
    if (a.mean != nullptr && at.lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (col < cols) {
        F<2> ww[4], bb[4];
        w.read(col, ww);
        b.read(col, bb);
        float f[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const F<2> o = fma(v[c][k] * F<2>::of(rstd), ww[k], bb[k]);
          f[2 * k] = o.get(0);
          f[2 * k + 1] = o.get(1);
        }
        Chunk<TX> out;
        out.set(f);
        out.template store<WHOLE>(a.y, row, col, cols);
      }
    }
  }
}

// 128 registers let four CTAs of 128 threads share an SM.  Two chunks of 16-bit v fit (33000 x 1001 bf16 91 us
// against 107 us with 168 registers; fused 158 us against 170 us; fused 8192 x 4096 97 us against 119 us), two of
// f32 do not (fused 65536 x 512: 113 us with 168, 176 us with 128; under f16 x 98 us and 128 us).  Four chunks go
// up to CTAs of 544 threads.
constexpr int backward_registers(int ch, int size) { return ch == 4 ? 96 : ch == 1 ? 112 : size == 2 ? 128 : 168; }

// TV: the normalised tensor's type (x or z).  partial [gridDim.x][2][cols], or NULL.  A team's rows
// all have one phase (their distance is a multiple of 8), so a thread's columns stay its own and
// the sums of the weight gradients stay with it: in registers, or (CH = 4) in shared memory.
template <typename TX, typename TV, int CH, bool FUSED, bool WHOLE>
__global__ void __maxnreg__(backward_registers(CH, sizeof(TV))) norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr bool REGS = CH < 4;
  __shared__ float scratch[2 * 2 * 32 * (kTeamBlock / 32)];
  extern __shared__ __align__(16) float columns[];
  const Team at(a);
  const int tpr = a.tpr, cols = a.cols, n = chunk_columns(cols);
  const uint64_t seed = FUSED ? uniform_seed(a.drop) : 0;
  const float inv_n = 1.0f / (float)cols;
  const int col0 = at.lane * 8 - phase_of<WHOLE>(at.first + at.within, cols);
  // With !REGS [2][CH * 4][tpr] pairs.
  F<2>* const acc = reinterpret_cast<F<2>*>(columns + 8 * n) + at.lane;
  F<2> dw[REGS ? CH : 1][4], db[REGS ? CH : 1][4];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (REGS)
        dw[c][k] = db[c][k] = F<2>::of(0.0f);
      else
        acc[(c * 4 + k) * tpr] = acc[((CH + c) * 4 + k) * tpr] = F<2>::of(0.0f);
    }
  }
  // Rows are fetched a turn ahead where the registers hold two.
  constexpr bool AHEAD = CH <= 2, KEEP_W = CH == 1;
  Chunk<TX> next_dy[AHEAD ? CH : 1];
  Chunk<TV> next_in[AHEAD ? CH : 1];
  float next_mean = 0.0f, next_rstd = 0.0f;
  const auto fetch = [&](int64_t row, Chunk<TX>* dy, Chunk<TV>* in, float& mean, float& rstd) {
    if (row >= a.rows) return;
    mean = a.mean[row];
    rstd = a.rstd[row];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (col < cols) {
        dy[c].template load<WHOLE>(a.dy, row, col, cols);
        in[c].template load<WHOLE>(a.v, row, col, cols);
      }
    }
  };
  if constexpr (AHEAD) fetch(at.first + at.within, next_dy, next_in, next_mean, next_rstd);
  const Columns<WHOLE> w{columns, n};
  w.fill(a.weight, a.w_dtype, cols, 1.0f);
  __syncthreads();
  F<2> ww[4];
  if (KEEP_W && col0 < cols) w.read(col0, ww);
  int turn = 0;
  for (int64_t head = at.first; head < a.rows; head += at.step, ++turn) {
    const int64_t row = head + at.within;
    const bool live = row < a.rows;
    Chunk<TX> dy[CH];
    Chunk<TV> in[CH], dz[FUSED ? CH : 1];
    float mean = 0.0f, rstd = 0.0f;
    if constexpr (AHEAD) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        dy[c] = next_dy[c];
        in[c] = next_in[c];
      }
      mean = next_mean;
      rstd = next_rstd;
      fetch(row + at.step, next_dy, next_in, next_mean, next_rstd);
    } else {
      fetch(row, dy, in, mean, rstd);
    }
    if constexpr (FUSED) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = col0 + c * tpr * 8;
        if (live && col < cols && a.dz.p != nullptr) dz[c].template load<WHOLE>(a.dz, row, col, cols);
      }
    }
    const F<2> scale = F<2>::of(rstd), shift = F<2>::of(-mean);
    F<2> s0 = F<2>::of(0.0f), s1 = s0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (live && col < cols) {
        if constexpr (!KEEP_W) w.read(col, ww);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // dy is zero outside the row, and so is every sum's term there.
          const F<2> d = dy[c].pair(k), xh = (in[c].pair(k) + shift) * scale, g = d * ww[k];
          s0 = s0 + g;
          s1 = fma(g, xh, s1);
          if constexpr (REGS) {
            dw[c][k] = fma(d, xh, dw[c][k]);
            db[c][k] = db[c][k] + d;
          } else {
            F<2>&aw = acc[(c * 4 + k) * tpr], &ab = acc[((CH + c) * 4 + k) * tpr];
            aw = fma(d, xh, aw);
            ab = ab + d;
          }
        }
      }
    }
    float s[2] = {s0.get(0) + s0.get(1), s1.get(0) + s1.get(1)};
    team_sum<2>(s, at.team, tpr, scratch, turn);
    if (!live) continue;
    const F<2> m1 = F<2>::of(-s[0] * inv_n), m2 = F<2>::of(-s[1] * inv_n);
    // xh and g once more from what was read, instead of two more f32 values an element kept.
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
      if (col < cols) {
        if constexpr (!KEEP_W) w.read(col, ww);
        float dv[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const F<2> xh = (in[c].pair(k) + shift) * scale;
          F<2> o = fma(xh, m2, fma(dy[c].pair(k), ww[k], m1)) * scale;
          if constexpr (FUSED) {
            if (a.dz.p != nullptr) o = o + dz[c].pair(k);
          }
          dv[2 * k] = o.get(0);
          dv[2 * k + 1] = o.get(1);
        }
        if constexpr (FUSED) {
          if (a.dres.p != nullptr) {
            Chunk<TV> out;
            out.set(dv);
            out.template store<WHOLE>(a.dres, row, col, cols);
          }
          if (a.dx.p == nullptr) continue;
          const uint64_t block = (uint64_t)(row * cols + col) >> 2;
          drop_eight(a.drop, seed, (uint32_t)block, (uint32_t)(block >> 32), dv);
        }
        if (a.dx.p != nullptr) {
          Chunk<TX> out;
          out.set(dv);
          out.template store<WHOLE>(a.dx, row, col, cols);
        }
      }
    }
  }
  if (a.partial == nullptr) return;
  float* to = a.partial + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (REGS) {
    // Teams of a warp that share a phase, then whatever is left one after the other.
    int together = 1;  // teams summed by shuffles
    if (WHOLE && tpr < 32) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float f[4] = {dw[c][k].get(0), dw[c][k].get(1), db[c][k].get(0), db[c][k].get(1)};
          for (int o = tpr; o < 32; o <<= 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] += __shfl_xor_sync(0xffffffffu, f[i], o);
          }
          dw[c][k] = F<2>::of(f[0], f[1]);
          db[c][k] = F<2>::of(f[2], f[3]);
        }
      }
      together = 32 / tpr;
    }
    // The sums take the weight's place: [2][8 n] in its layout.
    __syncthreads();
    const Columns<WHOLE> sums[2] = {{columns, n}, {columns + 8 * n, n}};
    for (int i = threadIdx.x; i < 16 * n; i += blockDim.x) columns[i] = 0.0f;
    __syncthreads();
    for (int u = 0; u < a.teams; u += together) {
      if (at.team == u) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int col = col0 + c * tpr * 8;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (col + k >= 0 && col + k < cols) {
              sums[0].s[sums[0].place(col + k)] += dw[c][k >> 1].get(k & 1);
              sums[1].s[sums[1].place(col + k)] += db[c][k >> 1].get(k & 1);
            }
          }
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * cols; i += blockDim.x) {
      const int which = i >= cols ? 1 : 0, col = i - which * cols;
      to[i] = sums[which].s[sums[which].place(col)];
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = col0 + c * tpr * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (col + k >= 0 && col + k < cols) {
          to[col + k] = acc[(c * 4 + k / 2) * tpr].get(k & 1);
          to[cols + col + k] = acc[((CH + c) * 4 + k / 2) * tpr].get(k & 1);
        }
      }
    }
  }
}

// dweight / dbias from the CTAs' partial sums [parts][2][cols]: 32 columns per CTA, 32 threads
// deep over the parts, then a fixed tree.  A programmatic dependent launch: its launch latency lies under the
// backward, whose last CTA's end is what lets it start (the backward gives no earlier signal).
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* __restrict__ partial, int parts, int cols,
                                                                void* dweight, void* dbias, int w_dtype) {
  __shared__ float sums[32][33];
  const int which = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x;
  cudaGridDependencySynchronize();
  float s = 0.0f;
  if (col < cols) {
    const float* from = partial + (int64_t)which * cols + col;
#pragma unroll 8
    for (int p = threadIdx.y; p < parts; p += 32) s += from[(int64_t)p * 2 * cols];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sums[threadIdx.x][threadIdx.y];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  void* out = which == 0 ? dweight : dbias;
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < cols && out != nullptr) store_any(out, w_dtype, c, s);
}

// Chunks a thread takes: enough to spread a row's fixed costs (sums, barriers, square root) over, as
// far as the registers hold them.  Measured at 65536 x 1024 bf16: the forward takes 52 us with four and
// 60 us with two; the backward 87 us with two (their sums of weight gradients are registers) and
// 103 us with one.  A few rows are over before that matters, and one chunk is the shortest way
// (backward of 16 x 512: 6.7 us with one, 9.0 us with two).  The fused forward would rather have two
// (33000 x 1001: 122 us against 146 us), but it sums in the plain one's order: where types and alignment
// are the same, y has the bits of the separate norm of z.
Split make_split(const plstm_norm_desc& d, bool whole, bool backward) {
  Split s;
  const int chunks = whole ? d.cols / 8 : chunk_columns(d.cols);
  if (backward) {
    const bool few = chunks <= 257 && d.rows * chunks <= (int64_t)kSMs * kTeamBlock * 4;
    s.ch = chunks <= 48 || few ? 1 : chunks <= 513 ? 2 : 4;
  } else {
    s.ch = chunks <= 32 ? 1 : chunks <= (d.x_dtype == PLSTM_F32 ? 513 : 64) ? 2 : 4;
  }
  const int threads = (chunks + s.ch - 1) / s.ch;
  if (threads >= 32) {
    s.tpr = (threads + 31) / 32 * 32;
  } else {
    s.tpr = 1;
    while (s.tpr < threads) s.tpr *= 2;
  }
  s.teams = std::max(1, kTeamBlock / s.tpr);
  return s;
}

size_t forward_smem(const plstm_norm_desc& d) { return (size_t)16 * chunk_columns(d.cols) * sizeof(float); }
size_t backward_smem(const plstm_norm_desc& d, const Split& s) {
  const size_t n = chunk_columns(d.cols);
  return (s.ch < 4 ? 16 * n : 8 * n + (size_t)2 * 8 * s.ch * s.tpr) * sizeof(float);
}

// CTAs of a launch: what the rows need, at most as many as are resident at once (`per_sm` an SM), so
// that no second wave of a few CTAs follows the first.  The backward's rows a turn are a multiple of 8.
int64_t forward_ctas(const plstm_norm_desc& d, const Split& s, int per_sm) {
  return std::min<int64_t>((d.rows + s.teams - 1) / s.teams, (int64_t)kSMs * per_sm);
}
int64_t backward_ctas(const plstm_norm_desc& d, const Split& s, int per_sm) {
  const int64_t unit = 8 / std::min(8, s.teams & -s.teams);  // CTAs whose teams are a multiple of 8
  const int64_t need = ((d.rows + s.teams - 1) / s.teams + unit - 1) / unit * unit;
  return std::min(need, std::max(unit, (int64_t)kSMs * per_sm / unit * unit));
}
constexpr int kBackwardThreads = 1024;  // per SM, the most that the workspace provides for
int backward_most(const Split& s) { return std::max(1, kBackwardThreads / s.block()); }

// CTAs of a kernel that an SM holds, remembered for the last device, block and shared-memory size asked
// for; on a miss the kernel is also allowed all the shared memory that any shape needs (one value, so
// that threads launching different shapes do not take it back from one another).
constexpr int kMostShared = 216 * 1024;  // with the kernels' own 2 KB and the system's 1 KB below 227 KB
template <typename Kernel>
int32_t resident(Kernel kernel, std::atomic<uint64_t>& memo, int device, int block, size_t smem, int* per_sm) {
  const uint64_t key = (uint64_t)device << 52 | (uint64_t)block << 40 | (uint64_t)smem << 8, seen = memo.load(std::memory_order_relaxed);
  if ((seen & ~(uint64_t)255) == key && (seen & 255) != 0) {
    *per_sm = (int)(seen & 255);
    return PLSTM_OK;
  }
  if (smem > 40 * 1024)
    PLSTM_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
  PLSTM_TRY_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kernel, block, smem));
  *per_sm = std::max(1, *per_sm);
  memo.store(key | (uint64_t)*per_sm, std::memory_order_relaxed);
  return PLSTM_OK;
}

template <bool BACKWARD, typename Kernel>
int32_t launch(Kernel kernel, std::atomic<uint64_t>& memo, const plstm_norm_desc& d, const NormArgs& a, const Split& s,
               size_t smem, int* grid, cudaStream_t st) {
  int per_sm = 0;
  if (const int32_t rc = resident(kernel, memo, d.device, s.block(), smem, &per_sm)) return rc;
  *grid = (int)(BACKWARD ? backward_ctas(d, s, std::min(per_sm, backward_most(s))) : forward_ctas(d, s, per_sm));
  kernel<<<*grid, s.block(), smem, st>>>(a);
  PLSTM_TRY_CUDA(cudaGetLastError());
  note_launches(1);
  return PLSTM_OK;
}

template <typename TX, typename TZ, int CH, bool FUSED, bool WHOLE>
int32_t launch_kernel(bool backward, const plstm_norm_desc& d, const NormArgs& a, const Split& s, int* grid,
                      cudaStream_t st) {
  static std::atomic<uint64_t> memo[2];
  if (backward)
    return launch<true>(norm_backward_kernel<TX, TZ, CH, FUSED, WHOLE>, memo[1], d, a, s, backward_smem(d, s), grid, st);
  return launch<false>(norm_forward_kernel<TX, TZ, CH, FUSED, WHOLE>, memo[0], d, a, s, forward_smem(d), grid, st);
}

template <typename TX, typename TZ, bool FUSED, bool WHOLE>
int32_t launch_split(bool backward, const plstm_norm_desc& d, NormArgs& a, int* grid, cudaStream_t st) {
  const Split s = make_split(d, WHOLE, backward);
  a.tpr = s.tpr;
  a.teams = s.teams;
  if (s.ch == 1) return launch_kernel<TX, TZ, 1, FUSED, WHOLE>(backward, d, a, s, grid, st);
  if (s.ch == 2) return launch_kernel<TX, TZ, 2, FUSED, WHOLE>(backward, d, a, s, grid, st);
  return launch_kernel<TX, TZ, 4, FUSED, WHOLE>(backward, d, a, s, grid, st);
}

template <typename TX, typename TZ>
int32_t dispatch(bool backward, const plstm_norm_desc& d, NormArgs& a, bool fused, bool whole, int* grid, cudaStream_t st) {
  if constexpr (sizeof(TX) == sizeof(TZ)) {
    if (!fused)
      return whole ? launch_split<TX, TZ, false, true>(backward, d, a, grid, st)
                   : launch_split<TX, TZ, false, false>(backward, d, a, grid, st);
  }
  return whole ? launch_split<TX, TZ, true, true>(backward, d, a, grid, st)
               : launch_split<TX, TZ, true, false>(backward, d, a, grid, st);
}

// `grid` receives the CTAs launched.
int32_t dispatch_types(bool backward, const plstm_norm_desc& d, NormArgs& a, bool fused, bool whole, int* grid,
                       cudaStream_t st) {
  if (d.x_dtype == PLSTM_F32)
    return dispatch<float, float>(backward, d, a, fused, whole, grid, st);
  if (d.x_dtype == PLSTM_F16 && d.z_dtype == PLSTM_F16)
    return dispatch<__half, __half>(backward, d, a, fused, whole, grid, st);
  if (d.x_dtype == PLSTM_F16)
    return dispatch<__half, float>(backward, d, a, fused, whole, grid, st);
  if (d.z_dtype == PLSTM_BF16)
    return dispatch<__nv_bfloat16, __nv_bfloat16>(backward, d, a, fused, whole, grid, st);
  return dispatch<__nv_bfloat16, float>(backward, d, a, fused, whole, grid, st);
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

// A chunk at column col of row r lies at r * stride + col with r * cols + col a multiple of 8.
Mat make_mat(const plstm_norm_desc& d, const void* p, int64_t stride, int32_t dtype) {
  const int64_t size = (int64_t)dtype_size(dtype);
  if (d.rows == 1) stride = d.cols;
  return Mat{p, stride, (d.rows - 1) * stride + d.cols, aligned16(p) && (stride - d.cols) * size % 16 == 0};
}
bool all_whole(const plstm_norm_desc& d, std::initializer_list<const Mat*> all) {
  if (d.cols % 8 != 0) return false;
  for (const Mat* m : all)
    if (!m->vec) return false;
  return true;
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
  const bool fused = residual != nullptr || (d != nullptr && d->rows == 0);  // without rows a residual may be NULL
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
  a.rows = d->rows;
  a.cols = d->cols;
  a.eps = d->eps;
  a.x = make_mat(*d, x, d->x_stride, d->x_dtype);
  a.residual = make_mat(*d, residual, d->residual_stride, d->z_dtype);
  a.z = make_mat(*d, z, d->cols, d->z_dtype);
  a.y = make_mat(*d, y, d->cols, d->x_dtype);
  a.weight = weight;
  a.bias = bias;
  a.mean = stats;
  a.rstd = stats != nullptr ? stats + d->rows : nullptr;
  a.w_dtype = d->w_dtype;
  const bool whole = fused ? all_whole(*d, {&a.x, &a.residual, &a.z, &a.y}) : all_whole(*d, {&a.x, &a.y});
  int grid = 0;
  return dispatch_types(false, *d, a, fused, whole, &grid, static_cast<cudaStream_t>(stream));
}

int32_t plstm_layer_norm_backward_workspace_size(const plstm_norm_desc* d, size_t* bytes) {
  clear_error();
  PLSTM_CHECK_ARG(bytes != nullptr, "bytes is NULL");
  if (const int32_t rc = check_desc(d, true)) return rc;
  // The larger of the two splits that alignment chooses between.
  int64_t parts = 0;
  for (const bool whole : {false, d->cols % 8 == 0}) {
    const Split s = make_split(*d, whole, true);
    parts = std::max(parts, backward_ctas(*d, s, backward_most(s)));
  }
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
    a.rows = d->rows;
    a.cols = d->cols;
    a.dy = make_mat(*d, dy, d->dy_stride, d->x_dtype);
    a.dz = make_mat(*d, dz, d->dz_stride, d->z_dtype);
    a.v = make_mat(*d, v, fused ? d->cols : d->x_stride, d->z_dtype);
    a.dx = make_mat(*d, dx, d->cols, d->x_dtype);
    a.dres = make_mat(*d, dresidual, d->cols, d->z_dtype);
    a.weight = weight;
    a.mean = const_cast<float*>(stats);
    a.rstd = const_cast<float*>(stats) + d->rows;
    a.partial = grads ? static_cast<float*>(workspace) : nullptr;
    a.w_dtype = d->w_dtype;
    if (dz == nullptr) a.dz.vec = 1;
    const bool whole = all_whole(*d, {&a.dy, &a.v, &a.dx}) && (!fused || all_whole(*d, {&a.dz, &a.dres}));
    if (const int32_t rc = dispatch_types(true, *d, a, fused != 0, whole, &parts, st)) return rc;
  }
  if (grads) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((d->cols + 31) / 32, 2);
    cfg.blockDim = dim3(32, 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    PLSTM_TRY_CUDA(cudaLaunchKernelEx(&cfg, norm_weight_grad_kernel, static_cast<const float*>(workspace), parts,
                                      (int)d->cols, dweight, dbias, (int)d->w_dtype));
    note_launches(1);
  }
  return PLSTM_OK;
}

}  // extern "C"
