// Norms, gate and residual scale around a block, forward and backward:
//   u = N1(y),  s = alpha r + beta g u,  o = N2(s).
// Memory-bound: forward reads r and y and writes s and o (4 C values a row), backward reads r, y, ds, do and writes dr, dy (6 C
// values a row); nothing else of a row leaves the registers, and s is computed again in the backward pass, unrounded, instead of
// being read.  A row belongs to a team of warps and lies in its registers between the passes over it.
#include <float.h>
#include <string.h>

#include "host_common.h"
#include "row_io.cuh"

namespace souffle {

struct NormArgs {
  int rows, cols, gate_rows, branch_norm, out_norm;
  float alpha, beta, eps1, eps2;
  long long r_stride, y_stride, s_stride, o_stride, q_stride;
  const void *r, *y, *gate, *w1, *b1, *w2, *b2;
  void *s, *o;
  signed char* q;
  float* q_scale;
};

// Rows of a gate: row m takes gate row m / (rows / gate_rows).
__device__ __forceinline__ int gate_row(const NormArgs& a, int row) { return row / (a.rows / a.gate_rows); }

template <class T, class P, bool kVec, int kGroups>
__global__ void __launch_bounds__(256) souffle_residual_norm(const NormArgs a, int warps_per_row) {
  __shared__ __align__(16) char box[kTeamBox];
  const int teams = blockDim.x / (32 * warps_per_row), warp = threadIdx.x >> 5;
  const int row = blockIdx.x * teams + warp / warps_per_row;       // several teams only where a team is one warp
  if (row >= a.rows) return;
  const Columns<kVec> cols = {(int)(threadIdx.x % (32 * warps_per_row)), 32 * warps_per_row, a.cols};
  Team team;
  team.begin(box, warps_per_row, warp % warps_per_row, 1, cols, kGroups);

  float u[kGroups][8], h[kGroups][8], v[8];
  const T* y = static_cast<const T*>(a.y) + row * a.y_stride;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) cols.load(y, i, u[i]);
  if (a.r) {
    const T* r = static_cast<const T*>(a.r) + row * a.r_stride;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) cols.load(r, i, h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
  }
  if (a.branch_norm != SOUFFLE_NORM_NONE) {
    const float2 st = row_stats<kGroups>(team, cols, u, a.branch_norm == SOUFFLE_NORM_RMS, a.eps1);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[i][j] = (u[i][j] - st.x) * st.y;
      if (a.w1) {
        cols.load(static_cast<const P*>(a.w1), i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[i][j] *= v[j];
      }
      if (a.b1) {
        cols.load(static_cast<const P*>(a.b1), i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[i][j] += v[j];
      }
    }
  }
  if (a.gate) {
    const P* g = static_cast<const P*>(a.gate) + (long long)gate_row(a, row) * a.cols;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      cols.load(g, i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[i][j] *= v[j];
    }
  }
#pragma unroll
  for (int i = 0; i < kGroups; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = cols.has(i, j) ? fmaf(a.alpha, h[i][j], a.beta * u[i][j]) : 0.0f;
  if (a.s) {
    T* s = static_cast<T*>(a.s) + row * a.s_stride;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) cols.store(s, i, h[i]);
  }
  if (a.out_norm == SOUFFLE_NORM_NONE) return;
  const float2 st = row_stats<kGroups>(team, cols, h, a.out_norm == SOUFFLE_NORM_RMS, a.eps2);
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = (h[i][j] - st.x) * st.y;
    if (a.w2) {
      cols.load(static_cast<const P*>(a.w2), i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= v[j];
    }
    if (a.b2) {
      cols.load(static_cast<const P*>(a.b2), i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] += v[j];
    }
  }
  if (a.o) {
    T* o = static_cast<T*>(a.o) + row * a.o_stride;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) cols.store(o, i, h[i]);
  }
  if (a.q) quantise_row<kGroups>(team, cols, h, a.q + row * a.q_stride, a.q_scale + row);
}

// ---- backward ----------------------------------------------------------------------------------------------------
//   ds' = ds + N2'(do),  dr = alpha ds',  du = beta g ds',  dg = sum beta ds' u,  dy = N1'(du),
//   N'(d) = (w d - mean(w d) - xhat mean(w d xhat)) / deviation  (rms: without the mean of w d),  dw = sum d xhat,  db = sum d.
// The sums over rows: a team takes consecutive rows and keeps its columns' five sums in registers; the teams of a CTA are added
// through shared memory, the CTAs by a second, small kernel, all in a fixed order.  Gates that change within the batch are
// written when their last row is done: directly where one team had all their rows, otherwise into the team's slot 0 (a gate
// whose first row is the team's first or lies before it) or 1 (a later one).
enum { SUM_W1 = 0, SUM_B1 = 1, SUM_W2 = 2, SUM_B2 = 3, SUM_GATE = 4, SUMS = 5 };

struct NormGradArgs {
  NormArgs f;
  long long ds_stride, do_stride, dr_stride, dy_stride;
  const void *ds, *dout;
  void *dr, *dy, *dgate, *dvec[4];     // dvec: SUM_W1 .. SUM_B2
  float *part, *slots;                 // [ctas][SUMS][cols], [teams][2][cols]
  int teams;                           // of the whole grid
};

__device__ __forceinline__ int first_row(long long team, int rows, int teams) { return (int)(team * rows / teams); }

// kSharedSums: the sums lie in shared memory, [SUMS][8][threads], where 1024 threads leave no registers for them.
template <class T, class P, bool kVec, bool kSharedSums>
__global__ void __launch_bounds__(kSharedSums ? 1024 : 512) souffle_residual_norm_grad(const NormGradArgs g, int warps_per_row) {
  extern __shared__ __align__(16) char smem[];
  const NormArgs& a = g.f;
  const int teams = blockDim.x / (32 * warps_per_row), warp = threadIdx.x >> 5, mine = warp / warps_per_row;
  const int id = blockIdx.x * teams + mine;
  const Columns<kVec> cols = {(int)(threadIdx.x % (32 * warps_per_row)), 32 * warps_per_row, a.cols};
  Team team;
  team.begin(smem + mine * kTeamBox, warps_per_row, warp % warps_per_row, 1 + mine, cols, 1);
  float* sums = reinterpret_cast<float*>(smem + teams * kTeamBox);

  float acc[SUMS][8];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (kSharedSums) sums[(k * 8 + j) * blockDim.x + threadIdx.x] = 0.0f;
      else acc[k][j] = 0.0f;
    }
  auto add = [&](int k, int j, float v) {
    if (kSharedSums) sums[(k * 8 + j) * blockDim.x + threadIdx.x] += v;
    else acc[k][j] += v;
  };
  auto take = [&](int k, float (&v)[8], bool clear) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float& at = kSharedSums ? sums[(k * 8 + j) * blockDim.x + threadIdx.x] : acc[k][j];
      v[j] = at;
      if (clear) at = 0.0f;
    }
  };

  const int begin = first_row(id, a.rows, g.teams), end = first_row(id + 1LL, a.rows, g.teams);
  const int per_gate = a.gate ? a.rows / a.gate_rows : 0;
  const bool n1 = a.branch_norm != SOUFFLE_NORM_NONE, n2 = a.out_norm != SOUFFLE_NORM_NONE;
  for (int row = begin; row < end; ++row) {
    float y[8], h[8], d[8], e[8], w[8], gate[8];
    cols.load(static_cast<const T*>(a.y) + row * a.y_stride, 0, y);
    if (a.r) {
      cols.load(static_cast<const T*>(a.r) + row * a.r_stride, 0, h);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = 0.0f;
    }
    if (g.ds) {
      cols.load(static_cast<const T*>(g.ds) + row * g.ds_stride, 0, d);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = 0.0f;
    }
    if (n2) cols.load(static_cast<const T*>(g.dout) + row * g.do_stride, 0, e);
    if (a.gate) {
      cols.load(static_cast<const P*>(a.gate) + (long long)(row / per_gate) * a.cols, 0, gate);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) gate[j] = 1.0f;
    }
    float u[8], rstd1 = 1.0f;
    if (n1) {                          // y becomes yhat, u = N1(y)
      float (&y1)[1][8] = *reinterpret_cast<float (*)[1][8]>(&y);
      const float2 st = row_stats<1>(team, cols, y1, a.branch_norm == SOUFFLE_NORM_RMS, a.eps1);
      rstd1 = st.y;
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = y[j] = cols.has(0, j) ? (y[j] - st.x) * st.y : 0.0f;
      if (a.w1) {
        cols.load(static_cast<const P*>(a.w1), 0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] *= w[j];
      }
      if (a.b1) {
        cols.load(static_cast<const P*>(a.b1), 0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] += w[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = y[j];
    }
    if (n2) {                          // h becomes hhat, d the gradient of s
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = fmaf(a.alpha, h[j], a.beta * (gate[j] * u[j]));
      float (&h1)[1][8] = *reinterpret_cast<float (*)[1][8]>(&h);
      const float2 st = row_stats<1>(team, cols, h1, a.out_norm == SOUFFLE_NORM_RMS, a.eps2);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[j] = cols.has(0, j) ? (h[j] - st.x) * st.y : 0.0f;
        if (g.dvec[SUM_W2]) add(SUM_W2, j, e[j] * h[j]);
        if (g.dvec[SUM_B2]) add(SUM_B2, j, e[j]);
      }
      if (a.w2) {
        cols.load(static_cast<const P*>(a.w2), 0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] *= w[j];
      }
      float2 m = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m.x += e[j];
        m.y = fmaf(e[j], h[j], m.y);
      }
      m = team.sum(m);
      m.x = a.out_norm == SOUFFLE_NORM_RMS ? 0.0f : m.x * team.inv_cols;
      m.y *= team.inv_cols;
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = fmaf(st.y, e[j] - m.x - h[j] * m.y, d[j]);
    }
    if (g.dr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = a.alpha * d[j];
      cols.store(static_cast<T*>(g.dr) + row * g.dr_stride, 0, w);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      d[j] *= a.beta;
      if (g.dgate) add(SUM_GATE, j, d[j] * u[j]);
      d[j] *= gate[j];
    }
    if (n1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (g.dvec[SUM_W1]) add(SUM_W1, j, d[j] * y[j]);
        if (g.dvec[SUM_B1]) add(SUM_B1, j, d[j]);
      }
      if (a.w1) {
        cols.load(static_cast<const P*>(a.w1), 0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] *= w[j];
      }
      float2 m = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (cols.has(0, j)) m.x += d[j];
        m.y = fmaf(d[j], y[j], m.y);
      }
      m = team.sum(m);
      m.x = a.branch_norm == SOUFFLE_NORM_RMS ? 0.0f : m.x * team.inv_cols;
      m.y *= team.inv_cols;
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = rstd1 * (d[j] - m.x - y[j] * m.y);
    }
    if (g.dy) cols.store(static_cast<T*>(g.dy) + row * g.dy_stride, 0, d);
    if (g.dgate && a.gate_rows > 1 && ((row + 1) % per_gate == 0 || row + 1 == end)) {
      const int first = row / per_gate * per_gate;
      float v[8];
      take(SUM_GATE, v, true);
      if (first >= begin && first + per_gate <= end) cols.store(static_cast<P*>(g.dgate) + (long long)(row / per_gate) * a.cols, 0, v);
      else cols.store(g.slots + (2LL * id + (first > begin)) * a.cols, 0, v);
    }
  }

  // the teams of the CTA, one sum at a time
  const bool have[SUMS] = {g.dvec[SUM_W1] != nullptr, g.dvec[SUM_B1] != nullptr, g.dvec[SUM_W2] != nullptr, g.dvec[SUM_B2] != nullptr,
                           g.dgate && a.gate_rows == 1};
#pragma unroll
  for (int k = 0; k < SUMS; ++k) {
    if (!have[k]) continue;
    float* part = g.part + ((long long)blockIdx.x * SUMS + k) * a.cols;
    float v[8];
    take(k, v, false);
    if (teams == 1) {
      cols.store(part, 0, v);
      continue;
    }
    for (int t = 0; t < teams; ++t) {
      __syncthreads();
      if (t == mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (cols.has(0, j)) sums[cols.at(0, j)] = t == 0 ? v[j] : sums[cols.at(0, j)] + v[j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) part[c] = sums[c];
  }
}

// Adds up what the CTAs left.  y < 4: a vector's sum; y = 4: the one gate row's; y = SUMS + t: that of the gate whose last rows are
// team t's and whose first ones are not (any other gate was written by its one team).
constexpr int kFinishLanes = 16;
template <class P>
__global__ void __launch_bounds__(32 * kFinishLanes) souffle_residual_norm_grad_sums(const NormGradArgs g, int ctas) {
  __shared__ float sm[kFinishLanes][33];
  const NormArgs& a = g.f;
  const int cx = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + cx, k = blockIdx.y;
  P* to;
  float v = 0.0f;
  if (k < SUMS) {
    to = static_cast<P*>(k < SUM_GATE ? g.dvec[k] : a.gate_rows == 1 ? g.dgate : nullptr);
    if (!to) return;
    if (c < a.cols)
      for (int i = lane; i < ctas; i += kFinishLanes) v += g.part[((long long)i * SUMS + k) * a.cols + c];
  } else {
    const int t1 = k - SUMS, per_gate = a.rows / a.gate_rows, begin = first_row(t1, a.rows, g.teams), end = first_row(t1 + 1LL, a.rows, g.teams);
    const int first = begin / per_gate * per_gate;
    if (first == begin || begin == end || first + per_gate > end) return;
    const int t0 = (int)(((first + 1LL) * g.teams - 1) / a.rows);       // the team of row `first`
    to = static_cast<P*>(g.dgate) + (long long)(begin / per_gate) * a.cols;
    if (c < a.cols)
      for (int t = t0 + lane; t <= t1; t += kFinishLanes) {
        const int from = first_row(t, a.rows, g.teams);
        if (from < first_row(t + 1LL, a.rows, g.teams)) v += g.slots[(2LL * t + (first > from)) * a.cols + c];
      }
  }
  sm[lane][cx] = v;
  __syncthreads();
  if (lane || c >= a.cols) return;
  for (int i = 1; i < kFinishLanes; ++i) v += sm[i][cx];
  to[c] = from_f32<P>(v);
}

// ---- host --------------------------------------------------------------------------------------------------------

constexpr int kMaxNormCols = 8192;

static size_t dtype_size(int t) { return t == SOUFFLE_F32 ? 4 : 2; }
// whether rows of `stride` elements from `p` on can be read 16 bytes at a time
static bool wide_rows(const void* p, long long stride, size_t size) { return !p || (((uintptr_t)p | (uintptr_t)(stride * (long long)size)) & 15u) == 0; }

static int check_norm(const SouffleResidualNorm& d, bool forward, bool* vec) {
  if (d.rows < 0 || d.cols < 1 || d.cols > kMaxNormCols)
    return fail(SOUFFLE_BAD_SHAPE, "residual norm of %d x %d: rows >= 0 and 1 <= cols <= %d are wanted", d.rows, d.cols, kMaxNormCols);
  if (d.dtype < SOUFFLE_F32 || d.dtype > SOUFFLE_BF16 || (d.param_dtype != d.dtype && d.param_dtype != SOUFFLE_F32))
    return fail(SOUFFLE_BAD_ARGUMENT, "dtype %d with param_dtype %d: values are fp32, fp16 or bf16, vectors the same or fp32", d.dtype, d.param_dtype);
  for (int n : {d.branch_norm, d.out_norm})
    if (n < SOUFFLE_NORM_NONE || n > SOUFFLE_NORM_RMS) return fail(SOUFFLE_BAD_ARGUMENT, "norm %d is none of SOUFFLE_NORM_*", n);
  if (!(d.branch_eps >= 0.0f) || !(d.out_eps >= 0.0f)) return fail(SOUFFLE_BAD_ARGUMENT, "eps must not be negative or NaN");
  if ((d.branch_norm == SOUFFLE_NORM_NONE && (d.branch_weight || d.branch_bias)) || (d.out_norm == SOUFFLE_NORM_NONE && (d.out_weight || d.out_bias)))
    return fail(SOUFFLE_BAD_ARGUMENT, "a weight or bias without its norm");
  if ((d.branch_norm == SOUFFLE_NORM_RMS && d.branch_bias) || (d.out_norm == SOUFFLE_NORM_RMS && d.out_bias))
    return fail(SOUFFLE_BAD_ARGUMENT, "a root-mean-square norm has no bias");
  if ((d.gate != nullptr) != (d.gate_rows != 0) || d.gate_rows < 0 || (d.gate_rows > 0 && d.rows % d.gate_rows != 0))
    return fail(SOUFFLE_BAD_SHAPE, "gate of %d rows for %d rows: it has to divide them", d.gate_rows, d.rows);
  if (d.rows > 0 && !d.branch) return fail(SOUFFLE_BAD_POINTER, "null branch");
  if (d.residual_stride < (d.residual ? d.cols : 0) || d.branch_stride < d.cols) return fail(SOUFFLE_BAD_SHAPE, "rows overlap: a stride is below %d", d.cols);
  if (forward) {
    if ((d.sum && d.sum_stride < d.cols) || (d.out && d.out_stride < d.cols) || (d.out_q && d.out_q_stride < d.cols))
      return fail(SOUFFLE_BAD_SHAPE, "rows overlap: a stride is below %d", d.cols);
    if (d.out_norm == SOUFFLE_NORM_NONE && (d.out || d.out_q)) return fail(SOUFFLE_BAD_ARGUMENT, "out without a norm for it");
    if (d.rows > 0 && !d.sum && !d.out && !d.out_q) return fail(SOUFFLE_BAD_POINTER, "nothing to write");
    if ((d.out_q != nullptr) != (d.out_scale != nullptr)) return fail(SOUFFLE_BAD_POINTER, "out_q and out_scale come together");
    if (d.out_q && (!aligned16(d.out_q) || d.out_q_stride % 16)) return fail(SOUFFLE_BAD_POINTER, "quantised rows begin on 16-byte boundaries");
  }
  const size_t e = dtype_size(d.dtype);
  for (const void* p : {d.residual, d.branch, (const void*)d.sum, (const void*)d.out})
    if ((uintptr_t)p % e) return fail(SOUFFLE_BAD_POINTER, "a matrix is not aligned to its elements");
  for (const void* p : {d.gate, d.branch_weight, d.branch_bias, d.out_weight, d.out_bias})
    if ((uintptr_t)p % dtype_size(d.param_dtype)) return fail(SOUFFLE_BAD_POINTER, "a vector is not aligned to its elements");
  if ((uintptr_t)d.out_scale % 4) return fail(SOUFFLE_BAD_POINTER, "out_scale is not aligned to its elements");
  *vec = d.cols % 8 == 0 && wide_rows(d.residual, d.residual_stride, e) && wide_rows(d.branch, d.branch_stride, e) &&
         (!forward || (wide_rows(d.sum, d.sum_stride, e) && wide_rows(d.out, d.out_stride, e)));
  for (const void* p : {d.gate, d.branch_weight, d.branch_bias, d.out_weight, d.out_bias}) *vec = *vec && wide_rows(p, 0, 1);
  return SOUFFLE_OK;
}

static NormArgs norm_args(const SouffleResidualNorm& d) {
  NormArgs a;
  memset(&a, 0, sizeof(a));
  a.rows = d.rows; a.cols = d.cols; a.gate_rows = d.gate_rows; a.branch_norm = d.branch_norm; a.out_norm = d.out_norm;
  a.alpha = d.residual_scale; a.beta = d.branch_scale; a.eps1 = d.branch_eps; a.eps2 = d.out_eps;
  a.r_stride = d.residual_stride; a.y_stride = d.branch_stride; a.s_stride = d.sum_stride; a.o_stride = d.out_stride; a.q_stride = d.out_q_stride;
  a.r = d.residual; a.y = d.branch; a.gate = d.gate;
  a.w1 = d.branch_weight; a.b1 = d.branch_bias; a.w2 = d.out_weight; a.b2 = d.out_bias;
  a.s = d.sum; a.o = d.out; a.q = static_cast<signed char*>(d.out_q); a.q_scale = d.out_scale;
  return a;
}

template <class T, class P, bool kVec>
static int forward_groups(const NormArgs& a, cudaStream_t st) {
  const int groups8 = (a.cols + 7) / 8;
  // A warp per row up to 1024 columns, several beyond that, four groups of eight columns a thread.
  const int warps = groups8 <= 128 ? 1 : (groups8 + 127) / 128;
  const int groups = (groups8 + 32 * warps - 1) / (32 * warps);
  const int threads = warps == 1 ? 128 : 32 * warps, teams = threads / (32 * warps);
  const int grid = (a.rows + teams - 1) / teams;
  switch (groups) {
    case 1: souffle_residual_norm<T, P, kVec, 1><<<grid, threads, 0, st>>>(a, warps); break;
    case 2: souffle_residual_norm<T, P, kVec, 2><<<grid, threads, 0, st>>>(a, warps); break;
    case 3: souffle_residual_norm<T, P, kVec, 3><<<grid, threads, 0, st>>>(a, warps); break;
    default: souffle_residual_norm<T, P, kVec, 4><<<grid, threads, 0, st>>>(a, warps); break;
  }
  SF_CUDA(cudaGetLastError());
  return SOUFFLE_OK;
}

// The grid of the backward kernel: teams of `warps` warps, as many in a CTA as its registers allow, at most one row each.
struct GradGrid { int warps, per_cta, ctas; };
static GradGrid grad_grid(int rows, int cols, int sms) {
  GradGrid g;
  g.warps = (cols + 255) / 256;
  g.per_cta = g.warps > 16 ? 1 : 16 / g.warps > 15 ? 15 : 16 / g.warps;       // named barriers 1 .. 15
  const int need = (rows + g.per_cta - 1) / g.per_cta;
  g.ctas = need < sms ? need : sms;
  return g;
}

template <class T, class P, bool kVec, bool kSharedSums>
static int backward_launch(NormGradArgs& g, const GradGrid& gg, cudaStream_t st) {
  auto fn = souffle_residual_norm_grad<T, P, kVec, kSharedSums>;
  const int threads = 32 * gg.warps * gg.per_cta;
  const int smem = gg.per_cta * kTeamBox + (kSharedSums ? SUMS * 8 * threads : gg.per_cta > 1 ? g.f.cols : 0) * (int)sizeof(float);
  if (smem > 48 * 1024) SF_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  fn<<<gg.ctas, threads, smem, st>>>(g, gg.warps);
  SF_CUDA(cudaGetLastError());
  const bool gates = g.dgate && g.f.gate_rows > 1;
  bool any = g.dgate;
  for (void* p : g.dvec) any = any || p;
  if (any) {
    souffle_residual_norm_grad_sums<P><<<dim3((g.f.cols + 31) / 32, SUMS + (gates ? g.teams : 0)), 32 * kFinishLanes, 0, st>>>(g, gg.ctas);
    SF_CUDA(cudaGetLastError());
  }
  return SOUFFLE_OK;
}

// Calls f with the types of (dtype, param_dtype) as arguments' types.
template <class F> static int with_types(int dtype, int param_dtype, F f) {
  if (dtype == SOUFFLE_F32) return f(0.0f, 0.0f);
  if (dtype == SOUFFLE_F16) return param_dtype == SOUFFLE_F32 ? f(__half(), 0.0f) : f(__half(), __half());
  return param_dtype == SOUFFLE_F32 ? f(__nv_bfloat16(), 0.0f) : f(__nv_bfloat16(), __nv_bfloat16());
}

}  // namespace souffle

using namespace souffle;

extern "C" {

int souffle_residual_norm_forward(const SouffleResidualNorm* call, souffle_stream_t stream) {
  if (!call) return fail(SOUFFLE_BAD_ARGUMENT, "null call record");
  bool vec = false;
  int rc = check_norm(*call, true, &vec), sms;
  if (rc || call->rows == 0) return rc;
  if ((rc = current_sms(&sms))) return rc;
  const NormArgs a = norm_args(*call);
  return with_types(call->dtype, call->param_dtype, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    return vec ? forward_groups<T, P, true>(a, (cudaStream_t)stream) : forward_groups<T, P, false>(a, (cudaStream_t)stream);
  });
}

// The largest grid that any device of this library's kind gives: it has at most 160 SMs.
static constexpr int kMostSms = 160;
size_t souffle_residual_norm_backward_workspace_bytes(int32_t rows, int32_t cols, int32_t gate_rows) {
  if (rows < 1 || cols < 1 || cols > kMaxNormCols) return 0;
  const GradGrid g = grad_grid(rows, cols, kMostSms);
  return ((size_t)g.ctas * SUMS + (gate_rows > 1 ? 2 * (size_t)g.ctas * g.per_cta : 0)) * cols * sizeof(float);
}

int souffle_residual_norm_backward(const SouffleResidualNormGrad* call, souffle_stream_t stream) {
  if (!call) return fail(SOUFFLE_BAD_ARGUMENT, "null call record");
  const SouffleResidualNorm& d = call->f;
  bool vec = false;
  int rc = check_norm(d, false, &vec), sms = 0;
  if (rc) return rc;
  const bool n2 = d.out_norm != SOUFFLE_NORM_NONE;
  if (d.rows > 0 && n2 != (call->grad_out != nullptr)) return fail(SOUFFLE_BAD_POINTER, "grad_out comes with a norm of the sum");
  if (d.rows > 0 && !n2 && !call->grad_sum) return fail(SOUFFLE_BAD_POINTER, "null grad_sum");
  if ((call->d_branch_weight && d.branch_norm == SOUFFLE_NORM_NONE) || (call->d_branch_bias && d.branch_norm != SOUFFLE_NORM_LAYER) ||
      (call->d_out_weight && !n2) || (call->d_out_bias && d.out_norm != SOUFFLE_NORM_LAYER) || (call->d_gate && !d.gate) || (call->d_residual && !d.residual))
    return fail(SOUFFLE_BAD_ARGUMENT, "a gradient of something that is not there");
  const size_t e = dtype_size(d.dtype), pe = dtype_size(d.param_dtype);
  const struct { const void* p; int64_t stride; } mats[4] = {{call->grad_sum, call->grad_sum_stride}, {call->grad_out, call->grad_out_stride},
                                                             {call->d_residual, call->d_residual_stride}, {call->d_branch, call->d_branch_stride}};
  for (auto& m : mats) {
    if (m.p && m.stride < d.cols) return fail(SOUFFLE_BAD_SHAPE, "rows overlap: a stride is below %d", d.cols);
    if ((uintptr_t)m.p % e) return fail(SOUFFLE_BAD_POINTER, "a matrix is not aligned to its elements");
    vec = vec && wide_rows(m.p, m.stride, e);
  }
  for (const void* p : {call->d_gate, call->d_branch_weight, call->d_branch_bias, call->d_out_weight, call->d_out_bias}) {
    if ((uintptr_t)p % pe) return fail(SOUFFLE_BAD_POINTER, "a vector is not aligned to its elements");
    vec = vec && wide_rows(p, 0, 1);
  }
  if (d.rows == 0) {                   // sums over no rows
    for (void* p : {call->d_branch_weight, call->d_branch_bias, call->d_out_weight, call->d_out_bias})
      if (p) SF_CUDA(cudaMemsetAsync(p, 0, pe * d.cols, (cudaStream_t)stream));
    if (call->d_gate) SF_CUDA(cudaMemsetAsync(call->d_gate, 0, pe * d.cols * d.gate_rows, (cudaStream_t)stream));
    return SOUFFLE_OK;
  }
  if (!aligned16(call->workspace) || call->workspace_bytes < souffle_residual_norm_backward_workspace_bytes(d.rows, d.cols, d.gate_rows))
    return fail(SOUFFLE_BAD_POINTER, "workspace is null, misaligned or smaller than souffle_residual_norm_backward_workspace_bytes()");
  if ((rc = current_sms(&sms))) return rc;
  const GradGrid gg = grad_grid(d.rows, d.cols, sms < kMostSms ? sms : kMostSms);
  NormGradArgs g;
  memset(&g, 0, sizeof(g));
  g.f = norm_args(d);
  g.ds_stride = call->grad_sum_stride; g.do_stride = call->grad_out_stride; g.dr_stride = call->d_residual_stride; g.dy_stride = call->d_branch_stride;
  g.ds = call->grad_sum; g.dout = call->grad_out;
  g.dr = call->d_residual; g.dy = call->d_branch; g.dgate = call->d_gate;
  g.dvec[SUM_W1] = call->d_branch_weight; g.dvec[SUM_B1] = call->d_branch_bias; g.dvec[SUM_W2] = call->d_out_weight; g.dvec[SUM_B2] = call->d_out_bias;
  g.part = static_cast<float*>(call->workspace);
  g.slots = g.part + (size_t)gg.ctas * SUMS * d.cols;
  g.teams = gg.ctas * gg.per_cta;
  return with_types(d.dtype, d.param_dtype, [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    cudaStream_t st = (cudaStream_t)stream;
    if (gg.warps > 16) return vec ? backward_launch<T, P, true, true>(g, gg, st) : backward_launch<T, P, false, true>(g, gg, st);
    return vec ? backward_launch<T, P, true, false>(g, gg, st) : backward_launch<T, P, false, false>(g, gg, st);
  });
}

}  // extern "C"
