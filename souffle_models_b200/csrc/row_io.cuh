// Rows of fp32, fp16 or bf16 values in the registers of a team of warps: which thread holds which columns, loads and stores,
// sums over the team and a row's statistics.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace souffle {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight neighbouring values, from and to 16-byte aligned memory.
template <class T> struct alignas(16) Eight { T v[8]; };
template <class T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f32(e.v[j]);
}
template <class T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  Eight<T> e;
#pragma unroll
  for (int j = 0; j < 8; ++j) e.v[j] = from_f32<T>(v[j]);
  *reinterpret_cast<Eight<T>*>(p) = e;
}

// The columns that thread `t` of a team of `team` threads holds: with kVec, group i is the eight columns from 8 (t + i team) on; without,
// its eight columns are `team` apart, so that a team reads neighbouring elements whatever the alignment.
template <bool kVec> struct Columns {
  int t, team, cols;
  __device__ __forceinline__ int at(int i, int j) const { return kVec ? 8 * (t + i * team) + j : (8 * i + j) * team + t; }
  __device__ __forceinline__ bool has(int i, int j) const { return kVec ? 8 * (t + i * team) < cols : at(i, j) < cols; }
  // (pointer to a row) -> group i; columns past the row read as 0
  template <class T> __device__ __forceinline__ void load(const T* row, int i, float (&v)[8]) const {
    if (kVec) {
      if (has(i, 0)) {
        load8(row + at(i, 0), v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = has(i, j) ? to_f32(row[at(i, j)]) : 0.0f;
    }
  }
  template <class T> __device__ __forceinline__ void store(T* row, int i, const float (&v)[8]) const {
    if (kVec) {
      if (has(i, 0)) store8(row + at(i, 0), v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (has(i, j)) row[at(i, j)] = from_f32<T>(v[j]);
    }
  }
  __device__ __forceinline__ int count(int groups) const {        // how many of the row's columns the thread holds
    int n = 0;
    for (int i = 0; i < groups; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) n += has(i, j);
    return n;
  }
};

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A team of warps that works on one row.  `box` is its shared memory, 2 x 32 float2, used in turn, so that one barrier an
// exchange is enough: a warp that writes a half again has left the barrier behind the other half's exchange, in front of which
// everybody had read this one.
constexpr int kTeamBox = 64 * sizeof(float2) + 32 * sizeof(float);
struct Team {
  int warps, warp, lane, barrier;      // barrier: a named one of the team's own
  float2* box;
  float* counts;                       // shared: columns that each warp holds
  int turn;
  float inv_cols, warp_cols;           // 1 / columns of the row; columns that this warp holds
  // `all`: shared memory of kTeamBox bytes; readers of `counts` come behind the first exchange's barrier
  template <bool kVec>
  __device__ __forceinline__ void begin(char* all, int warps_, int warp_, int barrier_, const Columns<kVec>& cols, int groups) {
    warps = warps_;
    warp = warp_;
    lane = threadIdx.x & 31;
    barrier = barrier_;
    box = reinterpret_cast<float2*>(all);
    counts = reinterpret_cast<float*>(all + 64 * sizeof(float2));
    turn = 0;
    inv_cols = 1.0f / (float)cols.cols;
    warp_cols = (float)__reduce_add_sync(0xffffffffu, cols.count(groups));
    if (warps > 1 && lane == 0) counts[warp] = warp_cols;
  }
  __device__ __forceinline__ void gather(float2 mine) {
    turn ^= 32;
    if (lane == 0) box[turn + warp] = mine;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(32 * warps) : "memory");
  }
  // sums of both over the team, the same bits in every thread
  __device__ __forceinline__ float2 sum(float2 v) {
    v.x = warp_total(v.x);
    v.y = warp_total(v.y);
    if (warps == 1) return v;
    gather(v);
    v = box[turn];
    for (int w = 1; w < warps; ++w) {
      v.x += box[turn + w].x;
      v.y += box[turn + w].y;
    }
    return v;
  }
};

// Largest of the bits of |x| over the team: as integers, so that an infinity or a NaN beats every number.
__device__ __forceinline__ uint32_t team_max_bits(Team& team, uint32_t bits) {
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (team.warps == 1) return bits;
  team.gather(make_float2(__uint_as_float(bits), 0.0f));
  for (int w = 0; w < team.warps; ++w) bits = max(bits, __float_as_uint(team.box[team.turn + w].x));
  return bits;
}

// (mean, 1 / sqrt(var + eps)) of a row.  Layer: warps take their own mean and squared deviations from it (two passes over
// registers) and merge by  M2 = sum_w M2_w + n_w (mean_w - mean)^2.  Rms: mean 0.
template <int kGroups, bool kVec>
__device__ __forceinline__ float2 row_stats(Team& team, const Columns<kVec>& cols, const float (&x)[kGroups][8], bool rms, float eps) {
  float a = 0.0f;
  if (rms) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) a = fmaf(x[i][j], x[i][j], a);       // columns past the row hold 0
    a = team.sum(make_float2(a, 0.0f)).x;
    return make_float2(0.0f, rsqrtf(a * team.inv_cols + eps));
  }
#pragma unroll
  for (int i = 0; i < kGroups; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) a += x[i][j];
  a = warp_total(a);
  const float mean_w = a / fmaxf(team.warp_cols, 1.0f);
  float m2 = 0.0f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = cols.has(i, j) ? x[i][j] - mean_w : 0.0f;
      m2 = fmaf(d, d, m2);
    }
  m2 = warp_total(m2);
  float mean = mean_w;
  if (team.warps > 1) {
    team.gather(make_float2(a, m2));
    mean = 0.0f;
    for (int w = 0; w < team.warps; ++w) mean += team.box[team.turn + w].x;
    mean *= team.inv_cols;
    m2 = 0.0f;
    for (int w = 0; w < team.warps; ++w) {
      const float2 of = team.box[team.turn + w];
      const float n = team.counts[w], d = of.x / fmaxf(n, 1.0f) - mean;
      m2 += fmaf(n * d, d, of.y);
    }
  }
  return make_float2(mean, rsqrtf(m2 * team.inv_cols + eps));
}

// A row in 8-bit integers: q = rint(x min(127 / a, FLT_MAX)) with a = max |x|, scale a / 127.  A row with an infinity or a NaN has scale
// NaN and q = 0, so that whatever is multiplied with it is NaN.  (The multiplier is clamped for rows of zeros and of values so
// small that 127 / a overflows.)
struct RowScale { float inv, scale; };
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return {0.0f, __uint_as_float(0x7fc00000u)};
  const float a = __uint_as_float(max_bits);
  return {fminf(127.0f / a, 3.402823466e38f), a / 127.0f};
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// four values, in the order of the bytes
__device__ __forceinline__ uint32_t pack_s8(float a, float b, float c, float d) {
  return (uint32_t)(__float2int_rn(a) & 255) | (uint32_t)(__float2int_rn(b) & 255) << 8 | (uint32_t)(__float2int_rn(c) & 255) << 16 |
         (uint32_t)(__float2int_rn(d)) << 24;
}
template <int kGroups, bool kVec>
__device__ __forceinline__ void quantise_row(Team& team, const Columns<kVec>& cols, const float (&x)[kGroups][8], signed char* q, float* scale) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kGroups; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (cols.has(i, j)) most = max(most, abs_bits(x[i][j]));
  most = team_max_bits(team, most);
  const RowScale rs = row_scale(most);
  const bool fine = most < 0x7f800000u;      // 0 * inf is no number
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fine ? x[i][j] * rs.inv : 0.0f;
    if (kVec) {
      if (cols.has(i, 0)) *reinterpret_cast<uint2*>(q + cols.at(i, 0)) = make_uint2(pack_s8(v[0], v[1], v[2], v[3]), pack_s8(v[4], v[5], v[6], v[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (cols.has(i, j)) q[cols.at(i, j)] = (signed char)__float2int_rn(v[j]);
    }
  }
  if (team.warp == 0 && team.lane == 0) *scale = rs.scale;
}

}  // namespace souffle
