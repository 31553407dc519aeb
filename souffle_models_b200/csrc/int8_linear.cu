// Products in 8-bit integers with a scale per token and one per channel:
//   out[m][n] = act(sum_k q[m][k] w[n][k] * x_scale[m] * w_scale[n] + bias[n]),
// the sum exact in 32-bit integers, the rest in fp32, rounded once; and the rows' quantisation (row_io.cuh has its definition).
#include <string.h>

#include "host_common.h"
#include "row_io.cuh"
#include "sm100_ptx.cuh"

namespace souffle {

struct LinearArgs {
  int rows, inner, cols, out_dtype, act;
  long long x_stride, w_stride, out_stride;
  const void* x;
  const float* x_scale;
  const signed char* w;
  const float* w_scale;
  const void* bias;
  void* out;
};

// ---- quantised rows ----------------------------------------------------------------------------------------------

// A team of warps per row.  Rows of up to 8 kGroups columns a thread stay in registers between the search for the maximum and the
// rounding; longer ones are read twice, the second time from L2.
template <class T, bool kVec, int kGroups>
__global__ void __launch_bounds__(256) souffle_quantise_rows(const T* __restrict__ x, long long x_stride, int rows, int cols_n, signed char* q,
                                                             long long q_stride, float* scale, int warps_per_row) {
  __shared__ __align__(16) char box[kTeamBox];
  const int teams = blockDim.x / (32 * warps_per_row), warp = threadIdx.x >> 5;
  const int row = blockIdx.x * teams + warp / warps_per_row;
  if (row >= rows) return;
  const T* from = x + row * x_stride;
  signed char* to = q + row * q_stride;
  const Columns<kVec> cols = {(int)(threadIdx.x % (32 * warps_per_row)), 32 * warps_per_row, cols_n};
  Team team;
  team.begin(box, warps_per_row, warp % warps_per_row, 1, cols, 0);
  if (kGroups * 256 * warps_per_row >= cols_n) {
    float v[kGroups][8];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) cols.load(from, i, v[i]);
    quantise_row<kGroups>(team, cols, v, to, scale + row);
    return;
  }
  uint32_t most = 0;
  const int groups = (cols_n + 256 * warps_per_row - 1) / (256 * warps_per_row);
  for (int i = 0; i < groups; ++i) {
    float v[8];
    cols.load(from, i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, abs_bits(v[j]));
  }
  most = team_max_bits(team, most);
  const RowScale rs = row_scale(most);
  const bool fine = most < 0x7f800000u;
  for (int i = 0; i < groups; ++i) {
    float v[8];
    cols.load(from, i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (cols.has(i, j)) to[cols.at(i, j)] = (signed char)__float2int_rn(fine ? v[j] * rs.inv : 0.0f);
  }
  if (threadIdx.x % (32 * warps_per_row) == 0) scale[row] = rs.scale;
}

// ---- epilogue ----------------------------------------------------------------------------------------------------

__device__ __forceinline__ float load_value(const void* p, int dtype, long long i) {
  return dtype == SOUFFLE_F32 ? static_cast<const float*>(p)[i] : dtype == SOUFFLE_F16 ? to_f32(static_cast<const __half*>(p)[i])
                                                                                      : to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_value(void* p, int dtype, long long i, float v) {
  if (dtype == SOUFFLE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == SOUFFLE_F16) static_cast<__half*>(p)[i] = from_f32<__half>(v);
  else static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
}
// tanh-form GELU as v * sigmoid(2u), u = sqrt(2 / pi) (v + 0.044715 v^3): one exponential and one division, exact to a few ulp, so
// that fp32 outputs keep their bits.
__device__ __forceinline__ float gelu_sigmoid(float v) {
  const float u = v * fmaf(v * v, 0.044715f * 0.7978845608028654f, 0.7978845608028654f);
  return __fdividef(v, 1.0f + ex2_fast(-2.885390081777927f * u));
}
__device__ __forceinline__ float activate(float v, int act) {
  if (act == SOUFFLE_ACT_RELU) return v < 0.0f ? 0.0f : v;       // a NaN stays one
  return act == SOUFFLE_ACT_GELU ? gelu_sigmoid(v) : v;
}

// ---- few tokens --------------------------------------------------------------------------------------------------

// 16 bytes of a row from column k on, zeros past `inner`
__device__ __forceinline__ int4 load16(const signed char* row, int k, int inner) {
  if (k + 16 <= inner) return __ldg(reinterpret_cast<const int4*>(row + k));
  int w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 16 && k + i < inner; ++i) w[i >> 2] |= (int)(uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
  return make_int4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void mma_s8(int (&c)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A CTA has 16 channels and 8 kTok tokens; its warps take turns in the inner dimension, 64 columns at a time, and are added
// through shared memory.  Weights and tokens come straight from memory in the operands' own layout, 16 bytes a lane: lane 4 g + t
// holds columns 16 t .. 16 t + 15 of channels g and g + 8 and of token g, which both operands of the product agree on, so the order of
// the columns inside the 64 does not matter to the sum.
constexpr int kFewWarps = 8;
template <int kTok>
__global__ void __launch_bounds__(32 * kFewWarps) souffle_int8_few(const LinearArgs a) {
  __shared__ int part[kFewWarps][kTok][16 * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8 * kTok;
  const signed char* x = static_cast<const signed char*>(a.x);
  int acc[kTok][4];
#pragma unroll
  for (int i = 0; i < kTok; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
  const int4 none = make_int4(0, 0, 0, 0);
  for (int k0 = 64 * warp; k0 < a.inner; k0 += 64 * kFewWarps) {
    const int k = k0 + 16 * t;
    const int4 w0 = n0 + g < a.cols ? load16(a.w + (n0 + g) * a.w_stride, k, a.inner) : none;
    const int4 w1 = n0 + g + 8 < a.cols ? load16(a.w + (n0 + g + 8) * a.w_stride, k, a.inner) : none;
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const int m = m0 + 8 * i + g;
      const int4 b = m < a.rows ? load16(x + m * a.x_stride, k, a.inner) : none;
      mma_s8(acc[i], w0.x, w1.x, w0.y, w1.y, b.x, b.y);
      mma_s8(acc[i], w0.z, w1.z, w0.w, w1.w, b.z, b.w);
    }
  }
#pragma unroll
  for (int i = 0; i < kTok; ++i) {       // [token][channel]
    int* p = part[warp][i];
    p[(2 * t) * 16 + g] = acc[i][0];
    p[(2 * t + 1) * 16 + g] = acc[i][1];
    p[(2 * t) * 16 + g + 8] = acc[i][2];
    p[(2 * t + 1) * 16 + g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 128 * kTok; e += 32 * kFewWarps) {
    const int m = m0 + (e >> 4), n = n0 + (e & 15);
    if (m >= a.rows || n >= a.cols) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) sum += part[w][e >> 7][e & 127];
    float v = (float)sum * a.x_scale[m] * a.w_scale[n];
    if (a.bias) v += load_value(a.bias, a.out_dtype, n);
    store_value(a.out, a.out_dtype, m * a.out_stride + n, activate(v, a.act));
  }
}

// ---- host --------------------------------------------------------------------------------------------------------

static bool is_float_type(int t) { return t >= SOUFFLE_F32 && t <= SOUFFLE_BF16; }
static size_t value_size(int t) { return t == SOUFFLE_F32 ? 4 : 2; }
constexpr int kMaxInner = 131072;

template <class T>
static int quantise_launch(const T* x, long long x_stride, int rows, int cols, signed char* q, long long q_stride, float* scale, cudaStream_t st) {
  const bool vec = cols % 8 == 0 && ((uintptr_t)x & 15u) == 0 && (x_stride * (long long)sizeof(T)) % 16 == 0;
  const int groups8 = (cols + 7) / 8;
  int warps = (groups8 + 127) / 128;
  if (warps > 8) warps = 8;
  const int threads = warps == 1 ? 128 : 32 * warps, teams = threads / (32 * warps), grid = (rows + teams - 1) / teams;
  const int groups = (groups8 + 32 * warps - 1) / (32 * warps);
  auto go = [&](auto fn) { fn<<<grid, threads, 0, st>>>(x, x_stride, rows, cols, q, q_stride, scale, warps); };
  if (vec) groups <= 1 ? go(souffle_quantise_rows<T, true, 1>) : groups == 2 ? go(souffle_quantise_rows<T, true, 2>) : go(souffle_quantise_rows<T, true, 4>);
  else groups <= 1 ? go(souffle_quantise_rows<T, false, 1>) : groups == 2 ? go(souffle_quantise_rows<T, false, 2>) : go(souffle_quantise_rows<T, false, 4>);
  SF_CUDA(cudaGetLastError());
  return SOUFFLE_OK;
}
static int quantise(const void* x, int dtype, long long x_stride, int rows, int cols, signed char* q, long long q_stride, float* scale, cudaStream_t st) {
  if (dtype == SOUFFLE_F32) return quantise_launch(static_cast<const float*>(x), x_stride, rows, cols, q, q_stride, scale, st);
  if (dtype == SOUFFLE_F16) return quantise_launch(static_cast<const __half*>(x), x_stride, rows, cols, q, q_stride, scale, st);
  return quantise_launch(static_cast<const __nv_bfloat16*>(x), x_stride, rows, cols, q, q_stride, scale, st);
}
static long long padded16(long long n) { return (n + 15) / 16 * 16; }

}  // namespace souffle

using namespace souffle;

extern "C" {

int souffle_int8_quantize_rows(const void* x, int32_t dtype, int64_t x_stride, int32_t rows, int32_t cols, void* q, int64_t q_stride, float* scale,
                               souffle_stream_t stream) {
  if (rows < 0 || cols < 1) return fail(SOUFFLE_BAD_SHAPE, "quantised rows of %d x %d: rows >= 0 and cols >= 1 are wanted", rows, cols);
  if (!is_float_type(dtype)) return fail(SOUFFLE_BAD_ARGUMENT, "dtype %d: fp32, fp16 or bf16 rows are quantised", dtype);
  if (x_stride < cols || q_stride < cols || q_stride % 16) return fail(SOUFFLE_BAD_SHAPE, "strides %lld and %lld for %d columns: rows must not overlap, quantised ones begin on 16-byte boundaries", (long long)x_stride, (long long)q_stride, cols);
  if (rows == 0) return SOUFFLE_OK;
  if (!x || (uintptr_t)x % value_size(dtype) || !aligned16(q) || !scale || (uintptr_t)scale % 4) return fail(SOUFFLE_BAD_POINTER, "null or misaligned pointer");
  int sms, rc = current_sms(&sms);
  if (rc) return rc;
  return quantise(x, dtype, x_stride, rows, cols, static_cast<signed char*>(q), q_stride, scale, (cudaStream_t)stream);
}

size_t souffle_int8_linear_workspace_bytes(int32_t rows, int32_t inner, int32_t x_dtype) {
  if (rows < 1 || inner < 1 || x_dtype == SOUFFLE_I8) return 0;
  return (size_t)padded16(4LL * rows) + (size_t)rows * padded16(inner);       // scales, then quantised rows
}

int souffle_int8_linear_forward(const SouffleInt8Linear* call, souffle_stream_t stream) {
  if (!call) return fail(SOUFFLE_BAD_ARGUMENT, "null call record");
  const SouffleInt8Linear& d = *call;
  if (d.rows < 0 || d.cols < 1 || d.inner < 1 || d.inner > kMaxInner)
    return fail(SOUFFLE_BAD_SHAPE, "8-bit product of %d x %d x %d: rows >= 0, cols >= 1 and 1 <= inner <= %d are wanted", d.rows, d.cols, d.inner, kMaxInner);
  if (!(is_float_type(d.x_dtype) || d.x_dtype == SOUFFLE_I8) || !is_float_type(d.out_dtype))
    return fail(SOUFFLE_BAD_ARGUMENT, "x_dtype %d, out_dtype %d: rows are int8, fp32, fp16 or bf16, outputs fp32, fp16 or bf16", d.x_dtype, d.out_dtype);
  if (d.activation < SOUFFLE_ACT_NONE || d.activation > SOUFFLE_ACT_GELU) return fail(SOUFFLE_BAD_ARGUMENT, "activation %d is none of SOUFFLE_ACT_*", d.activation);
  if (d.x_stride < d.inner || d.w_stride < d.inner || d.out_stride < d.cols) return fail(SOUFFLE_BAD_SHAPE, "rows overlap: a stride is below the row's length");
  const bool given = d.x_dtype == SOUFFLE_I8;
  if (d.w_stride % 16 || (given && d.x_stride % 16)) return fail(SOUFFLE_BAD_SHAPE, "quantised rows begin on 16-byte boundaries: strides %lld and %lld", (long long)d.w_stride, (long long)d.x_stride);
  if (given != (d.x_scale != nullptr)) return fail(SOUFFLE_BAD_ARGUMENT, "x_scale comes with int8 rows and only with them");
  if (d.rows == 0) return SOUFFLE_OK;
  const size_t oe = value_size(d.out_dtype);
  if (!d.x || (given ? !aligned16(d.x) : (uintptr_t)d.x % value_size(d.x_dtype) != 0) || (uintptr_t)d.x_scale % 4 || !aligned16(d.w) || !d.w_scale ||
      (uintptr_t)d.w_scale % 4 || (uintptr_t)d.bias % oe || !d.out || (uintptr_t)d.out % oe)
    return fail(SOUFFLE_BAD_POINTER, "null or misaligned pointer");
  const size_t need = souffle_int8_linear_workspace_bytes(d.rows, d.inner, d.x_dtype);
  if (need && (!aligned16(d.workspace) || d.workspace_bytes < need)) return fail(SOUFFLE_BAD_POINTER, "workspace is null, misaligned or smaller than souffle_int8_linear_workspace_bytes()");
  int sms, rc = current_sms(&sms);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  LinearArgs a;
  a.rows = d.rows; a.inner = d.inner; a.cols = d.cols; a.out_dtype = d.out_dtype; a.act = d.activation;
  a.x_stride = d.x_stride; a.w_stride = d.w_stride; a.out_stride = d.out_stride;
  a.x = d.x; a.x_scale = d.x_scale; a.w = static_cast<const signed char*>(d.w); a.w_scale = d.w_scale; a.bias = d.bias; a.out = d.out;
  if (!given) {
    float* scale = static_cast<float*>(d.workspace);
    signed char* q = static_cast<signed char*>(d.workspace) + padded16(4LL * d.rows);
    if ((rc = quantise(d.x, d.x_dtype, d.x_stride, d.rows, d.inner, q, padded16(d.inner), scale, st))) return rc;
    a.x = q; a.x_scale = scale; a.x_stride = padded16(d.inner);
  }
  const int ny = (d.rows + 15) / 16;
  for (int y0 = 0; y0 < ny; y0 += 65535) {                 // a grid has at most 65535 rows of blocks
    LinearArgs b = a;
    b.x = static_cast<const signed char*>(a.x) + 16LL * y0 * a.x_stride;
    b.x_scale = a.x_scale + 16LL * y0;
    b.out = static_cast<char*>(a.out) + 16LL * y0 * a.out_stride * (long long)oe;
    b.rows = a.rows - 16 * y0;
    const int n = ny - y0 < 65535 ? ny - y0 : 65535;
    souffle_int8_few<2><<<dim3((d.cols + 15) / 16, n), 32 * kFewWarps, 0, st>>>(b);
    SF_CUDA(cudaGetLastError());
  }
  return SOUFFLE_OK;
}

}  // extern "C"
