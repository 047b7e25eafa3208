// The steps around the 8-bit dense GEMMs, each one pass over its rows:
//
//   rms_norm_quant: s = x (+ residual); residual_out = round16(s);
//                   y = s * rstd * w, rstd = 1 / sqrt(mean(s^2) + eps); y -> 8 bits
//   act_mul_quant:  y = act(gate) * up of rows [gate | up]; y -> 8 bits
//
// with the two forms of 8 bits that the GEMMs read: e4m3 with one fp32 scale per
// (row, 128 columns) - strix_w8a8_fp8_gemm - and int8 with one per row -
// strix_w8a8_int8_gemm. In the reference these are separate passes of vLLM and of
// the GEMMs themselves (csrc/gemm/w8a8_wmma_gemm.hip:508-529 quantises inside the
// product); sums and statistics are fp32, the 8-bit values are rounded once, from
// the fp32 y.
//
// Bound: HBM. Bytes per element: norm 2 + 2 read, 2 + 1 written (residual form);
// act 4 read, 1 written. A row stays in registers between its statistics and its
// rounding, so it is read once.
#include "cluster.cuh"
#include "quant8.cuh"

namespace strix {
namespace {

using namespace quant8;

constexpr int kMaxRowThreads = 1024;

// Sum over the CTA, the same value in every thread. `scratch` holds 32 floats and is
// free again after the next __syncthreads().
__device__ __forceinline__ float block_sum(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = int(threadIdx.x & 31) < warps ? scratch[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float block_max(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = int(threadIdx.x & 31) < warps ? scratch[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 16 lanes hold a group of 128 values, eight each.
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o, 16));
  return v;
}

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
  float m = fabsf(y[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(y[i]));
  return m;
}

struct NormArgs {
  const uint16_t *x, *residual;   // residual NULL: none
  uint16_t* residual_out;         // NULL: not stored; may be x or residual
  const void* w;                  // 16-bit as x, or fp32
  uint8_t* q;
  float* scales;
  int64_t x_st, r_st, ro_st, q_st, s_st;
  int k8;                         // vectors of eight per row
  float inv_k, eps;
};

// One CTA per row; thread t holds vectors t, t + T, ... (V of them) of the row. T is a
// multiple of 32, so 16 consecutive lanes always hold one group of 128.
template <bool F8, bool F16, bool WF32, int V>
__global__ void __launch_bounds__(kMaxRowThreads) rms_norm_quant_kernel(const NormArgs p) {
  pdl_enter();
  __shared__ float s_sum[32], s_max[32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, T = blockDim.x;
  float v[V][8];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * T + tid;
    if (c >= p.k8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      continue;
    }
    unpack8<F16>(*reinterpret_cast<const uint4*>(p.x + row * p.x_st + c * 8), v[i]);
    if (p.residual != nullptr) {
      float r[8];
      unpack8<F16>(*reinterpret_cast<const uint4*>(p.residual + row * p.r_st + c * 8), r);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += r[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[i][j] * v[i][j];
  }
  if (p.residual_out != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * T + tid;
      if (c >= p.k8) continue;
      uint4 o;
      if constexpr (F16)
        o = make_uint4(pack_f16x2(v[i][0], v[i][1]), pack_f16x2(v[i][2], v[i][3]),
                       pack_f16x2(v[i][4], v[i][5]), pack_f16x2(v[i][6], v[i][7]));
      else
        o = make_uint4(pack_bf16x2(v[i][0], v[i][1]), pack_bf16x2(v[i][2], v[i][3]),
                       pack_bf16x2(v[i][4], v[i][5]), pack_bf16x2(v[i][6], v[i][7]));
      *reinterpret_cast<uint4*>(p.residual_out + row * p.ro_st + c * 8) = o;
    }
  }
  const float rstd = __frsqrt_rn(__fadd_rn(block_sum(sum, s_sum) * p.inv_k, p.eps));
  float row_max = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * T + tid;
    float w[8];
    if (c >= p.k8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = 0.f;
    } else if constexpr (WF32) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p.w) + c * 2);
      const float4 b = __ldg(reinterpret_cast<const float4*>(p.w) + c * 2 + 1);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else {
      unpack8<F16>(__ldg(reinterpret_cast<const uint4*>(p.w) + c), w);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = c < p.k8 ? v[i][j] * rstd * w[j] : 0.f;
    if constexpr (!F8) row_max = max_nan(row_max, abs_max8(v[i]));
  }
  if constexpr (F8) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * T + tid;
      const float s = scale_of(group_max(abs_max8(v[i])), kTopF8);
      if (c >= p.k8) continue;
      *reinterpret_cast<uint2*>(p.q + row * p.q_st + c * 8) = pack8<true>(v[i], __fdiv_rn(1.f, s));
      if ((c & 15) == 0) p.scales[row * p.s_st + (c >> 4)] = s;
    }
  } else {
    const float s = scale_of(block_max(row_max, s_max), kTopI8);
    const float inv = __fdiv_rn(1.f, s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * T + tid;
      if (c < p.k8) *reinterpret_cast<uint2*>(p.q + row * p.q_st + c * 8) = pack8<false>(v[i], inv);
    }
    if (tid == 0) p.scales[row * p.s_st] = s;
  }
}

struct ActArgs {
  const void* x;       // [rows, 2 k]: gate columns, then up columns
  uint8_t* q;
  float* scales;
  int64_t x_st, q_st, s_st, rows;
  int k8, act;
};

// IN: 0 bf16, 1 fp16, 2 fp32
template <int IN>
__device__ __forceinline__ void load8(const void* base, int64_t elem, float (&v)[8]) {
  if constexpr (IN == 2) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elem);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    unpack8<IN == 1>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem), v);
  }
}

template <int IN>
__device__ __forceinline__ void gated8(const ActArgs& p, int64_t row, int c, float (&y)[8]) {
  float u[8];
  load8<IN>(p.x, row * p.x_st + c * 8, y);
  load8<IN>(p.x, row * p.x_st + (p.k8 + c) * 8, u);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = gate(y[j], p.act) * u[j];
}

// e4m3, a scale per 128 columns: a team of 16 lanes per (row, group), no exchange
// beyond the team.
template <int IN>
__global__ void __launch_bounds__(256) act_mul_quant_fp8_kernel(const ActArgs p) {
  pdl_enter();
  const int groups = (p.k8 + 15) >> 4, sub = threadIdx.x & 15;
  const int64_t team = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 4;
  const bool live = team < p.rows * groups;
  const int64_t row = live ? team / groups : 0;
  const int g = live ? int(team - row * groups) : 0, c = g * 16 + sub;
  const bool have = live && c < p.k8;
  float y[8] = {};
  if (have) gated8<IN>(p, row, c, y);
  const float s = scale_of(group_max(abs_max8(y)), kTopF8);
  if (!have) return;
  *reinterpret_cast<uint2*>(p.q + row * p.q_st + c * 8) = pack8<true>(y, __fdiv_rn(1.f, s));
  if (sub == 0) p.scales[row * p.s_st + g] = s;
}

// int8, a scale per row: one CTA per row, the row in registers as in the norm.
template <int IN, int V>
__global__ void __launch_bounds__(kMaxRowThreads) act_mul_quant_token_kernel(const ActArgs p) {
  pdl_enter();
  __shared__ float s_max[32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, T = blockDim.x;
  float y[V][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * T + tid;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] = 0.f;
    if (c < p.k8) gated8<IN>(p, row, c, y[i]);
    m = max_nan(m, abs_max8(y[i]));
  }
  const float s = scale_of(block_max(m, s_max), kTopI8);
  const float inv = __fdiv_rn(1.f, s);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * T + tid;
    if (c < p.k8) *reinterpret_cast<uint2*>(p.q + row * p.q_st + c * 8) = pack8<false>(y[i], inv);
  }
  if (tid == 0) p.scales[row * p.s_st] = s;
}

// Threads and vectors per thread of a row kernel: the fewest vectors that hold the
// row in at most 1,024 threads.
struct RowShape {
  int threads, v;
};
RowShape row_shape(int64_t k8) {
  int v = 1;
  while (v < 8 && k8 > int64_t(v) * kMaxRowThreads) v *= 2;
  return {int((k8 + v * 32 - 1) / (v * 32)) * 32, v};
}

constexpr int64_t kMaxRowK = 8 * 8 * kMaxRowThreads;

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Whether [a, a + a_bytes) and [b, b + b_bytes) share a byte.
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + uintptr_t(b_bytes) && y < x + uintptr_t(a_bytes);
}

template <bool F8, bool F16, bool WF32>
int launch_norm(const NormArgs& p, int64_t rows, cudaStream_t st) {
  const RowShape s = row_shape(p.k8);
  const unsigned grid = unsigned(rows);
  if (s.v == 1) launch_chain(rms_norm_quant_kernel<F8, F16, WF32, 1>, grid, s.threads, 0, st, p);
  else if (s.v == 2) launch_chain(rms_norm_quant_kernel<F8, F16, WF32, 2>, grid, s.threads, 0, st, p);
  else if (s.v == 4) launch_chain(rms_norm_quant_kernel<F8, F16, WF32, 4>, grid, s.threads, 0, st, p);
  else launch_chain(rms_norm_quant_kernel<F8, F16, WF32, 8>, grid, s.threads, 0, st, p);
  return launch_status("rms_norm_quant");
}

template <int IN>
int launch_act(const ActArgs& p, bool fp8, cudaStream_t st) {
  if (fp8) {
    const int64_t teams = p.rows * ((p.k8 + 15) / 16);
    launch_chain(act_mul_quant_fp8_kernel<IN>, unsigned((teams + 15) / 16), 256, 0, st, p);
  } else {
    const RowShape s = row_shape(p.k8);
    const unsigned grid = unsigned(p.rows);
    if (s.v == 1) launch_chain(act_mul_quant_token_kernel<IN, 1>, grid, s.threads, 0, st, p);
    else if (s.v == 2) launch_chain(act_mul_quant_token_kernel<IN, 2>, grid, s.threads, 0, st, p);
    else if (s.v == 4) launch_chain(act_mul_quant_token_kernel<IN, 4>, grid, s.threads, 0, st, p);
    else launch_chain(act_mul_quant_token_kernel<IN, 8>, grid, s.threads, 0, st, p);
  }
  return launch_status("act_mul_quant");
}

}  // namespace
}  // namespace strix

using namespace strix;

extern "C" int strix_rms_norm_quant(const void* x, const void* residual, void* residual_out,
                                    const void* weight, void* q, float* scales, int64_t rows, int64_t k,
                                    int64_t x_stride, int64_t r_stride, int64_t ro_stride,
                                    int64_t q_stride, int64_t s_stride, float eps, int in_f16,
                                    int weight_f32, int fp8, strix_stream_t stream) {
  STRIX_CHECK(rows >= 0 && k > 0, "bad shapes");
  STRIX_CHECK(k % (fp8 ? 16 : 8) == 0 && k <= kMaxRowK,
              "K must be a multiple of %d, at most %d", fp8 ? 16 : 8, int(kMaxRowK));
  if (rows == 0) return STRIX_OK;
  STRIX_CHECK(rows < (int64_t(1) << 31), "too many rows");
  STRIX_CHECK(x != nullptr && weight != nullptr && q != nullptr && scales != nullptr, "pointers must not be NULL");
  STRIX_CHECK(residual_out == nullptr || residual != nullptr, "residual_out needs a residual");
  STRIX_CHECK(aligned(x, 16) && aligned(residual, 16) && aligned(residual_out, 16) && aligned(weight, 16) &&
                  aligned(q, 8) && x_stride % 8 == 0 && r_stride % 8 == 0 && ro_stride % 8 == 0 &&
                  q_stride % 8 == 0,
              "16-byte aligned rows required");
  STRIX_CHECK(x_stride >= 0 && r_stride >= 0 && q_stride >= (rows > 1 ? k : 0) &&
                  s_stride >= (rows > 1 ? (fp8 ? (k + 127) / 128 : 1) : 0) &&
                  (residual_out == nullptr || rows == 1 || ro_stride >= k),
              "output rows must not overlap");
  if (residual_out != nullptr) {
    // a row is read whole before any of it is written, so the sum may replace x or the
    // residual in place; any other overlap would let one row's sum into another's input
    const int64_t out_bytes = ((rows - 1) * ro_stride + k) * 2;
    STRIX_CHECK((residual_out == x && ro_stride == x_stride) ||
                    !overlap(residual_out, out_bytes, x, ((rows - 1) * x_stride + k) * 2),
                "residual_out must be x itself or apart from it");
    STRIX_CHECK((residual_out == residual && ro_stride == r_stride) ||
                    !overlap(residual_out, out_bytes, residual, ((rows - 1) * r_stride + k) * 2),
                "residual_out must be residual itself or apart from it");
  }
  NormArgs p;
  p.x = static_cast<const uint16_t*>(x), p.residual = static_cast<const uint16_t*>(residual);
  p.residual_out = static_cast<uint16_t*>(residual_out), p.w = weight;
  p.q = static_cast<uint8_t*>(q), p.scales = scales;
  p.x_st = x_stride, p.r_st = r_stride, p.ro_st = ro_stride, p.q_st = q_stride, p.s_st = s_stride;
  p.k8 = int(k / 8), p.inv_k = float(1.0 / double(k)), p.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp8) {
    if (in_f16) return weight_f32 ? launch_norm<true, true, true>(p, rows, st) : launch_norm<true, true, false>(p, rows, st);
    return weight_f32 ? launch_norm<true, false, true>(p, rows, st) : launch_norm<true, false, false>(p, rows, st);
  }
  if (in_f16) return weight_f32 ? launch_norm<false, true, true>(p, rows, st) : launch_norm<false, true, false>(p, rows, st);
  return weight_f32 ? launch_norm<false, false, true>(p, rows, st) : launch_norm<false, false, false>(p, rows, st);
}

extern "C" int strix_act_mul_quant(const void* x, void* q, float* scales, int64_t rows, int64_t k,
                                   int64_t x_stride, int64_t q_stride, int64_t s_stride, int gate_act,
                                   int in_type, int fp8, strix_stream_t stream) {
  STRIX_CHECK(gate_act == 1 || gate_act == 2, "activation must be silu or gelu_tanh");
  STRIX_CHECK(in_type >= 0 && in_type <= 2, "x must be bf16, fp16 or fp32");
  STRIX_CHECK(rows >= 0 && k > 0, "bad shapes");
  STRIX_CHECK(k % (fp8 ? 16 : 8) == 0 && (fp8 ? k < (int64_t(1) << 30) : k <= kMaxRowK),
              "K must be a multiple of %d%s", fp8 ? 16 : 8, fp8 ? "" : ", at most 65536");
  if (rows == 0) return STRIX_OK;
  STRIX_CHECK(rows < (int64_t(1) << 31) && rows * ((k + 127) / 128) < (int64_t(1) << 34), "too many rows");
  STRIX_CHECK(x != nullptr && q != nullptr && scales != nullptr, "pointers must not be NULL");
  STRIX_CHECK(aligned(x, 16) && aligned(q, 8) && x_stride % (in_type == 2 ? 4 : 8) == 0 && q_stride % 8 == 0,
              "16-byte aligned rows required");
  STRIX_CHECK(x_stride >= 0 && q_stride >= (rows > 1 ? k : 0) &&
                  s_stride >= (rows > 1 ? (fp8 ? (k + 127) / 128 : 1) : 0),
              "output rows must not overlap");
  ActArgs p;
  p.x = x, p.q = static_cast<uint8_t*>(q), p.scales = scales;
  p.x_st = x_stride, p.q_st = q_stride, p.s_st = s_stride, p.rows = rows;
  p.k8 = int(k / 8), p.act = gate_act;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (in_type == 0) return launch_act<0>(p, fp8 != 0, st);
  if (in_type == 1) return launch_act<1>(p, fp8 != 0, st);
  return launch_act<2>(p, fp8 != 0, st);
}
