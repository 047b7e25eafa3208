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
#include "quant8.cuh"

namespace strix {
namespace {

using namespace quant8;

constexpr int kMaxRowThreads = 1024;

// Sum over the CTA, the same value in every thread. `scratch` holds 32 floats; it may be
// written again after the next __syncthreads() of the CTA.
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

struct NormArgs {
  const uint16_t *x, *residual;   // residual NULL: none
  uint16_t* residual_out;         // NULL: not stored; may be x or residual
  const void* w;                  // 16-bit as x, or fp32
  uint8_t* q;
  float* scales;
  int64_t x_st, r_st, ro_st, q_st, s_st, rows;
  int k8;                         // vectors of eight per row
  float inv_k, eps;
};

// A CTA walks rows blockIdx.x, + gridDim.x, ...; thread t holds vectors t, t + T, ... (V
// of them) of a row. T is a multiple of 32, so 16 consecutive lanes always hold one
// group of 128. The next row's loads are issued as soon as this one's values are in
// fp32 registers, and stay in flight through its reductions; the weights stay in
// registers (as 16-bit pairs) for all rows. The sum may replace x or the residual in
// place: no row is read by two CTAs, and a row is read before any of it is written.
// Measured (bf16, residual): 4,096 x 5,120 23.5 us, 8,192 x 5,120 47 us = 6.2 TB/s (a CTA per row
// without the row ahead: 34 and 63 us); one row of 5,120 2.3 us, a launch and its latency.
// Two vectors per thread need 64 registers; four (rows beyond 16,384 columns) have none left
// for the row ahead: 2,000 x 32,768 82 us = 5.6 TB/s. Eight (beyond 32,768 columns) do not fit
// 64 registers at all and spill about 500 bytes per thread: 2,000 x 32,784 157 us = 2.9 TB/s,
// 1,000 x 65,536 140 us = 3.3.
template <bool F8, bool F16, bool WF32, int V>
__global__ void __launch_bounds__(kMaxRowThreads) rms_norm_quant_kernel(const NormArgs p) {
  pdl_enter();
  __shared__ float s_sum[2][32], s_max[2][32];
  constexpr bool kAhead = V <= 2;   // rows beyond 16,384 columns have no registers to spare for it
  const int tid = threadIdx.x, T = blockDim.x;
  uint4 xr[V], rr[V], wr[V];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * T + tid;
      xr[i] = rr[i] = make_uint4(0u, 0u, 0u, 0u);
      if (c >= p.k8) continue;
      xr[i] = *reinterpret_cast<const uint4*>(p.x + row * p.x_st + c * 8);
      if (p.residual != nullptr) rr[i] = *reinterpret_cast<const uint4*>(p.residual + row * p.r_st + c * 8);
    }
  };
  auto weights = [&](int c) {
    return c < p.k8 ? __ldg(reinterpret_cast<const uint4*>(p.w) + c) : make_uint4(0u, 0u, 0u, 0u);
  };
  if constexpr (kAhead) fetch(blockIdx.x);
  if constexpr (!WF32 && kAhead) {
#pragma unroll
    for (int i = 0; i < V; ++i) wr[i] = weights(i * T + tid);
  }
  int par = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, par ^= 1) {
    float v[V][8];
    float sum = 0.f;
    if constexpr (!kAhead) fetch(row);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      unpack8<F16>(xr[i], v[i]);
      if (p.residual != nullptr) {
        float r[8];
        unpack8<F16>(rr[i], r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += r[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[i][j] * v[i][j];
    }
    if (kAhead && row + gridDim.x < p.rows) fetch(row + gridDim.x);
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
    const float rstd = __frsqrt_rn(__fadd_rn(block_sum(sum, s_sum[par]) * p.inv_k, p.eps));
    float row_max = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = i * T + tid;
      float w[8];
      if constexpr (WF32) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        if (c < p.k8) {
          a = __ldg(reinterpret_cast<const float4*>(p.w) + c * 2);
          b = __ldg(reinterpret_cast<const float4*>(p.w) + c * 2 + 1);
        }
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
      } else {
        unpack8<F16>(kAhead ? wr[i] : weights(c), w);
      }
      // past the row's end: zeros, whatever rstd is (0 * inf would be a NaN)
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
        *reinterpret_cast<uint2*>(p.q + row * p.q_st + c * 8) = pack8<true>(v[i], rcp(s));
        if ((c & 15) == 0) p.scales[row * p.s_st + (c >> 4)] = s;
      }
    } else {
      const float s = scale_of(block_max(row_max, s_max[par]), kTopI8);
      const float inv = rcp(s);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = i * T + tid;
        if (c < p.k8) *reinterpret_cast<uint2*>(p.q + row * p.q_st + c * 8) = pack8<false>(v[i], inv);
      }
      if (tid == 0) p.scales[row * p.s_st] = s;
    }
  }
}

struct ActArgs {
  const void* x;       // [rows, 2 k]: gate columns, then up columns
  uint8_t* q;
  float* scales;
  int64_t x_st, q_st, s_st, rows;
  int k8;
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

// y[u] = act(gate) * up of vector c[u] of row[u], for the U vectors with c[u] < k8; all
// loads are issued before the first is used.
template <int IN, bool GELU, int U>
__device__ __forceinline__ void gated8(const ActArgs& p, const int64_t (&row)[U], const int (&c)[U],
                                       float (&y)[U][8]) {
  if constexpr (IN == 2) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c[u] >= p.k8) continue;
      float up[8];
      load8<IN>(p.x, row[u] * p.x_st + c[u] * 8, y[u]);
      load8<IN>(p.x, row[u] * p.x_st + (p.k8 + c[u]) * 8, up);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[u][j] = gate<GELU>(y[u][j]) * up[j];
    }
  } else {
    uint4 g[U], h[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      g[u] = h[u] = make_uint4(0u, 0u, 0u, 0u);
      if (c[u] >= p.k8) continue;
      const uint16_t* x = static_cast<const uint16_t*>(p.x) + row[u] * p.x_st;
      g[u] = ldg_stream(x + c[u] * 8), h[u] = ldg_stream(x + (p.k8 + c[u]) * 8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float up[8];
      unpack8<IN == 1>(g[u], y[u]), unpack8<IN == 1>(h[u], up);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[u][j] = gate<GELU>(y[u][j]) * up[j];
    }
  }
}

// e4m3, a scale per 128 columns: a team of 16 lanes per (row, group), no exchange
// beyond the team. A team takes U groups, their loads first. Measured: 4,096 x 17,408
// bf16 60 us = 6.0 TB/s, at four fifths of the issue slots (27 instructions per output, of
// which an exponential, a reciprocal and half a conversion go to the slow units).
template <int IN, bool GELU, int U>
__global__ void __launch_bounds__(256) act_mul_quant_fp8_kernel(const ActArgs p) {
  pdl_enter();
  const int groups = (p.k8 + 15) >> 4, sub = threadIdx.x & 15;
  // 32 bits: the host refuses 2^31 groups, and a 64-bit division per team was a third of
  // the kernel's instructions
  const uint32_t total = uint32_t(p.rows) * uint32_t(groups);
  const uint32_t team0 = blockIdx.x * uint32_t(16 * U) + (threadIdx.x >> 4);
  float y[U][8];
  int64_t row[U];
  int c[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t team = team0 + u * 16, r = team / uint32_t(groups);
    row[u] = team < total ? r : 0;
    c[u] = team < total ? int(team - r * groups) * 16 + sub : p.k8;   // k8: nothing to do
#pragma unroll
    for (int j = 0; j < 8; ++j) y[u][j] = 0.f;
  }
  gated8<IN, GELU, U>(p, row, c, y);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float s = scale_of(group_max(abs_max8(y[u])), kTopF8);
    if (c[u] >= p.k8) continue;
    *reinterpret_cast<uint2*>(p.q + row[u] * p.q_st + c[u] * 8) = pack8<true>(y[u], rcp(s));
    if (sub == 0) p.scales[row[u] * p.s_st + (c[u] >> 4)] = s;
  }
}

// int8, a scale per row: one CTA per row, the row in registers as in the norm. Measured:
// 8,192 x 2,560 bf16 18 us = 5.8 TB/s; 16 x 17,408 5.5 us (16 CTAs, their latency).
template <int IN, bool GELU, int V>
__global__ void __launch_bounds__(kMaxRowThreads) act_mul_quant_token_kernel(const ActArgs p) {
  pdl_enter();
  __shared__ float s_max[32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, T = blockDim.x;
  float y[V][8];
  int64_t rows[V];
  int c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    rows[i] = row, c[i] = i * T + tid;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] = 0.f;
  }
  gated8<IN, GELU, V>(p, rows, c, y);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) m = max_nan(m, abs_max8(y[i]));
  const float s = scale_of(block_max(m, s_max), kTopI8);
  const float inv = rcp(s);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (c[i] < p.k8) *reinterpret_cast<uint2*>(p.q + row * p.q_st + c[i] * 8) = pack8<false>(y[i], inv);
  if (tid == 0) p.scales[row * p.s_st] = s;
}

// Threads and vectors per thread of a row kernel: the fewest vectors, and at least
// v_min, that hold the row in at most 1,024 threads.
struct RowShape {
  int threads, v;
};
RowShape row_shape(int64_t k8, int v_min) {
  int v = v_min;
  while (v < 8 && k8 > int64_t(v) * kMaxRowThreads) v *= 2;
  return {int((k8 + v * 32 - 1) / (v * 32)) * 32, v};
}

constexpr int64_t kMaxRowK = 8 * 8 * kMaxRowThreads;

// The current device and its multiprocessors (asked once per device).
int device_sms(int& dev, int& sms) {
  static int count[64] = {};
  STRIX_CUDA(cudaGetDevice(&dev));
  STRIX_CHECK(dev >= 0 && dev < 64, "device index %d out of range", dev);
  sms = count[dev];
  if (sms == 0) {
    STRIX_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    count[dev] = sms;
  }
  return STRIX_OK;
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Whether two matrices of `rows` rows of `width` bytes, the row strides in bytes, may share
// a byte. Rows side by side in one wider matrix (slices of its columns) do not.
bool overlap(const void* a, int64_t a_st, const void* b, int64_t b_st, int64_t rows, int64_t width) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const uintptr_t a_end = x + uintptr_t((rows - 1) * a_st + width), b_end = y + uintptr_t((rows - 1) * b_st + width);
  if (x >= b_end || y >= a_end) return false;
  if (a_st != b_st || a_st < 2 * width) return true;
  const int64_t apart = int64_t((x > y ? x - y : y - x) % uintptr_t(a_st));
  return apart < width || apart > a_st - width;
}

template <bool F8, bool F16, bool WF32, int V>
int launch_norm_v(const NormArgs& p, int threads, int sms, int dev, cudaStream_t st) {
  auto kernel = rms_norm_quant_kernel<F8, F16, WF32, V>;
  // CTAs of this size that an SM holds at once (asked once per device and size)
  static int resident[64][kMaxRowThreads / 32] = {};
  int per_sm = resident[dev][threads / 32 - 1];
  if (per_sm == 0) {
    STRIX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0));
    resident[dev][threads / 32 - 1] = per_sm;
  }
  STRIX_CHECK(per_sm > 0, "rms_norm_quant does not fit the device");
  const int64_t slots = int64_t(sms) * per_sm;
  launch_chain(kernel, unsigned(p.rows < slots ? p.rows : slots), threads, 0, st, p);
  return launch_status("rms_norm_quant");
}

template <bool F8, bool F16, bool WF32>
int launch_norm(const NormArgs& p, cudaStream_t st) {
  int dev = 0, sms = 0;
  const int rc = device_sms(dev, sms);
  if (rc != STRIX_OK) return rc;
  // one vector per thread where there are too few rows to fill the GPU (a row's time
  // counts), two where there are many (bytes in flight count)
  const RowShape s = row_shape(p.k8, p.rows > 2 * sms ? 2 : 1);
  if (s.v == 1) return launch_norm_v<F8, F16, WF32, 1>(p, s.threads, sms, dev, st);
  if (s.v == 2) return launch_norm_v<F8, F16, WF32, 2>(p, s.threads, sms, dev, st);
  if (s.v == 4) return launch_norm_v<F8, F16, WF32, 4>(p, s.threads, sms, dev, st);
  return launch_norm_v<F8, F16, WF32, 8>(p, s.threads, sms, dev, st);
}

template <int IN, bool GELU>
int launch_act(const ActArgs& p, bool fp8, cudaStream_t st) {
  if (fp8) {
    int dev = 0, sms = 0;
    const int rc = device_sms(dev, sms);
    if (rc != STRIX_OK) return rc;
    const int64_t teams = p.rows * ((p.k8 + 15) / 16);
    // two groups per team once that still leaves two CTAs per SM
    if (teams > int64_t(sms) * 64)
      launch_chain(act_mul_quant_fp8_kernel<IN, GELU, 2>, unsigned((teams + 31) / 32), 256, 0, st, p);
    else
      launch_chain(act_mul_quant_fp8_kernel<IN, GELU, 1>, unsigned((teams + 15) / 16), 256, 0, st, p);
  } else {
    const RowShape s = row_shape(p.k8, 1);
    const unsigned grid = unsigned(p.rows);
    if (s.v == 1) launch_chain(act_mul_quant_token_kernel<IN, GELU, 1>, grid, s.threads, 0, st, p);
    else if (s.v == 2) launch_chain(act_mul_quant_token_kernel<IN, GELU, 2>, grid, s.threads, 0, st, p);
    else if (s.v == 4) launch_chain(act_mul_quant_token_kernel<IN, GELU, 4>, grid, s.threads, 0, st, p);
    else launch_chain(act_mul_quant_token_kernel<IN, GELU, 8>, grid, s.threads, 0, st, p);
  }
  return launch_status("act_mul_quant");
}

template <int IN>
int launch_act(const ActArgs& p, int act, bool fp8, cudaStream_t st) {
  return act == 1 ? launch_act<IN, false>(p, fp8, st) : launch_act<IN, true>(p, fp8, st);
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
  // a single row's strides are not read: any will do
  if (rows == 1) x_stride = r_stride = ro_stride = q_stride = k, s_stride = (k + 127) / 128;
  STRIX_CHECK(aligned(x, 16) && aligned(residual, 16) && aligned(residual_out, 16) && aligned(weight, 16) &&
                  aligned(q, 8) && x_stride % 8 == 0 && r_stride % 8 == 0 && ro_stride % 8 == 0 &&
                  q_stride % 8 == 0,
              "16-byte aligned rows required");
  STRIX_CHECK(x_stride >= 0 && r_stride >= 0 && q_stride >= k && s_stride >= (fp8 ? (k + 127) / 128 : 1) &&
                  (residual_out == nullptr || ro_stride >= k),
              "output rows must not overlap");
  if (residual_out != nullptr) {
    // a row is read whole before any of it is written, so the sum may replace x or the
    // residual in place; any other overlap would let one row's sum into another's input
    STRIX_CHECK((residual_out == x && ro_stride == x_stride) ||
                    !overlap(residual_out, ro_stride * 2, x, x_stride * 2, rows, k * 2),
                "residual_out must be x itself or apart from it");
    STRIX_CHECK((residual_out == residual && ro_stride == r_stride) ||
                    !overlap(residual_out, ro_stride * 2, residual, r_stride * 2, rows, k * 2),
                "residual_out must be residual itself or apart from it");
  }
  NormArgs p;
  p.x = static_cast<const uint16_t*>(x), p.residual = static_cast<const uint16_t*>(residual);
  p.residual_out = static_cast<uint16_t*>(residual_out), p.w = weight;
  p.q = static_cast<uint8_t*>(q), p.scales = scales;
  p.x_st = x_stride, p.r_st = r_stride, p.ro_st = ro_stride, p.q_st = q_stride, p.s_st = s_stride;
  p.rows = rows, p.k8 = int(k / 8), p.inv_k = float(1.0 / double(k)), p.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (fp8) {
    if (in_f16) return weight_f32 ? launch_norm<true, true, true>(p, st) : launch_norm<true, true, false>(p, st);
    return weight_f32 ? launch_norm<true, false, true>(p, st) : launch_norm<true, false, false>(p, st);
  }
  if (in_f16) return weight_f32 ? launch_norm<false, true, true>(p, st) : launch_norm<false, true, false>(p, st);
  return weight_f32 ? launch_norm<false, false, true>(p, st) : launch_norm<false, false, false>(p, st);
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
  STRIX_CHECK(rows < (int64_t(1) << 31) && rows * ((k + 127) / 128) < (int64_t(1) << 31) - 64, "too many rows");
  STRIX_CHECK(x != nullptr && q != nullptr && scales != nullptr, "pointers must not be NULL");
  // a single row's strides are not read: any will do
  if (rows == 1) x_stride = 2 * k, q_stride = k, s_stride = (k + 127) / 128;
  STRIX_CHECK(aligned(x, 16) && aligned(q, 8) && x_stride % (in_type == 2 ? 4 : 8) == 0 && q_stride % 8 == 0,
              "16-byte aligned rows required");
  STRIX_CHECK(x_stride >= 0 && q_stride >= k && s_stride >= (fp8 ? (k + 127) / 128 : 1),
              "output rows must not overlap");
  ActArgs p;
  p.x = x, p.q = static_cast<uint8_t*>(q), p.scales = scales;
  p.x_st = x_stride, p.q_st = q_stride, p.s_st = s_stride, p.rows = rows;
  p.k8 = int(k / 8);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (in_type == 0) return launch_act<0>(p, gate_act, fp8 != 0, st);
  if (in_type == 1) return launch_act<1>(p, gate_act, fp8 != 0, st);
  return launch_act<2>(p, gate_act, fp8 != 0, st);
}
