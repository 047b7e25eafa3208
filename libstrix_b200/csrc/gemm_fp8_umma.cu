// Dense FP8 W8A8 product with a scale per block of 128, on tcgen05 kind::f8f6f4:
//
//   out[m, n] = sum_b sa[m, b] * sw[n / 128, b] * (sum_{k in block b} a[m, k] w[n, k]) (+ bias[n])
//
// a e4m3 [M, K] with one fp32 scale per (row, 128 columns), w e4m3 [N, K] with one
// per 128 x 128 block. The scales are arbitrary fp32 numbers and cannot ride the MMA
// (its block scales are powers of two), so each K block of 128 is one fresh
// accumulation in tensor memory, and the epilogue warps fold it into fp32 registers:
// acc += partial * (sa * sw). The reference has this product with 16-bit activations
// only (csrc/gemm/fp8_wmma_gemm.hip; the schema at csrc/torch_ops.cpp:256).
//
// K that is no multiple of 128: the TMA fills the last block with zero bytes, which
// are zeros of e4m3. Rows past M or N arrive as zeros and are not stored.
#include "cluster.cuh"
#include "quant8.cuh"
#include "tma.cuh"

namespace strix {

int32_t* umma_status_ptr();  // moe_gemm_umma.cu: device address of the shared status word

namespace {

using namespace umma;

constexpr int kBlk = 128;          // K block, bytes and columns alike

enum OutKind : int { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };

struct Fp8GemmArgs {
  void* out;                       // [M, N], row stride out_st
  const float *sa, *sw;
  const void* bias;                // NULL or [N], in the output's type
  int32_t* status;
  int64_t out_st, sa_sm, sa_sk, sw_sn, sw_sk;
  int M, N, nkb;
  int n_tiles, splits;             // wide kernel: tiles of BN weight rows; CTAs, or pairs of them, per tile along K
  // gated form: `out` holds the e4m3 rows, N counts gate and up rows together
  float* q_scales;                 // [M, N / 256], row stride qs_st
  int64_t qs_st;
  int gate_act;
  int out_kind, tma_out;           // tma_out: the wide kernel's rows may leave by TMA
};

__device__ __forceinline__ float load_bias(const void* bias, int kind, int n) {
  if (bias == nullptr) return 0.f;
  if (kind == kOutBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
  if (kind == kOutF16) return __half2float(static_cast<const __half*>(bias)[n]);
  return static_cast<const float*>(bias)[n];
}

__device__ __forceinline__ void store_one(void* out, int kind, int64_t at, float v) {
  if (kind == kOutBf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (kind == kOutF16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else static_cast<float*>(out)[at] = v;
}

__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_32x16(taddr, r); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32(taddr, r); }

// ================================================================ weight stream
// Few tokens: the weights are the MMA's A operand (128 rows fill M whatever the
// batch), NB tokens its N, and the kernel is a stream of the weights. A cluster of
// `splits` CTAs shares one tile of 128 weight rows along K and adds its partial sums
// through distributed shared memory in rank order, so a layer with few tiles still
// fills the GPU, the result does not depend on timing and no scratch is needed.
// Warp 0 loads (TMA), warp 1 issues, warp 2 stages the tokens' scales, warps 4-7
// fold. Two CTAs share an SM, so one's start and join hide behind the other's stream.
//
// GATED: a tile is 128 gate rows and the 128 up rows of the same outputs, two MMAs per
// K step over the same tokens; warps 8-11 fold the up rows. The join leaves a thread with
// both sums of an output, and the 128 threads of a token with one group of the 8-bit
// form. One CTA per SM (its stages are twice as large).
constexpr int kMaxSplits = 8;   // CTAs of a cluster

template <int NB, bool GATED>
struct StreamLayout {
  static constexpr int kTiles = GATED ? 2 : 1;                     // of 128 weight rows
  static constexpr int kCtas = GATED ? 1 : 2;                      // per SM
  static constexpr int kFoldWarps = 4 * kTiles, kThreads = 128 + 32 * kFoldWarps;
  static constexpr int kWBytes = kTiles * 128 * kBlk, kTBytes = NB * kBlk;
  static constexpr int kStageBytes = kWBytes + kTBytes;
  static constexpr int kStages = ((GATED ? 204 : 100) * 1024) / kStageBytes;
  static constexpr int kAcc = 4;                                   // K blocks in tensor memory
  static constexpr int kTmemCols = kAcc * kTiles * NB < 32 ? 32 : kAcc * kTiles * NB;
  static constexpr int kSmem = 1024 + kStages * (kStageBytes + NB * 4);
  static_assert(kStages * kStageBytes >= kTiles * NB * 128 * 4, "the join reuses the ring");
};

template <int NB, bool GATED>
__global__ void __launch_bounds__(StreamLayout<NB, GATED>::kThreads, StreamLayout<NB, GATED>::kCtas) gemm_fp8_stream_kernel(
    const Fp8GemmArgs p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a) {
  pdl_enter();
  using L = StreamLayout<NB, GATED>;
  constexpr int S = L::kStages, NA = L::kAcc, T = L::kTiles;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  float* s_scale = reinterpret_cast<float*>(ring + S * L::kStageBytes);    // [S][NB]
  __shared__ __align__(8) uint64_t full_bar[S], done_bar[S], sfull_bar[S], sempty_bar[S], tempty_bar[NA], drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_abort;

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int rank = int(blockIdx.x) % p.splits, n0 = int(blockIdx.x) / p.splits * 128;
  // K blocks [k0, k0 + nk) of this CTA
  const int base = p.nkb / p.splits, rem = p.nkb % p.splits;
  const int nk = base + (rank < rem ? 1 : 0), k0 = rank * base + min(rank, rem);
  int armed = 0;

  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full_bar[i], 1), mbar_init(&done_bar[i], 1);
      mbar_init(&sfull_bar[i], 32), mbar_init(&sempty_bar[i], L::kFoldWarps);
    }
    for (int i = 0; i < NA; ++i) mbar_init(&tempty_bar[i], L::kFoldWarps);
    mbar_init(&drain_bar, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, L::kTmemCols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0), ring_s = smem_u32(ring);

  float acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = 0.f;

  if (warp == 0) {
    const bool one = elect_one();
    if (one) tma::prefetch_map(&map_w), tma::prefetch_map(&map_a);
    bool ok = true;
    int t = 0, s = 0;
    uint32_t ph = 1;
    for (; t < nk; ++t) {
      ok = mbar_wait_warp(&done_bar[s], ph);
      if (!ok) break;
      if (one) {
        const uint32_t st = ring_s + s * L::kStageBytes;
        tma::mbar_expect_tx(&full_bar[s], L::kStageBytes);
        tma::load_2d(st, &map_w, (k0 + t) * kBlk, n0, &full_bar[s]);
        if constexpr (GATED) tma::load_2d(st + 128 * kBlk, &map_w, (k0 + t) * kBlk, p.N / 2 + n0, &full_bar[s]);
        tma::load_2d(st + L::kWBytes, &map_a, (k0 + t) * kBlk, 0, &full_bar[s]);
      }
      __syncwarp();
      if (++s == S) s = 0, ph ^= 1;
    }
    armed = t;
    if (!ok && lane == 0) atomicExch(p.status, 1), s_abort = 1;
  } else if (warp == 1) {
    constexpr uint32_t idesc = instr_desc(D_F32, 0, 0, 128, NB);
    const uint32_t w_lo0 = smem_desc_lo(ring_s);
    const bool one = elect_one();
    bool ok = true;
    int s = 0, b = 0;
    uint32_t ph = 0, aph = 1;
    for (int t = 0; t < nk; ++t) {
      ok = mbar_wait_warp(&tempty_bar[b], aph) && mbar_wait_warp(&full_bar[s], ph);
      if (!ok) break;
      tc_fence_after_sync();
      if (one) {
        const uint32_t w_lo = w_lo0 + s * (L::kStageBytes >> 4), t_lo = w_lo + (L::kWBytes >> 4);
#pragma unroll
        for (int i = 0; i < T; ++i) {
          const uint32_t d = tmem + (b * T + i) * NB, w_i = w_lo + i * (128 * kBlk >> 4);
          mma_ss_lo<KIND_F8F6F4, false>(d, w_i, t_lo, idesc);
          mma_ss_lo<KIND_F8F6F4, true>(d, w_i + 2, t_lo + 2, idesc);
          mma_ss_lo<KIND_F8F6F4, true>(d, w_i + 4, t_lo + 4, idesc);
          mma_ss_lo<KIND_F8F6F4, true>(d, w_i + 6, t_lo + 6, idesc);
        }
        mma_commit(&done_bar[s]);   // frees the stage and publishes the sums
      }
      __syncwarp();
      if (++s == S) s = 0, ph ^= 1;
      if (++b == NA) b = 0, aph ^= 1;
    }
    if (!ok && lane == 0) atomicExch(p.status, 1), s_abort = 1;
  } else if (warp == 2) {
    // the tokens' scales of one K block per ring position, copied ahead
    bool dead = false;
    int s = 0;
    uint32_t ph = 1;
    for (int t = 0; t < nk; ++t) {
      if (!mbar_wait_warp(&sempty_bar[s], ph)) {
        dead = true;
        break;
      }
      for (int j = lane; j < NB; j += 32) {
        const bool live = j < p.M;
        cp_async_4_zfill(smem_u32(s_scale + s * NB + j),
                         p.sa + (live ? int64_t(j) * p.sa_sm + int64_t(k0 + t) * p.sa_sk : 0), live);
      }
      mbar_arrive_cp_async(&sfull_bar[s]);
      if (++s == S) s = 0, ph ^= 1;
    }
    cp_async_commit();
    cp_async_wait<0>();   // nothing of this warp is in flight when the CTA ends
    if (dead && lane == 0) atomicExch(p.status, 1), s_abort = 1;
  } else if (warp >= 4) {
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    const int part_of = (warp - 4) >> 2;   // GATED: 0 gate rows, 1 up rows
    const float* sw = p.sw + int64_t((part_of * (p.N / 2) + n0) / kBlk) * p.sw_sn + int64_t(k0) * p.sw_sk;
    float w_next = nk > 0 ? __ldg(sw) : 0.f;
    bool dead = false;
    int s = 0, b = 0;
    uint32_t ph = 0;
    for (int t = 0; t < nk; ++t) {
      const float ws = w_next;
      if (t + 1 < nk) w_next = __ldg(sw + int64_t(t + 1) * p.sw_sk);
      if (!mbar_wait_warp(&sfull_bar[s], ph) || !mbar_wait_warp(&done_bar[s], ph)) {
        dead = true;
        break;
      }
      tc_fence_after_sync();
      const float4* sc = reinterpret_cast<const float4*>(s_scale + s * NB);
      // loads of tensor memory CH columns at a time, the next one under way behind the sums;
      // two products per instruction: scale * weight scale, and its multiply-add
      constexpr int CH = NB < 32 ? NB : 32;
      const uint32_t src = tmem + lane_base + (b * T + part_of) * NB;
      const float2 w2 = make_float2(ws, ws);
      uint32_t r[2][CH];
      tmem_ld(src, r[0]);
#pragma unroll
      for (int c = 0; c < NB / CH; ++c) {
        tmem_ld_wait();
        if (c + 1 < NB / CH) tmem_ld(src + (c + 1) * CH, r[(c + 1) & 1]);
#pragma unroll
        for (int j = 0; j < CH; j += 4) {
          const float4 q = sc[(c * CH + j) >> 2];
          const float2 f0 = __fmul2_rn(make_float2(q.x, q.y), w2), f1 = __fmul2_rn(make_float2(q.z, q.w), w2);
          const uint32_t* x = &r[c & 1][j];
          float* a = &acc[c * CH + j];
          const float2 s0 = __ffma2_rn(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), f0, make_float2(a[0], a[1]));
          const float2 s1 = __ffma2_rn(make_float2(__uint_as_float(x[2]), __uint_as_float(x[3])), f1, make_float2(a[2], a[3]));
          a[0] = s0.x, a[1] = s0.y, a[2] = s1.x, a[3] = s1.y;
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[b]), mbar_arrive(&sempty_bar[s]);
      if (++s == S) s = 0, ph ^= 1;
      if (++b == NA) b = 0;
    }
    if (dead) atomicExch(p.status, 1), s_abort = 1;
  }

  tc_fence_before_sync();
  __syncthreads();
  if (s_abort) {   // wait for the copies and MMAs still in flight before TMEM and the ring go
    if (tid == 0) drain_armed_loads(full_bar, S, armed);
    if (warp == 1 && elect_one()) drain_issued_mmas(&drain_bar);
    tc_fence_before_sync();
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc(tmem, L::kTmemCols);

  // thread r of warps 4-7 holds the sums of weight row n0 + r for the NB tokens
  const int row = (warp & 3) * 32 + lane, n = n0 + row;
  if (!GATED && p.splits == 1) {
    if (warp >= 4 && n < p.N) {
      const float bias = load_bias(p.bias, p.out_kind, n);
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (j < p.M) store_one(p.out, p.out_kind, int64_t(j) * p.out_st + n, acc[j] + bias);
    }
    return;
  }
  // the join: every CTA lays its partial tile [token][row] into its ring (whose copies and
  // MMAs have ended), then groups of 128 threads sum tokens over the cluster
  float* part = reinterpret_cast<float*>(ring);
  if (warp >= 4) {
    float* mine = part + (GATED ? (warp - 4) >> 2 : 0) * (NB * 128);
#pragma unroll
    for (int j = 0; j < NB; ++j) mine[j * 128 + row] = acc[j];
  }
  cluster::sync();
  constexpr int G = L::kThreads / 128;
  const int grp = warp >> 2, col = n0 + row;
  const uint32_t own = smem_u32(part) + row * 4;
  auto joined = [&](int at) {   // the sum of float `at` x 128 + row over the cluster, in rank order
    float v[kMaxSplits];   // all reads on their way before the first is added
#pragma unroll
    for (int c = 0; c < kMaxSplits; ++c)
      v[c] = c < p.splits ? cluster::ld_shared_f32(cluster::map_shared(own + at * 512, c)) : 0.f;
#pragma unroll
    for (int c = 1; c < kMaxSplits; ++c) v[0] += v[c];
    return v[0];
  };
  if constexpr (GATED) {
    __shared__ float s_amax[2][G][4];
    int par = 0;
    // all threads take the same rounds: they meet at a barrier in each
    for (int j0 = rank * G; j0 < p.M; j0 += G * p.splits, par ^= 1) {
      const int j = j0 + grp;
      const bool live = j < p.M;
      float y = 0.f;
      if (live) y = quant8::gate(joined(j), p.gate_act) * joined(NB + j);
      float amax = fabsf(y);
#pragma unroll
      for (int o = 16; o; o >>= 1) amax = quant8::max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (lane == 0) s_amax[par][grp][warp & 3] = amax;
      __syncthreads();
      const float* a4 = s_amax[par][grp];
      const float sc = quant8::scale_of(quant8::max_nan(quant8::max_nan(a4[0], a4[1], a4[2]), a4[3]), quant8::kTopF8);
      if (live) {
        static_cast<uint8_t*>(p.out)[int64_t(j) * p.out_st + col] =
            uint8_t(quant8::pack_e4m3x4(y * quant8::rcp(sc), 0.f, 0.f, 0.f));
        if (row == 0) p.q_scales[int64_t(j) * p.qs_st + n0 / kBlk] = sc;
      }
    }
  } else {
    const float bias = col < p.N ? load_bias(p.bias, p.out_kind, col) : 0.f;
    for (int j = rank * G + grp; j < p.M; j += G * p.splits) {
      const float v = joined(j);
      if (col < p.N) store_one(p.out, p.out_kind, int64_t(j) * p.out_st + col, v + bias);
    }
  }
  cluster::sync();   // nobody leaves while a peer still reads its shared memory
}

template <int NB, bool GATED>
int launch_stream(Fp8GemmArgs p, const void* a, int64_t a_st, const void* w, int64_t w_st, int64_t k, int dev,
                  cudaStream_t st) {
  using L = StreamLayout<NB, GATED>;
  STRIX_CHECK(p.M <= NB, "the weight stream takes up to %d tokens here", NB);
  auto kernel = gemm_fp8_stream_kernel<NB, GATED>;
  static int places[64][kMaxSplits + 1] = {};   // clusters of c CTAs that find an SM each (asked once)
  if (!places[dev][1]) {
    STRIX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
    for (int c = kMaxSplits; c >= 1; --c)
      STRIX_CUDA(cluster::places(&places[dev][c], kernel, unsigned(c), unsigned(L::kThreads), L::kSmem));
  }
  const int64_t tiles = GATED ? p.N / 256 : (p.N + 127) / 128;
  // As many CTAs per tile as leave each two K blocks and every cluster a place at once: a
  // second round costs more than shorter CTAs give. Measured on 16 x 5,120 x 17,408 (40
  // tiles; clusters of 6 are the largest that all fit): 36.8, 22.7, 20.0, 19.2, 18.7, 18.8,
  // 25.8 and 23.1 us with 1 to 8; on 272 tiles 29.8 us with one, 32.9 with two.
  int splits = 1;
  for (int c = 2; c <= kMaxSplits; ++c)
    if (tiles <= int64_t(places[dev][c]) * L::kCtas && p.nkb >= 2 * c) splits = c;
  p.splits = splits;
  STRIX_CHECK(tiles * splits < (int64_t(1) << 31), "matrix too large");
  CUtensorMap map_w, map_a;
  STRIX_CHECK(tma::make_map_u8(&map_w, w, uint64_t(p.N), uint64_t(k), uint64_t(w_st), 128) &&
                  tma::make_map_u8(&map_a, a, uint64_t(p.M), uint64_t(k), uint64_t(a_st), NB),
              "tensor map encoding failed");
  STRIX_CUDA(cluster::launch(kernel, unsigned(tiles * splits), unsigned(splits), L::kThreads, L::kSmem, st, p, map_w, map_a));
  return launch_status("w8a8_fp8_gemm");
}

// ================================================================== wide tiles
// Many tokens: the tensor cores set the pace. A pair of CTAs (cta_group::2) owns a tile
// of 256 tokens x BN weight rows: each CTA loads its 128 token rows and BN / 2 of the
// weight rows per K block, half of what two single tiles would read, and folds the
// sums of its own 128 tokens. Persistent, one pair per two SMs, tiles with the tokens
// fastest so that the pairs at work share weight rows in L2.
// Warp 0 loads, warp 1 issues (rank 0 only), warps 4-11 fold: two threads per token
// row, BN / 2 columns each, in registers that setmaxnreg moves to them. A thread's
// columns lie in one weight block, so a K block costs it one scale.
// The fold of 128 x 256 sums is 64 packed multiply-adds per thread and K block, half
// the time of the block's MMAs; two accumulators in tensor memory keep both going, and
// what counts is how soon one is handed back. Measured at 4,096 x 34,816 x 5,120:
// 1.52 ms at first; 0.79 with the hand-back a release of CTA scope (cluster scope waits
// for global loads); 0.66 with the issuing warp kept converged; 0.59 without the abort
// flag and the divisions in the folding loop (2,460 TFLOP/s). A K block takes 660 cycles,
// as many as torch._scaled_mm without block scales spends on one; that runs in 0.51 ms
// because the power cap leaves it a higher clock. Rows leave through shared memory and TMA.
// Few tiles (65 to some hundred tokens): a cluster of up to four pairs shares one along K;
// each lays its sums into its ring, and every CTA adds a share of the tokens over the
// cluster, in the order of K.
// A role that gives up a wait does not tell the others within the loop: their own
// bounded waits end theirs.
constexpr int kWideConsumers = 8, kWideThreads = (4 + kWideConsumers) * 32;

// (a0, a1) += (r0, r1) * f, both products in one instruction. Volatile, so that it stays
// between the loads of tensor memory it is written between.
__device__ __forceinline__ void fold2(float& a0, float& a1, uint32_t r0, uint32_t r1, uint64_t f2) {
  asm volatile(
      "{\n\t.reg .b64 a, r;\n\t"
      "mov.b64 a, {%0, %1};\n\tmov.b64 r, {%2, %3};\n\t"
      "fma.rn.f32x2 a, r, %4, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(r0), "r"(r1), "l"(f2));
}

constexpr int kMaxPairs = 4;   // pairs of CTAs that share a tile along K

template <int BN>
struct WideLayout {
  static constexpr int kABytes = 128 * kBlk, kBBytes = BN / 2 * kBlk;   // per CTA
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (192 * 1024) / kStageBytes;
  static constexpr int kAcc = 512 / BN;
  static constexpr int kOutBytes = kWideConsumers * 32 * 128;          // 32 rows x 128 bytes per warp
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kOutBytes;
  static constexpr int kPartRow = BN * 4 + 16;   // a token's partial sums; odd in 16 bytes: no bank conflicts
  static_assert(128 * kPartRow <= kStages * kStageBytes, "the join reuses the ring");
  static_assert(kSmem <= 227 * 1024 - 512, "shared memory of a CTA");
};

// GATED: of the 256 columns of a tile, each half holds 64 gate rows and the 64 up rows of
// the same outputs, so that a thread has both; the two threads of a token row hold the
// tile's 128 outputs, one group of the 8-bit form, and exchange their maxima.
template <int BN, bool GATED>
__global__ void __launch_bounds__(kWideThreads, 1) gemm_fp8_wide_kernel(
    const Fp8GemmArgs p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
    const __grid_constant__ CUtensorMap map_o) {
  pdl_enter();
  using L = WideLayout<BN>;
  constexpr int S = L::kStages, NA = L::kAcc, NC = BN / (kWideConsumers / 4);
  extern __shared__ uint8_t raw_smem[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full_bar[S], done_bar[S], tempty_bar[NA], amax_bar[4], drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_abort;

  static_assert(!GATED || BN == 256, "128 outputs per tile");
  // GATED: [tile parity][half of the outputs][token], where the other form stages its rows
  float(*s_amax)[2][128] = reinterpret_cast<float(*)[2][128]>(ring + S * L::kStageBytes);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t crank = cluster::rank(), lead = crank & ~1u;   // lead: the CTA that issues for this pair
  const int rank = int(crank & 1), kpart = int(crank >> 1);
  const int pair = int(blockIdx.x) / (2 * p.splits), pairs = int(gridDim.x) / (2 * p.splits);
  // K blocks [k0, k0 + nk) of this pair (all of them unless a cluster shares a tile along K)
  const int base = p.nkb / p.splits, rem = p.nkb % p.splits;
  const int nk = base + (kpart < rem ? 1 : 0), k0 = kpart * base + min(kpart, rem);
  const int m_tiles = (p.M + 255) / 256, total = m_tiles * p.n_tiles;   // n_tiles of BN rows
  int armed = 0;

  if (tid == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&full_bar[i], 1), mbar_init(&done_bar[i], 1);
    for (int i = 0; i < NA; ++i) mbar_init(&tempty_bar[i], 2 * kWideConsumers);
    for (int i = 0; i < 4; ++i) mbar_init(&amax_bar[i], 2);
    mbar_init(&drain_bar, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(&tmem_slot, 512);
  tc_fence_before_sync();
  cluster::sync();   // both CTAs' barriers exist before either is signalled from the other
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0), ring_s = smem_u32(ring);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      const bool one = elect_one();
      if (one) tma::prefetch_map(&map_w), tma::prefetch_map(&map_a);
      const uint32_t full0 = cluster::map_shared(smem_u32(&full_bar[0]), lead);
      bool ok = true;
      int t = 0, s = 0;
      uint32_t ph = 1;
      for (int item = pair; item < total && ok; item += pairs) {
        const int nt = item / m_tiles, mt = item - nt * m_tiles;
        for (int kb = k0; kb < k0 + nk; ++kb) {
          ok = mbar_wait_warp(&done_bar[s], ph);
          if (!ok) break;
          if (one) {
            const uint32_t st = ring_s + s * L::kStageBytes;
            if (rank == 0) tma::mbar_expect_tx(&full_bar[s], 2 * L::kStageBytes);   // both CTAs' bytes
            tma::load_2d_pair(st, &map_a, kb * kBlk, mt * 256 + rank * 128, full0 + s * 8);
            if constexpr (GATED) {
              const int row = nt * 128 + rank * 64;
              tma::load_2d_pair(st + L::kABytes, &map_w, kb * kBlk, row, full0 + s * 8);
              tma::load_2d_pair(st + L::kABytes + 64 * kBlk, &map_w, kb * kBlk, p.N / 2 + row, full0 + s * 8);
            } else {
              tma::load_2d_pair(st + L::kABytes, &map_w, kb * kBlk, nt * BN + rank * (BN / 2), full0 + s * 8);
            }
          }
          __syncwarp();
          ++t;
          if (++s == S) s = 0, ph ^= 1;
        }
      }
      armed = t;
      if (!ok && lane == 0) atomicExch(p.status, 1), s_abort = 1;
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t idesc = instr_desc(D_F32, 0, 0, 256, BN);
      const uint32_t a_lo0 = smem_desc_lo(ring_s);
      const bool one = elect_one();
      bool ok = true;
      int s = 0, b = 0;
      uint32_t ph = 0, aph = 1;
      for (int item = pair; item < total && ok; item += pairs) {
        for (int kb = 0; kb < nk; ++kb) {
          ok = mbar_wait_warp(&tempty_bar[b], aph) && mbar_wait_warp(&full_bar[s], ph);
          if (!ok) break;
          tc_fence_after_sync();
          if (one) {
            const uint32_t a_lo = a_lo0 + s * (L::kStageBytes >> 4), b_lo = a_lo + (L::kABytes >> 4);
            const uint32_t d = tmem + b * BN;
            mma_f8_pair<false>(d, a_lo, b_lo, idesc);
            mma_f8_pair<true>(d, a_lo + 2, b_lo + 2, idesc);
            mma_f8_pair<true>(d, a_lo + 4, b_lo + 4, idesc);
            mma_f8_pair<true>(d, a_lo + 6, b_lo + 6, idesc);
            mma_commit_pair(&done_bar[s], lead);   // frees the stage and publishes the sums, in both CTAs
          }
          __syncwarp();
          if (++s == S) s = 0, ph ^= 1;
          if (++b == NA) b = 0, aph ^= 1;
        }
      }
      if (!ok && lane == 0) atomicExch(p.status, 1), s_abort = 1;
    }
    if (p.splits > 1) cluster::sync();   // the folding warps' exchange of partial sums
  } else {
    // 128 x 40 + 256 x 232 registers: the launch's 384 x 168
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int trow = (warp & 3) * 32 + lane;          // TMEM lane = token of this CTA's 128
    const int cg = (warp - 4) >> 2;                   // which half of the BN columns
    const uint32_t src0 = tmem + (uint32_t((warp & 3) * 32) << 16) + cg * NC;
    const uint32_t tempty0 = cluster::map_shared(smem_u32(&tempty_bar[0]), lead);
    int s = 0, b = 0;
    uint32_t ph = 0, xph = 0;
    bool dead = false;
    for (int item = pair; item < total && !dead; item += pairs) {
      const int nt = item / m_tiles, mt = item - nt * m_tiles;
      const int m = mt * 256 + rank * 128 + trow, n0 = GATED ? nt * 128 : nt * BN + cg * NC;
      const bool m_ok = m < p.M;
      // rows and blocks past the edge read the last valid scale; their sums are not stored
      const float* sa = p.sa + int64_t(m_ok ? m : p.M - 1) * p.sa_sm + int64_t(k0) * p.sa_sk;
      const float* sw = p.sw + int64_t((n0 < p.N ? n0 : p.N - 1) / kBlk) * p.sw_sn + int64_t(k0) * p.sw_sk;
      // GATED: the up rows' block, as far from the gate rows' as the halves are
      const int64_t up_block = GATED ? int64_t(p.N / 2 / kBlk) * p.sw_sn : 0;
      float a_next = __ldg(sa), w_next = __ldg(sw), u_next = GATED ? __ldg(sw + up_block) : 0.f;
      float acc[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[j] = 0.f;
      for (int kb = 0; kb < nk; ++kb) {
        const float f = a_next * w_next, fu = a_next * u_next;
        uint64_t f2, fu2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(f2) : "f"(f));
        asm("mov.b64 %0, {%1, %1};" : "=l"(fu2) : "f"(fu));
        if (kb + 1 < nk) {
          sa += p.sa_sk, sw += p.sw_sk;
          a_next = __ldg(sa), w_next = __ldg(sw);
          if constexpr (GATED) u_next = __ldg(sw + up_block);
        }
        if (!mbar_wait_warp(&done_bar[s], ph)) {
          dead = true;
          break;
        }
        tc_fence_after_sync();
        const uint32_t src = src0 + b * BN;
        // columns per load, two loads in registers: the gated form's second scale leaves room
        // for 16 only (with 32 the loop spills at most register budgets)
        constexpr int CH = GATED ? 16 : 32;
        uint32_t r[2][CH];
        tmem_ld(src, r[0]);
#pragma unroll
        for (int c = 0; c < NC / CH; ++c) {
          tmem_ld_wait();
          if (c + 1 < NC / CH) {
            tmem_ld(src + (c + 1) * CH, r[(c + 1) & 1]);
          } else {   // everything read: the accumulator may be written again
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty0 + b * 8);
          }
#pragma unroll
          for (int j = 0; j < CH; j += 2) {
            fold2(acc[c * CH + j], acc[c * CH + j + 1], r[c & 1][j], r[c & 1][j + 1], GATED && c * CH >= 64 ? fu2 : f2);
          }
        }
        if (++s == S) s = 0, ph ^= 1;
        if (++b == NA) b = 0;
      }
      if (dead) break;
      if (p.splits > 1) {
        // the one tile of this cluster: the partial sums [token][column] into the ring, whose
        // copies and MMAs have ended (the last K block's are the last)
        float4* mine = reinterpret_cast<float4*>(ring + trow * L::kPartRow + cg * (NC * 4));
#pragma unroll
        for (int j = 0; j < NC; j += 4) mine[j >> 2] = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        break;
      }
      if constexpr (GATED) {
        // outputs nt * 128 + cg * 64 + j: gate in acc[j], up in acc[64 + j]
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = quant8::gate(acc[j], p.gate_act) * acc[64 + j];
        float amax = fabsf(acc[0]);
#pragma unroll
        for (int j = 1; j + 1 < 64; j += 2) amax = quant8::max_nan(amax, fabsf(acc[j]), fabsf(acc[j + 1]));
        amax = quant8::max_nan(amax, fabsf(acc[63]));
        s_amax[xph][cg][trow] = amax;
        __syncwarp();
        if (lane == 0) mbar_arrive(&amax_bar[warp & 3]);
        if (!mbar_wait_warp(&amax_bar[warp & 3], xph)) {
          dead = true;
          break;
        }
        const float sc = quant8::scale_of(quant8::max_nan(amax, s_amax[xph][cg ^ 1][trow]), quant8::kTopF8);
        const float inv = quant8::rcp(sc);
        xph ^= 1;
        if (m_ok) {
          uint4* q = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + int64_t(m) * p.out_st + n0 + cg * 64);
#pragma unroll
          for (int j = 0; j < 64; j += 16)
            q[j >> 4] = make_uint4(
                quant8::pack_e4m3x4(acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv),
                quant8::pack_e4m3x4(acc[j + 4] * inv, acc[j + 5] * inv, acc[j + 6] * inv, acc[j + 7] * inv),
                quant8::pack_e4m3x4(acc[j + 8] * inv, acc[j + 9] * inv, acc[j + 10] * inv, acc[j + 11] * inv),
                quant8::pack_e4m3x4(acc[j + 12] * inv, acc[j + 13] * inv, acc[j + 14] * inv, acc[j + 15] * inv));
          if (cg == 0) p.q_scales[int64_t(m) * p.qs_st + nt] = sc;
        }
        continue;
      }
      const uint32_t stage_at = S * L::kStageBytes + (warp - 4) * (32 * 128);   // this warp's 4 KB
      auto reuse = [&] {   // the last rows staged there have been read
        if (lane == 0) tma::store_wait_read<0>();
        __syncwarp();
      };
      if (p.bias != nullptr) {
        // the warp's columns once into shared memory, then four per broadcast read
        float* sb = reinterpret_cast<float*>(ring + stage_at);
        reuse();
#pragma unroll
        for (int i = 0; i < NC / 32; ++i)
          sb[i * 32 + lane] = n0 + i * 32 + lane < p.N ? load_bias(p.bias, p.out_kind, n0 + i * 32 + lane) : 0.f;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < NC; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(sb + j);
          acc[j] += v.x, acc[j + 1] += v.y, acc[j + 2] += v.z, acc[j + 3] += v.w;
        }
        __syncwarp();
      }
      // 128 bytes of each of the warp's 32 rows at a time through shared memory, in the
      // 128-byte swizzle (eight lanes write eight different chunks). Where the output's rows
      // start and end on 16-byte boundaries they leave by TMA, which leaves out what lies past
      // M or N; else row by row, a warp on 128 consecutive bytes (4,096 x 33,333 x 5,120: 0.66 ms,
      // where 34,816 columns take 0.59).
      const int row0 = mt * 256 + rank * 128 + (warp & 3) * 32;
      auto put = [&](int chunk, uint4 v) {
        *reinterpret_cast<uint4*>(ring + stage_at + sw128_offset(lane, chunk)) = v;
      };
      auto flush = [&](int col, int bytes) {
        if (p.tma_out) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0 && row0 < p.M && col < p.N) tma::store_2d(&map_o, ring_s + stage_at, col * bytes, row0);
          if (lane == 0) tma::store_commit();
          return;
        }
        __syncwarp();
        const uint8_t* src = ring + stage_at;
        for (int i = 0; i < 32 && row0 + i < p.M; ++i) {
          uint8_t* dst = static_cast<uint8_t*>(p.out) + (int64_t(row0 + i) * p.out_st + col) * bytes;
          if (bytes == 4) {
            if (col + lane < p.N)
              *reinterpret_cast<uint32_t*>(dst + lane * 4) = *reinterpret_cast<const uint32_t*>(src + sw128_offset(i, lane >> 2) + (lane & 3) * 4);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int e = h * 32 + lane;
              if (col + e < p.N)
                *reinterpret_cast<uint16_t*>(dst + e * 2) = *reinterpret_cast<const uint16_t*>(src + sw128_offset(i, e >> 3) + (e & 7) * 2);
            }
          }
        }
        __syncwarp();
      };
      if (p.out_kind == kOutF32) {
#pragma unroll
        for (int j = 0; j < NC; j += 32) {
          reuse();
#pragma unroll
          for (int c = 0; c < 8; ++c)
            put(c, make_uint4(__float_as_uint(acc[j + 4 * c]), __float_as_uint(acc[j + 4 * c + 1]),
                              __float_as_uint(acc[j + 4 * c + 2]), __float_as_uint(acc[j + 4 * c + 3])));
          flush(n0 + j, 4);
        }
      } else {
        const bool bf = p.out_kind == kOutBf16;
#pragma unroll
        for (int j = 0; j < NC; j += 64) {
          reuse();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = acc[j + 8 * c + 2 * i], y = acc[j + 8 * c + 2 * i + 1];
              o[i] = bf ? pack_bf16x2(x, y) : pack_f16x2(x, y);
            }
            put(c, make_uint4(o[0], o[1], o[2], o[3]));
          }
          flush(n0 + j, 2);
        }
      }
    }
    if (p.splits > 1) {
      // tokens kpart, kpart + splits, ... of the pair's 128 per CTA, one warp per token, four
      // neighbouring columns per lane, kRows tokens at a time: all their reads are under way
      // before the first sum is used. The partial sums are added in the order of K.
      cluster::sync();
      constexpr int kRows = 4;
      const int nt = pair / m_tiles, mt = pair - nt * m_tiles;
      const uint32_t own = ring_s + lane * 16;
      auto joined = [&](float4(&v)[kRows], int row, int at) {
        float4 x[kMaxPairs][kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
          for (int c = 0; c < kMaxPairs; ++c) {
            const int r = row + i * p.splits * kWideConsumers;
            x[c][i] = c < p.splits && r < 128
                          ? cluster::ld_shared_f32x4(cluster::map_shared(own + r * L::kPartRow + at, uint32_t(2 * c + rank)))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          v[i] = x[0][i];
#pragma unroll
          for (int c = 1; c < kMaxPairs; ++c)
            v[i].x += x[c][i].x, v[i].y += x[c][i].y, v[i].z += x[c][i].z, v[i].w += x[c][i].w;
        }
      };
      const int m0 = mt * 256 + rank * 128;
      for (int row0 = kpart + p.splits * (warp - 4); row0 < 128 && m0 + row0 < p.M && !dead;
           row0 += p.splits * kWideConsumers * kRows) {
        if constexpr (GATED) {
          // lane l: outputs 4 l .. of the tile, whose gate columns lie at 128 (o / 64) + o % 64
          // and the up columns 64 further: 256 bytes more for the upper 16 lanes
          float4 g[kRows], u[kRows];
          joined(g, row0, (lane >> 4) * 256);
          joined(u, row0, (lane >> 4) * 256 + 256);
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            const int row = row0 + i * p.splits * kWideConsumers, m = m0 + row;
            const float y[4] = {quant8::gate(g[i].x, p.gate_act) * u[i].x, quant8::gate(g[i].y, p.gate_act) * u[i].y,
                                quant8::gate(g[i].z, p.gate_act) * u[i].z, quant8::gate(g[i].w, p.gate_act) * u[i].w};
            float amax = quant8::max_nan(quant8::max_nan(fabsf(y[0]), fabsf(y[1]), fabsf(y[2])), fabsf(y[3]));
#pragma unroll
            for (int o = 16; o; o >>= 1) amax = quant8::max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const float sc = quant8::scale_of(amax, quant8::kTopF8), inv = quant8::rcp(sc);
            if (row >= 128 || m >= p.M) continue;
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + int64_t(m) * p.out_st + nt * 128 + lane * 4) =
                quant8::pack_e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
            if (lane == 0) p.q_scales[int64_t(m) * p.qs_st + nt] = sc;
          }
        } else {
#pragma unroll 1
          for (int h = 0; h < BN / 128; ++h) {
            const int n = nt * BN + h * 128 + lane * 4;
            float b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = n + e < p.N ? load_bias(p.bias, p.out_kind, n + e) : 0.f;
            float4 v4[kRows];
            joined(v4, row0, h * 512);
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
              const int row = row0 + i * p.splits * kWideConsumers, m = m0 + row;
              if (row >= 128 || m >= p.M) continue;
              const float v[4] = {v4[i].x + b[0], v4[i].y + b[1], v4[i].z + b[2], v4[i].w + b[3]};
              const int64_t at = int64_t(m) * p.out_st + n;
              if (p.tma_out && n + 4 <= p.N) {   // rows on 16-byte boundaries: whole words
                if (p.out_kind == kOutF32)
                  *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
                else
                  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
                      p.out_kind == kOutBf16 ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]))
                                             : make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n + e < p.N) store_one(p.out, p.out_kind, at + e, v[e]);
              }
            }
          }
        }
      }
    }
    if (lane == 0) tma::store_wait_read<0>();   // the staged rows have left shared memory
    if (dead) atomicExch(p.status, 1), s_abort = 1;
  }

  tc_fence_before_sync();
  __syncthreads();
  if (s_abort) {
    // rank 0's barriers count the bytes of both CTAs and its thread issued all MMAs
    if (rank == 0 && tid == 0) drain_armed_loads(full_bar, S, armed);
    if (rank == 0 && warp == 1 && elect_one()) {
      mma_commit_pair(&drain_bar, lead);
      mbar_wait(&drain_bar, 0);
    }
  }
  tc_fence_before_sync();
  cluster::sync();   // no signal of the other CTA is under way when this one ends
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// `room`: pairs that find a place at once. Tiles go to the pairs by turns, so a pair beyond
// that would begin its share when another has ended its own.
template <int BN, bool GATED>
int launch_wide(Fp8GemmArgs p, int splits, int64_t room, const void* a, int64_t a_st, const void* w, int64_t w_st,
                int64_t k, int dev, cudaStream_t st) {
  using L = WideLayout<BN>;
  auto kernel = gemm_fp8_wide_kernel<BN, GATED>;
  static bool done[64] = {};
  if (!done[dev]) {
    STRIX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem));
    done[dev] = true;
  }
  p.n_tiles = (p.N + BN - 1) / BN;   // GATED: 128 outputs, 256 of gate and up rows together
  const int64_t tiles = int64_t(p.n_tiles) * ((p.M + 255) / 256);
  STRIX_CHECK(tiles < (int64_t(1) << 30), "matrix too large");
  const int64_t bytes = p.out_kind == kOutF32 ? 4 : 2;
  // a TMA store cuts a row's end to 16 bytes, not to the element: a row of another length
  // would run over into what lies behind it
  p.tma_out = !GATED && reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && (p.N * bytes) % 16 == 0 &&
              (p.M == 1 || (p.out_st * bytes) % 16 == 0);
  const int64_t o_st = p.M == 1 ? p.N * bytes : p.out_st * bytes;
  CUtensorMap map_w, map_a, map_o = {};
  STRIX_CHECK(tma::make_map_u8(&map_w, w, uint64_t(p.N), uint64_t(k), uint64_t(w_st), GATED ? 64 : BN / 2) &&
                  tma::make_map_u8(&map_a, a, uint64_t(p.M), uint64_t(k), uint64_t(a_st), 128) &&
                  (!p.tma_out || tma::make_map_u8(&map_o, p.out, uint64_t(p.M), uint64_t(p.N) * bytes, uint64_t(o_st), 32)),
              "tensor map encoding failed");
  p.splits = splits;
  const int64_t pairs = splits > 1 || tiles < room ? tiles * splits : room;
  STRIX_CUDA(cluster::launch(kernel, unsigned(2 * pairs), unsigned(2 * splits), kWideThreads, L::kSmem, st, p, map_w, map_a, map_o));
  return launch_status("w8a8_fp8_gemm");
}

// Clusters of c pairs that the current device runs at once, c = 1 .. kMaxPairs (asked once;
// all instantiations take an SM each).
int pair_places(int dev, const int** out) {
  static int places[64][kMaxPairs + 1] = {};
  if (!places[dev][1]) {
    auto kernel = gemm_fp8_wide_kernel<256, false>;
    constexpr size_t smem = WideLayout<256>::kSmem;
    STRIX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    for (int c = kMaxPairs; c >= 1; --c)
      STRIX_CUDA(cluster::places(&places[dev][c], kernel, unsigned(2 * c), unsigned(kWideThreads), smem));
    STRIX_CHECK(places[dev][1] > 0, "no room for a pair of CTAs");
  }
  *out = places[dev];
  return STRIX_OK;
}

// Tile width and pairs per tile of the wide kernel, by the time each would take in ns. Fitted
// to single rounds of 16 and 136 K blocks: a block costs a pair 372 on a tile of 256 x 256
// and 272 on 256 x 128, a round of the larger tile 1,400 more at its ends; pairs that share a
// tile need a place each at once, and their join costs 4,500 and 2,700. Measured at 128 x
// 5,120 x 17,408: 256 wide 55.5 us with one pair per tile, 27.3 with three, 128 wide 40.5;
// at 768 x 2,048 x 2,048: 11.0 and 8.3 us (one pair each); at 512 x 5,120 x 5,120: 20.9 and 24.8.
struct WidePlan {
  int bn, splits;
};
WidePlan wide_plan(int64_t m, int64_t n, int nkb, bool gated, const int* places) {
  WidePlan best{256, 1};
  int64_t least = INT64_MAX;
  for (int bn : {256, 128}) {
    if (gated && bn != 256) break;
    const int64_t tiles = ((m + 255) / 256) * ((n + bn - 1) / bn);
    const int64_t block = bn == 256 ? 372 : 272, ends = bn == 256 ? 1400 : 0, join = bn == 256 ? 4500 : 2700;
    for (int c = 1; c <= kMaxPairs; ++c) {
      if (c > 1 && (tiles > places[c] || nkb < 2 * c)) break;
      const int64_t rounds = c > 1 ? 1 : (tiles + places[1] - 1) / places[1];
      const int64_t t = rounds * ((nkb + c - 1) / c * block + ends) + (c > 1 ? join : 0);
      if (t < least) least = t, best = {bn, c};
    }
  }
  return best;
}

// The checks that both entry points share; fills what the kernels read of the operands.
int fp8_operands(Fp8GemmArgs& p, const void* a_q, const float* a_scale, const void* w, const float* w_scale,
                 int64_t m, int64_t n, int64_t k, int64_t& a_stride, int64_t& w_stride, int& dev) {
  STRIX_CHECK(m >= 0 && n > 0 && k > 0, "bad shapes");
  STRIX_CHECK(k % 16 == 0, "K must be a multiple of 16");
  STRIX_CHECK(n < (int64_t(1) << 31) - 256 && m < (int64_t(1) << 31) - 256 && k < (int64_t(1) << 31) - 256,
              "matrix too large");
  if (m == 0) return STRIX_OK;
  STRIX_CHECK(a_q != nullptr && a_scale != nullptr && w != nullptr && w_scale != nullptr,
              "pointers must not be NULL");
  // the stride of a single row is not read, but a tensor map wants a valid one
  if (m == 1) a_stride = k;
  if (n == 1) w_stride = k;
  STRIX_CHECK(a_stride % 16 == 0 && w_stride % 16 == 0 && reinterpret_cast<uintptr_t>(a_q) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(w) % 16 == 0,
              "16-byte aligned rows required");
  STRIX_CHECK(a_stride >= k && w_stride >= k && a_stride < (int64_t(1) << 40) && w_stride < (int64_t(1) << 40),
              "rows must not overlap");
  p.sa = a_scale, p.sw = w_scale;
  p.status = umma_status_ptr();
  STRIX_CHECK(p.status != nullptr, "status word unavailable");
  p.M = int(m), p.N = int(n), p.nkb = int((k + kBlk - 1) / kBlk);
  STRIX_CUDA(cudaGetDevice(&dev));
  STRIX_CHECK(dev >= 0 && dev < 64, "device index %d out of range", dev);
  return STRIX_OK;
}

int run_gemm(const Fp8GemmArgs& p, const void* a, int64_t a_st, const void* w, int64_t w_st, int64_t k, int dev,
             cudaStream_t st) {
  if (p.M <= 16) return launch_stream<16, false>(p, a, a_st, w, w_st, k, dev, st);
  if (p.M <= 32) return launch_stream<32, false>(p, a, a_st, w, w_st, k, dev, st);
  if (p.M <= 64) return launch_stream<64, false>(p, a, a_st, w, w_st, k, dev, st);
  const int* places = nullptr;
  const int rc = pair_places(dev, &places);
  if (rc != STRIX_OK) return rc;
  const WidePlan plan = wide_plan(p.M, p.N, p.nkb, false, places);
  if (plan.bn == 128) return launch_wide<128, false>(p, plan.splits, places[1], a, a_st, w, w_st, k, dev, st);
  return launch_wide<256, false>(p, plan.splits, places[1], a, a_st, w, w_st, k, dev, st);
}

}  // namespace
}  // namespace strix

using namespace strix;

extern "C" int strix_w8a8_fp8_gemm(void* out, const void* a_q, const float* a_scale, const void* w,
                                   const float* w_scale, const void* bias, int64_t m, int64_t n, int64_t k,
                                   int64_t a_stride, int64_t w_stride, int64_t out_stride,
                                   int64_t sa_stride_m, int64_t sa_stride_k, int64_t sw_stride_n,
                                   int64_t sw_stride_k, int out_kind, strix_stream_t stream) {
  STRIX_CHECK(out_kind >= 0 && out_kind <= 2, "output must be bf16, fp16 or fp32");
  Fp8GemmArgs p{};
  int dev = 0;
  const int rc = fp8_operands(p, a_q, a_scale, w, w_scale, m, n, k, a_stride, w_stride, dev);
  if (rc != STRIX_OK || m == 0) return rc;
  STRIX_CHECK(out != nullptr && (m == 1 || out_stride >= n), "output rows must not overlap");
  p.out = out, p.bias = bias, p.out_kind = out_kind;
  p.out_st = out_stride, p.sa_sm = sa_stride_m, p.sa_sk = sa_stride_k;
  p.sw_sn = sw_stride_n, p.sw_sk = sw_stride_k;
  return run_gemm(p, a_q, a_stride, w, w_stride, k, dev, static_cast<cudaStream_t>(stream));
}

// Whether the gated product runs in one kernel. Otherwise (gate and up rows that share a
// weight block) fp32 rows go through a workspace.
static bool gated_in_one(int64_t n) { return n % 128 == 0; }

extern "C" int64_t strix_w8a8_fp8_gated_workspace(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n <= 0 || k <= 0 || m >= (int64_t(1) << 31) || n >= (int64_t(1) << 30)) return -1;
  if (gated_in_one(n)) return 0;
  return m <= INT64_MAX / (8 * n) ? m * 8 * n : -1;   // (m * 8 * n may pass 63 bits)
}

extern "C" int strix_w8a8_fp8_gated(void* q, float* scales, const void* a_q, const float* a_scale,
                                    const void* w, const float* w_scale, void* workspace,
                                    int64_t workspace_bytes, int64_t m, int64_t n, int64_t k,
                                    int64_t a_stride, int64_t w_stride, int64_t q_stride, int64_t s_stride,
                                    int64_t sa_stride_m, int64_t sa_stride_k, int64_t sw_stride_n,
                                    int64_t sw_stride_k, int gate_act, strix_stream_t stream) {
  STRIX_CHECK(gate_act == 1 || gate_act == 2, "activation must be silu or gelu_tanh");
  STRIX_CHECK(n > 0 && n < (int64_t(1) << 30) - 128 && n % 16 == 0, "N must be a multiple of 16");
  Fp8GemmArgs p{};
  int dev = 0;
  int rc = fp8_operands(p, a_q, a_scale, w, w_scale, m, 2 * n, k, a_stride, w_stride, dev);
  if (rc != STRIX_OK || m == 0) return rc;
  STRIX_CHECK(q != nullptr && scales != nullptr, "pointers must not be NULL");
  if (m == 1) q_stride = n, s_stride = (n + 127) / 128;   // not read: any will do
  STRIX_CHECK(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride % 16 == 0, "16-byte aligned rows required");
  STRIX_CHECK(q_stride >= n && s_stride >= (n + 127) / 128, "output rows must not overlap");
  p.sa_sm = sa_stride_m, p.sa_sk = sa_stride_k, p.sw_sn = sw_stride_n, p.sw_sk = sw_stride_k;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (gated_in_one(n)) {
    // (33 to 64 tokens: the weight stream took 40.0 and 44.9 us at 33 and 64 x 17,408 x 5,120, the
    // wide tiles 42.9 and 43.3)
    p.out = q, p.out_st = q_stride, p.q_scales = scales, p.qs_st = s_stride, p.gate_act = gate_act;
    if (m <= 16) return launch_stream<16, true>(p, a_q, a_stride, w, w_stride, k, dev, st);
    if (m <= 32) return launch_stream<32, true>(p, a_q, a_stride, w, w_stride, k, dev, st);
    const int* places = nullptr;
    rc = pair_places(dev, &places);
    if (rc != STRIX_OK) return rc;
    const int splits = wide_plan(m, 2 * n, p.nkb, true, places).splits;
    return launch_wide<256, true>(p, splits, places[1], a_q, a_stride, w, w_stride, k, dev, st);
  }
  const int64_t need = strix_w8a8_fp8_gated_workspace(m, n, k);
  STRIX_CHECK(need >= 0, "matrix too large");
  STRIX_CHECK(workspace_bytes >= need && workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
              "workspace must hold %lld bytes on a 16-byte boundary", (long long)need);
  p.out = workspace, p.out_kind = kOutF32, p.out_st = 2 * n;
  rc = run_gemm(p, a_q, a_stride, w, w_stride, k, dev, st);
  if (rc != STRIX_OK) return rc;
  return strix_act_mul_quant(workspace, q, scales, m, n, 2 * n, q_stride, s_stride, gate_act, 2, 1, stream);
}
