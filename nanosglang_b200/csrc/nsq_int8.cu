// int8 linear (W8A8): y = (xc . wc^T) * xs * ws + bias, with xc, wc int8 codes,
// one fp32 scale per token (xs) and per output channel (ws); the sums are
// exact int32. Rows are quantised by int8_quantize_kernel.
//
// run_int8_rows: mma.sync.m16n8k32 with the weight rows as the 16 rows and the
// tokens as the columns. Both operands want four consecutive k per register
// and the order of k is free, so every lane reads 16 consecutive bytes of its
// row and feeds them to two MMAs as they come: weights go from global memory
// to the tensor cores without shared memory or conversion.
#include <type_traits>

#include "nsq_common.cuh"
#include "nsq_internal.h"
#include "nsq_rows8.cuh"

namespace nsq {

namespace {

constexpr int kQThreads = 256;

// ---------------------------------------------------------------------------
// Row quantiser: TPR threads per row, NV vectors of 16 bytes each, which stay in
// registers between the maximum and the codes (one pass over DRAM, which bounds
// it: 8192 x 4096 bf16 18.9 us, 5.3 TB/s; 16 x 4096 1.6 us). The host says
// how many threads a row takes. int8_quantize_any_kernel takes any row
// length, alignment and type, element by element, and reads the row twice (the
// second time from L2).
// ---------------------------------------------------------------------------

// What of programmatic launch a quantiser takes part in: it waits for the kernel
// ahead, and lets the one behind start at once. That one may be a product which
// loads its weight before it waits, so only a quantiser launched for the
// product's x does. One called by itself may be writing that weight: it releases
// nothing, and its codes are visible to all before a block of it ends.
constexpr int kPdlWait = 1, kPdlRelease = 2;

__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
  if (dtype == NSQ_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return dtype == NSQ_DTYPE_BF16 ? elem_to_float<true>(u) : elem_to_float<false>(u);
}

__device__ __forceinline__ float block_nan_max(float m) {
  __shared__ float red[kQThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = nan_max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < kQThreads / 32; ++i) m = nan_max(m, red[i]);
  return m;
}

template <int TPR, int NV, bool BF16>
__global__ void __launch_bounds__(kQThreads) int8_quantize_kernel(const uint16_t* __restrict__ x, int M, int K,
                                                                  int8_t* __restrict__ codes,
                                                                  float* __restrict__ scale, int pdl) {
  if (pdl & kPdlWait) pdl_wait_prior_grids();
  if (pdl & kPdlRelease) pdl_launch_dependents();
  __shared__ uint32_t red[kQThreads / 32];
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (kQThreads / TPR) + threadIdx.x / TPR;
  const bool in = row < M;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * K);
  const int nvec = in ? K / 8 : 0;
  uint4 v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = j * TPR + lane;
    v[j] = i < nvec ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
  }
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) m = abs_max2(m, v[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  if constexpr (TPR > 32) {
    const int w0 = threadIdx.x / TPR * (TPR / 32);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) m = __vmaxu2(m, red[w0 + i]);
  }
  if (!in) return;  // (the last block's rest: nothing to write)
  const float s = row_scale<false>(abs_max_value<BF16>(m));
  if (lane == 0) scale[row] = s;
  const RowDiv dv(s);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = j * TPR + lane;
    if (i < nvec) reinterpret_cast<uint2*>(codes + row * K)[i] = row_codes8<false, BF16>(dv, v[j]);
  }
  if (pdl == kPdlWait) __threadfence();
}

__global__ void __launch_bounds__(kQThreads) int8_quantize_any_kernel(const void* __restrict__ x, int dtype, int64_t K,
                                                                      int8_t* __restrict__ codes,
                                                                      float* __restrict__ scale, int pdl) {
  if (pdl & kPdlWait) pdl_wait_prior_grids();
  if (pdl & kPdlRelease) pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < K; i += kQThreads) m = nan_max(m, fabsf(load_elem(x, dtype, row * K + i)));
  const float s = row_scale<false>(block_nan_max(m));
  if (threadIdx.x == 0) scale[row] = s;
  const RowDiv dv(s);
  for (int64_t i = threadIdx.x; i < K; i += kQThreads) {
    codes[row * K + i] = (int8_t)row_code<false>(dv(load_elem(x, dtype, row * K + i)));
  }
  if (pdl == kPdlWait) __threadfence();
}

// ---------------------------------------------------------------------------
// Product, rows of the weight streamed through mma.sync
// ---------------------------------------------------------------------------
constexpr int kRWarps = 8;

__device__ __forceinline__ void mma_16832_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ldg_w(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void dsmem_add(uint32_t cluster_addr, int v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.s32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

struct RowsParams {
  const int8_t* x;
  const uint16_t* x16;  // FUSED: x itself
  const float* xscale;
  const int8_t* w;
  const float* wscale;
  const void* bias;
  int bias_dtype;
  void* y;
  int M, K, N;
  int pdl_x;  // x and xscale come from the kernel ahead
  int split;  // CTAs of a cluster, along K
};

// The block's part of FUSED: token m's row by kRWarps / tokens warps (tokens
// rounded up to a power of two), its maximum, then its codes (the second read
// hits L1). Called by every thread once.
template <bool BF16>
__device__ __forceinline__ void rows_quantize(const RowsParams& p, int8_t* xs, int ldx, uint32_t* xmax_s,
                                              float* xscale_s) {
  if (p.pdl_x) pdl_wait_prior_grids();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = p.M == 1 ? 8 : p.M == 2 ? 4 : p.M <= 4 ? 2 : 1;  // warps per token
  const int m = warp / per;
  const bool in = m < p.M;
  const uint4* src = reinterpret_cast<const uint4*>(p.x16 + (int64_t)(in ? m : 0) * p.K);
  const int nvec = in ? p.K / 8 : 0, first = (warp % per) * 32 + lane;
  uint32_t mx = 0;
  for (int i = first; i < nvec; i += per * 32) mx = abs_max2(mx, __ldg(src + i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) xmax_s[warp] = mx;
  __syncthreads();
  for (int i = 0; i < per; ++i) mx = __vmaxu2(mx, xmax_s[m * per + i]);
  const float s = row_scale<false>(abs_max_value<BF16>(mx));
  if (in && first == 0) xscale_s[m] = s;
  const RowDiv dv(s);
  for (int i = first; i < nvec; i += per * 32) {
    *reinterpret_cast<uint2*>(xs + m * ldx + i * 8) = row_codes8<false, BF16>(dv, __ldg(src + i));
  }
  __syncthreads();
}

// 16 weight rows x 8 * MT tokens per cluster of `split` CTAs along K. The warps
// of all of them take 64-column chunks in turn and add their int32 sums in the
// first CTA's shared memory (exact, so the order is free).
// FUSED (up to 8 tokens, few elements): x is 16-bit; every CTA quantises all of
// it into its shared memory while its first weights are on their way, which
// takes less time than a launch of the row quantiser and its round trip.
// The weight's stream bounds it, for small layers the round trips of one pass
// (in a graph, all included: 1 x 896 -> 4864 3.8 us, 1 x 4096 -> 4096 7.0 us =
// 2.4 TB/s, 8 x 14336 -> 4096 21 us = 2.8 TB/s).
template <int MT, bool BF16, bool FUSED>
__global__ void __launch_bounds__(kRWarps * 32) int8_rows_kernel(const RowsParams p) {
  constexpr int kLd = 8 * MT + 1;
  __shared__ int acc_s[16][kLd];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % p.split;  // the cluster's rank along x
  const int n0 = blockIdx.x / p.split * 16, m0 = blockIdx.y * (8 * MT);
  for (int i = threadIdx.x; i < 16 * kLd; i += kRWarps * 32) (&acc_s[0][0])[i] = 0;
  extern __shared__ uint4 xs_raw[];  // FUSED: codes [M][ldx]; rows 64 bytes apart modulo 128: no bank conflicts
  int8_t* const xs = reinterpret_cast<int8_t*>(xs_raw);
  const int ldx = (p.K + 127) / 128 * 128 + 64;
  __shared__ uint32_t xmax_s[kRWarps];
  __shared__ float xscale_s[8];
  const int8_t* w0 = p.w + (int64_t)(n0 + g) * p.K;
  const int8_t* w1 = w0 + (int64_t)8 * p.K;
  const bool r0 = n0 + g < p.N, r1 = n0 + g + 8 < p.N;
  int d[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0;
  // kAhead chunks' weights are loaded before their products: with the other
  // warps of the SM, 64 KB and more in flight
  constexpr int kAhead = MT <= 2 ? 4 : 2;
  const int step = p.split * kRWarps * 64;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  int k0 = (rank * kRWarps + warp) * 64;
  bool waiting = FUSED || p.pdl_x;
  do {  // every warp once at least: all meet in the first round's quantisation
    uint4 a[kAhead], c[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = k0 + j * step + t * 16;
      a[j] = k < p.K && r0 ? ldg_w(w0 + k) : zero;
      c[j] = k < p.K && r1 ? ldg_w(w1 + k) : zero;
    }
    if (waiting) {  // the first weights are on their way while the codes of x are made
      if constexpr (FUSED) {
        rows_quantize<BF16>(p, xs, ldx, xmax_s, xscale_s);
      } else {
        pdl_wait_prior_grids();
      }
      waiting = false;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = k0 + j * step + t * 16;
      if (j > 0 && k0 + j * step >= p.K) break;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + 8 * i + g;
        uint4 b = zero;
        if (k < p.K && m < p.M) {
          b = FUSED ? *reinterpret_cast<const uint4*>(xs + m * ldx + k)
                    : *reinterpret_cast<const uint4*>(p.x + (int64_t)m * p.K + k);
        }
        mma_16832_s8(d[i], a[j].x, c[j].x, a[j].y, c[j].y, b.x, b.y);
        mma_16832_s8(d[i], a[j].z, c[j].z, a[j].w, c[j].w, b.z, b.w);
      }
    }
    k0 += kAhead * step;
  } while (k0 < p.K);
  const uint32_t acc0 = smem_u32(acc_s);
  if (p.split > 1) {
    cluster_sync_all();  // the first CTA's sums are zero
    const uint32_t first = dsmem_map(acc0, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint32_t at = first + (g * kLd + 8 * i + 2 * t) * 4;
      dsmem_add(at, d[i][0]);
      dsmem_add(at + 4, d[i][1]);
      dsmem_add(at + 8 * kLd * 4, d[i][2]);
      dsmem_add(at + 8 * kLd * 4 + 4, d[i][3]);
    }
    cluster_sync_all();  // and complete
    if (rank != 0) return;
  } else {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      atomicAdd(&acc_s[g][8 * i + 2 * t], d[i][0]);
      atomicAdd(&acc_s[g][8 * i + 2 * t + 1], d[i][1]);
      atomicAdd(&acc_s[g + 8][8 * i + 2 * t], d[i][2]);
      atomicAdd(&acc_s[g + 8][8 * i + 2 * t + 1], d[i][3]);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 16 * 8 * MT; i += kRWarps * 32) {
    const int n = n0 + (i & 15), m = m0 + (i >> 4);
    if (n < p.N && m < p.M) {
      const float y = (float)acc_s[i & 15][i >> 4] * (FUSED ? xscale_s[m] : p.xscale[m]) * __ldg(p.wscale + n);
      const float bn = load_bias(p.bias, p.bias_dtype, n);
      static_cast<uint16_t*>(p.y)[(int64_t)m * p.N + n] = float_to_elem<BF16>(p.bias ? y + bn : y);
    }
  }
}

template <typename F, typename... A>
cudaError_t launch(F kern, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, bool pdl, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace

template <int TPR, bool BF16>
static cudaError_t quantize_rows(const uint16_t* x, int M, int K, int8_t* codes, float* scale, cudaStream_t stream,
                                 int pdl) {
  const dim3 grid((unsigned)((M + kQThreads / TPR - 1) / (kQThreads / TPR)));
  const int per = (K / 8 + TPR - 1) / TPR;
  auto go = [&](auto kern) {
    return launch(kern, grid, kQThreads, 0, 1, stream, (pdl & kPdlWait) != 0, x, M, K, codes, scale, pdl);
  };
  if constexpr (TPR == 256) {
    if (per > 8) return go(int8_quantize_kernel<TPR, 16, BF16>);
  }
  return per <= 1   ? go(int8_quantize_kernel<TPR, 1, BF16>)
         : per <= 2 ? go(int8_quantize_kernel<TPR, 2, BF16>)
         : per <= 4 ? go(int8_quantize_kernel<TPR, 4, BF16>)
                    : go(int8_quantize_kernel<TPR, 8, BF16>);
}

cudaError_t launch_int8_quantize(const void* x, int dtype, int64_t rows, int64_t K, int8_t* codes, float* scale,
                                 cudaStream_t stream, bool before_product) {
  const int pdl = (pdl_enabled() ? kPdlWait : 0) | (before_product ? kPdlRelease : 0);
  const bool vec = dtype != NSQ_DTYPE_F32 && K % 8 == 0 && K <= 16 * 8 * kQThreads &&
                   ((reinterpret_cast<uintptr_t>(x) & 15) | (reinterpret_cast<uintptr_t>(codes) & 7)) == 0;
  if (!vec) {
    return launch(int8_quantize_any_kernel, dim3((unsigned)rows), kQThreads, 0, 1, stream, (pdl & kPdlWait) != 0, x,
                  dtype, K, codes, scale, pdl);
  }
  const uint16_t* x16 = static_cast<const uint16_t*>(x);
  auto go = [&](auto tpr) {
    constexpr int T = decltype(tpr)::value;
    return dtype == NSQ_DTYPE_BF16 ? quantize_rows<T, true>(x16, (int)rows, (int)K, codes, scale, stream, pdl)
                                   : quantize_rows<T, false>(x16, (int)rows, (int)K, codes, scale, stream, pdl);
  };
  // Threads of a row, measured (us; 32, 64, 128, 256 threads): few rows want all
  // of them (512 x 4096 5.4, 4.7, 3.7, 3.6); many rows a warp while it loads the
  // row in few steps (16384 x 896 9.5, 11.1, 14.0, 21.2; 8192 x 1536 9.2, 9.3,
  // 10.6, 13.4), then 128 (16384 x 2048 23.5, 23.2, 20.9, 26.7; 8192 x 4096
  // 23.9, 23.7, 18.4, 20.8) until these need more than eight steps.
  const bool few = rows < 8 * num_sms();
  if (few || K > 128 * 64) return go(std::integral_constant<int, 256>());
  return K > 1536 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 32>());
}

int run_int8_rows(const Int8Args& a, cudaStream_t stream) {
  const bool fused = a.x16 != nullptr;
  RowsParams p{a.x, static_cast<const uint16_t*>(a.x16), a.xscale, a.w, a.wscale, a.bias,
               a.bias ? a.bias_dtype : NSQ_DTYPE_NONE, a.y, a.M, a.K, a.N, a.after_quantize || pdl_enabled(), 1};
  const int mt = a.M <= 8 ? 1 : a.M <= 16 ? 2 : a.M <= 32 ? 4 : 8;
  const int64_t tiles = (int64_t)((a.N + 15) / 16) * ((a.M + 8 * mt - 1) / (8 * mt));
  // K over a cluster while the CTAs do not fill two per SM and each has 1024
  // columns left, at up to 8 tokens (4864 -> 896 at M = 1 8.1 -> 6.6 us); the
  // exchange through distributed shared memory costs more with more tokens
  // (at M = 16 10.8 -> 11.9 us)
  while (mt == 1 && p.split < 8 && tiles * p.split * 2 <= 2 * num_sms() && a.K / (2 * p.split) >= 1024) p.split *= 2;
  const dim3 grid((unsigned)((a.N + 15) / 16 * p.split), (unsigned)((a.M + 8 * mt - 1) / (8 * mt)));
  const int smem = fused ? a.M * ((a.K + 127) / 128 * 128 + 64) : 0;
#define NSQ_R(MT, F)                                                                                              \
  (a.y_bf16 ? launch(int8_rows_kernel<MT, true, F>, grid, kRWarps * 32, smem, p.split, stream, p.pdl_x, p)        \
            : launch(int8_rows_kernel<MT, false, F>, grid, kRWarps * 32, smem, p.split, stream, p.pdl_x, p))
  const cudaError_t e = fused     ? NSQ_R(1, true)
                        : mt == 1 ? NSQ_R(1, false)
                        : mt == 2 ? NSQ_R(2, false)
                        : mt == 4 ? NSQ_R(4, false)
                                  : NSQ_R(8, false);
#undef NSQ_R
  return e == cudaSuccess ? NSQ_OK : NSQ_ECUDA;
}

}  // namespace nsq
