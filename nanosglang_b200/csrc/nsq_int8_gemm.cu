// int8 linear, tensor-core path for more than a few tokens:
//   y^T = (wc . xc^T) * ws * xs + bias
// with tcgen05.mma kind::i8 (s8 x s8 -> s32, exact), weight rows as the 128
// (one CTA) or 256 (CTA pair) rows, tokens as the columns, both operands
// K-major 128-byte-swizzled tiles that TMA brings from global memory.
//
// What bounds it: at 256 x 256 x 128 per step a pair reads 64 KB from L2 for
// 512 cycles of int8 tensor work, so the L2 path and the tensor pipe are near
// balance; hence the largest tile whose accumulator still double-buffers in
// tensor memory (2 x 256 columns), and a tile order in which the tiles that
// run at the same time share their weight rows and tokens (32 token tiles by as
// many weight tiles as it takes). Measured: 8192 x 4096 x 14336 in 306 us, 3.1
// P/s (less under the sustained power limit); with the token scales loaded
// after the epilogue's wait instead of before 410 us, with stages of one
// k-block 600 us, with groups of 8 token tiles 3% more.
//
// Warp roles (per CTA, 352 threads): 0 TMA of the weight, 1 MMA issuer (of a
// pair, the even CTA's), 2 TMA of x (one lane issues a copy in about 100 cycles,
// so one warp for all four of a stage would set the pace), 3..10 epilogue. A
// stage holds two 128-column k-blocks, so a barrier round covers 8 MMAs.
// An MMA of one CTA takes about 62 cycles for its 128 rows and half a cycle a
// token (with 64 rows 51), which bounds small layers at few tokens: 128 x 4096
// -> 4096 takes 10.3 us, 5.3 of them in the MMAs. With one token tile (decode
// batches) it is the weight's bandwidth that counts: the rows are then dealt
// evenly over the SMs, fewer than 128 to a tile (the MMA's other rows compute on
// leftovers of the stage that nothing reads), and the ring keeps 150 KB or more
// per SM in flight.
// Where tiles are few and K is long, a cluster of up to 4 CTAs shares a tile
// along K (SPLIT): each copies its sums of every other one's slice of tokens
// there in bulk, adds up its own slice and finishes it (integers: exact in any
// order).
// The epilogue of one tile runs under the MMAs of
// the next: s32 -> fp32, scales, bias, one rounding, a staged [token][feature]
// tile, stored by TMA where it is whole blocks of 64 features, else 16 bytes at a
// time (300 x 896 -> 4864 8.9 us, 512 x 4096 -> 4096 16.0 us; with 2-byte stores,
// which are left for N % 8 != 0, 9.4 and 16.6).
// Every wait is bounded. No TMA multicast.
#include <atomic>

#include "nsq_common.cuh"
#include "nsq_internal.h"

namespace nsq {

namespace {

constexpr int kRows = 128;  // weight rows per CTA
constexpr int kBK = 128;    // columns per k-block: one 128-byte swizzled row
constexpr int kKps = 2;     // k-blocks per stage
constexpr int kEpi = 8;     // epilogue warps
constexpr int kGemmThreads = 32 * (3 + kEpi);
constexpr int kGroup = 32;   // token tiles that share a pass over the weight

// CG CTAs per tile, TOK tokens per tile.
template <int CG, int TOK>
struct GemmShape {
  static constexpr int kXRows = TOK / CG;  // tokens staged per CTA
  static constexpr int kWBytes = kRows * kBK, kXBytes = kXRows * kBK;
  static constexpr int kStage = kKps * (kWBytes + kXBytes);
  static constexpr int kTokRound = TOK < 128 ? TOK : 128;  // tokens of a staged y tile
  static constexpr int kWarpTok = kTokRound < 64 ? 32 : kTokRound / 2;  // of them, an epilogue warp's
  static constexpr int kYHalf = kTokRound * 64 * 2;        // 64 features
  static constexpr int kFit = (226 * 1024 - 2 * kYHalf - 1024) / kStage, NS = kFit < 6 ? kFit : 6;
  static constexpr int kY = NS * kStage;
  static constexpr int kBar = kY + 2 * kYHalf;
  // full[NS], done[NS], full_acc[2], empty_acc[2], drain, sums
  static constexpr int kBars = 2 * NS + 6;
  static constexpr int kTmemSlot = kBar + kBars * 8;
  static constexpr int kAbort = kTmemSlot + 4;
  static constexpr int kAlloc = kAbort + 4 + 1024;
  static constexpr uint32_t kTmemCols = 2 * TOK;
  static_assert(kAlloc <= 227 * 1024 && NS >= 3, "shared memory per CTA");
  static_assert(kStage % 1024 == 0 && kYHalf % 1024 == 0, "swizzled tiles are 1 KB aligned");
};

struct GemmParams {
  const float* xscale;
  const float* wscale;
  const void* bias;
  void* y;
  DevStatus* status;
  int M, N, bias_dtype;
  int num_w, num_t, num_kb, num_st;
  int wrows;  // weight rows of a CTA's tile
  int split;  // SPLIT: CTAs of a cluster that share a tile, along K
  int tma_y;  // STAGED: the tile is whole blocks of 64 features, stored by TMA; else by the threads
  int pdl_x;  // x and its scales come from the kernel ahead on the stream
  int withhold;  // failure-path test hook: the first CTA's first stage never completes
};

__device__ __forceinline__ void gemm_unit(const GemmParams& p, int u, int& wt, int& tt) {
  const int per = kGroup * p.num_w;
  const int grp = u / per, r = u - grp * per;
  const int g0 = grp * kGroup;
  const int gs = p.num_t - g0 < kGroup ? p.num_t - g0 : kGroup;
  wt = r / gs;
  tt = g0 + r - wt * gs;
}

// The MMA's N for token tile tt: all tokens, or the rest rounded up to 32
// (rows past M read as zero).
template <int TOK>
__device__ __forceinline__ int gemm_n(int M, int tt) {
  const int rem = M - tt * TOK;
  return rem >= TOK ? TOK : ((rem + 31) & ~31);
}

// kind::i8: D s32 (2), A and B s8 (1), both K-major
__host__ __device__ constexpr uint32_t idesc_s8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// The four MMAs of a k-block (K = 32 each, +32 bytes = +2 descriptor units a
// step), issued back to back by the elected lane of a converged warp. Only the
// first takes `accumulate`.
template <int CG>
__device__ __forceinline__ void umma_i8_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define NSQ_I8_PRE "{\n\t.reg .pred e, p, t;\n\t.reg .b32 r;\n\telect.sync r|e, 0xffffffff;\n\t"
#define NSQ_I8_4(M)                                                     \
  M "[%0], %1, %5, %9, p;\n\t" M "[%0], %2, %6, %9, t;\n\t"              \
  M "[%0], %3, %7, %9, t;\n\t" M "[%0], %4, %8, %9, t;\n\t"
#define NSQ_I8_GO(M)                                                                                                   \
  asm volatile(NSQ_I8_PRE "setp.ne.b32 p, %10, 0;\n\tsetp.eq.b32 t, %10, %10;\n\t" NSQ_I8_4(M) "}" ::"r"(d), "l"(a),   \
               "l"(a + 2), "l"(a + 4), "l"(a + 6), "l"(b), "l"(b + 2), "l"(b + 4), "l"(b + 6), "r"(idesc),              \
               "r"(accumulate)                                                                                         \
               : "memory")
  if constexpr (CG == 1) {
    NSQ_I8_GO("@e tcgen05.mma.cta_group::1.kind::i8 ");
  } else {
    NSQ_I8_GO("@e tcgen05.mma.cta_group::2.kind::i8 ");
  }
#undef NSQ_I8_PRE
#undef NSQ_I8_4
#undef NSQ_I8_GO
}

// Whether the phase is complete, without waiting for it.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// TMA load whose bytes are counted on a barrier of the pair's even CTA.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int c0,
                                                 int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)float_to_elem<BF16>(a) | ((uint32_t)float_to_elem<BF16>(b) << 16);
}

template <int CG, int TOK, bool BF16, bool STAGED, bool SPLIT>
__global__ void __launch_bounds__(kGemmThreads, 1) int8_gemm_kernel(const __grid_constant__ CUtensorMap xmap,
                                                                    const __grid_constant__ CUtensorMap wmap,
                                                                    const __grid_constant__ CUtensorMap ymap,
                                                                    const GemmParams p) {
  using S = GemmShape<CG, TOK>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // a stage's tiles landed (pair: both CTAs', even CTA's barrier)
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* done = full + S::NS;                                 // its MMAs finished (both CTAs)
  uint64_t* full_acc = done + S::NS;                             // an accumulator is complete (both CTAs)
  uint64_t* empty_acc = full_acc + 2;                            // and read out by every epilogue warp (even CTA)
  uint64_t* drain = empty_acc + 2;
  uint64_t* sums = drain + 1;  // SPLIT: the other CTAs' sums of this one's slice have landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kTmemSlot);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  // SPLIT: one tile per cluster, and the stages [st0, st1) of it
  const int share = SPLIT ? p.split : CG;
  const int cid = blockIdx.x / share, ncl = gridDim.x / share;
  const int krank = SPLIT ? (int)cluster_ctarank() : 0;
  const int st0 = SPLIT ? p.num_st * krank / p.split : 0, st1 = SPLIT ? p.num_st * (krank + 1) / p.split : p.num_st;
  // the sums of a token: kRows of them, a 16-byte multiple that keeps rows off one another's banks
  constexpr uint32_t kSumBytes = (kRows + 4) * 4;
  const int slice = SPLIT ? TOK / p.split : 0;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < S::NS; ++i) {
      mbar_init(&full[i], 1 + (p.withhold && i == 0 && blockIdx.x == 0));
      mbar_init(&done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full_acc[i], 1);
      mbar_init(&empty_acc[i], CG * kEpi);
    }
    mbar_init(drain, 1);
    mbar_init(sums, 1);
    fence_barrier_init();
    if (SPLIT) mbar_arrive_expect_tx(sums, (uint32_t)((p.split - 1) * slice) * kSumBytes);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, S::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, S::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2 || SPLIT) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int units = p.num_w * p.num_t;
  bool ok = true;
  auto commit = [&](uint64_t* bar) {
    if constexpr (CG == 2) {
      tc_commit_pair_mc_elect(bar, 0x3);
    } else {
      tc_commit_elect(bar);
    }
  };

  if (warp == 0 || warp == 2) {
    // ---------------- TMA producers: the weight, x ----------------
    const bool is_x = warp == 2;
    if (lane == 0) {
      const CUtensorMap* map = is_x ? &xmap : &wmap;
      tma_prefetch_desc(map);
      const uint32_t full0 = CG == 2 ? dsmem_map(smem_u32(&full[0]), 0) : 0;
      uint8_t* const place = smem + (is_x ? kKps * S::kWBytes : 0);
      const int bytes = is_x ? S::kXBytes : S::kWBytes;
      // The weight does not depend on the kernel ahead: its first stages are on
      // their way while that one still runs.
      if (is_x && p.pdl_x) pdl_wait_prior_grids();
      int it = 0, s = 0;
      uint32_t phase = 1;  // of done[s], one use back
      for (int u = cid; u < units && ok; u += ncl) {
        int wt, tt;
        gemm_unit(p, u, wt, tt);
        const int row = is_x ? tt * TOK + (int)rank * (gemm_n<TOK>(p.M, tt) / CG) : (wt * CG + (int)rank) * p.wrows;
        for (int st = st0; st < st1; ++st, ++it) {
          if (!(ok = mbar_wait(&done[s], phase, p.status, is_x ? 214 : 210, abort_flag))) break;
          const int kb0 = st * kKps;
          const int nk = p.num_kb - kb0 < kKps ? p.num_kb - kb0 : kKps;
          // the even CTA arms the barrier for the bytes of both
          if (!is_x && leader) {
            mbar_arrive_expect_tx(&full[s], (uint32_t)(CG * nk) * (uint32_t)(p.wrows * kBK + S::kXBytes));
          }
#pragma unroll
          for (int i = 0; i < kKps; ++i) {
            if (i < nk) {
              if constexpr (CG == 2) {
                tma_load_2d_pair(place + s * S::kStage + i * bytes, map, full0 + s * 8, (kb0 + i) * kBK, row);
              } else {
                tma_load_2d(place + s * S::kStage + i * bytes, map, &full[s], (kb0 + i) * kBK, row);
              }
            }
          }
          if (++s == S::NS) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && !is_x && leader) {  // let copies in flight land before the CTA (of a pair, both) can exit
        for (int j = it > S::NS ? it - S::NS : 0; j < it; ++j) {
          mbar_wait(&full[j % S::NS], (j / S::NS) & 1, nullptr, 0, nullptr);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (leader) {
      // The next stage's barrier is looked at between this one's two groups of
      // MMAs, so that the tensor pipe has work while the answer comes back.
      const uint32_t base0 = smem_u32(smem);
      int it = 0, tc = 0, s = 0;
      uint32_t phase = 0;
      bool ready = false;  // full[s] was seen complete
      for (int u = cid; u < units && ok; u += ncl, ++tc) {
        int wt, tt;
        gemm_unit(p, u, wt, tt);
        const uint32_t idesc = idesc_s8(CG * kRows, gemm_n<TOK>(p.M, tt));
        const int buf = tc & 1;
        const uint32_t d = tmem + buf * TOK;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty_acc[buf], ((tc >> 1) & 1) ^ 1, p.status, 211, abort_flag));
        if (!ok) break;
        tc_fence_after();
        for (int st = st0; st < st1; ++st, ++it) {
          if (!ready) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[s], phase, p.status, 212, abort_flag));
            if (!ok) break;
          }
          tc_fence_after();
          const uint32_t base = base0 + s * S::kStage;
          umma_i8_elect<CG>(d, sw128_kmajor_desc(base), sw128_kmajor_desc(base + kKps * S::kWBytes), idesc, st > st0);
          const int s1 = s + 1 == S::NS ? 0 : s + 1;
          const uint32_t phase1 = s1 == 0 ? phase ^ 1 : phase;
          ready = __all_sync(0xffffffffu, mbar_test(&full[s1], phase1));
          if (p.num_kb - st * kKps >= 2) {
            umma_i8_elect<CG>(d, sw128_kmajor_desc(base + S::kWBytes),
                              sw128_kmajor_desc(base + kKps * S::kWBytes + S::kXBytes), idesc, 1u);
          }
          commit(&done[s]);
          s = s1;
          phase = phase1;
        }
        if (!ok) break;
        commit(&full_acc[buf]);
      }
      // every MMA issued has finished before tensor memory is released
      commit(drain);
      mbar_wait(drain, 0, nullptr, 0, nullptr);
    }
  } else if constexpr (!SPLIT) {
    // ---------------- epilogue ----------------
    if (p.pdl_x) pdl_wait_prior_grids();  // the scales of x, and y's buffer
    const int sub = warp & 3;             // tensor-memory sub-partition: 32 weight rows
    const int half = (warp - 3) >> 2;     // half of a round's tokens
    const int etid = threadIdx.x - 96;
    const int g = lane >> 2, t = lane & 3;
    const bool has_bias = p.bias_dtype != NSQ_DTYPE_NONE;
    const uint32_t empty0 = CG == 2 ? dsmem_map(smem_u32(&empty_acc[0]), 0) : 0;
    const uint32_t ystage = smem_u32(smem + S::kY + (sub >> 1) * S::kYHalf);
    const uint32_t ychunk = (uint32_t)((sub & 1) * 4 + (lane >> 3));
    int tc = 0;
    for (int u = cid; u < units && ok; u += ncl, ++tc) {
      int wt, tt;
      gemm_unit(p, u, wt, tt);
      const int buf = tc & 1;
      const int f0 = (wt * CG + (int)rank) * p.wrows;  // first feature of this CTA
      const int f1 = f0 + p.wrows < p.N ? f0 + p.wrows : p.N;
      // fragment rows of this lane: features sub * 32 + 8 q + g
      float wsc[4], bf[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = f0 + sub * 32 + 8 * q + g;
        wsc[q] = n < f1 ? __ldg(p.wscale + n) : 0.f;
        bf[q] = has_bias && n < f1 ? load_bias(p.bias, p.bias_dtype, n) : 0.f;
      }
      // the scales of this lane's tokens, too, come before the wait for the accumulator
      constexpr int kWarpTok = S::kWarpTok, kRounds = TOK / S::kTokRound, kChunks = kWarpTok / 32;
      float xs[kRounds][kChunks][8];
#pragma unroll
      for (int rd = 0; rd < kRounds; ++rd) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int m = tt * TOK + rd * S::kTokRound + half * kWarpTok + c * 32 + 8 * (j >> 1) + 2 * t + (j & 1);
            xs[rd][c][j] = m < p.M ? p.xscale[m] : 0.f;
          }
        }
      }
      ok = mbar_wait(&full_acc[buf], (tc >> 1) & 1, p.status, 213, abort_flag);
      if (!named_bar_all(1, kEpi * 32, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(sub * 32) << 16) + buf * TOK;
#pragma unroll
      for (int rd = 0; rd < kRounds; ++rd) {
        if constexpr (STAGED) {
          if (etid == 0) bulk_wait_group_read<0>();  // the staged tile's last store has read it
          named_bar_sync(1, kEpi * 32);
        }
        const int col0 = rd * S::kTokRound + half * kWarpTok;
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
          const int c = ch * 32;
          if (half * kWarpTok >= S::kTokRound || tt * TOK + col0 + c >= p.M) break;
          uint32_t r0[16], r1[16];
          tmem_ld_16x256b_x4(acc + col0 + c, r0);
          tmem_ld_16x256b_x4(acc + (16u << 16) + col0 + c, r1);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // tokens 8j + 2t, + 1 of features g, g + 8, g + 16, g + 24
            float v[4][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              v[0][e] = (float)(int)r0[4 * j + e];
              v[1][e] = (float)(int)r0[4 * j + 2 + e];
              v[2][e] = (float)(int)r1[4 * j + e];
              v[3][e] = (float)(int)r1[4 * j + 2 + e];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                v[q][e] = v[q][e] * xs[rd][ch][2 * j + e] * wsc[q];
                if (has_bias) v[q][e] += bf[q];
              }
            }
            if constexpr (STAGED) {
              const uint32_t row = (uint32_t)(half * kWarpTok + c + 8 * j + (lane & 7));
              stmatrix_x4_trans(ystage + row * 128 + ((ychunk ^ (row & 7)) << 4), pack2<BF16>(v[0][0], v[0][1]),
                                pack2<BF16>(v[1][0], v[1][1]), pack2<BF16>(v[2][0], v[2][1]),
                                pack2<BF16>(v[3][0], v[3][1]));
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int m = tt * TOK + col0 + c + 8 * j + 2 * t + e, n = f0 + sub * 32 + 8 * q + g;
                  if (m < p.M && n < f1) {
                    static_cast<uint16_t*>(p.y)[(int64_t)m * p.N + n] = float_to_elem<BF16>(v[q][e]);
                  }
                }
              }
            }
          }
        }
        if (rd == TOK / S::kTokRound - 1) {  // the accumulator is read out
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) {
              mbar_arrive_cluster(empty0 + buf * 8);
            } else {
              mbar_arrive(&empty_acc[buf]);
            }
          }
        }
        if constexpr (STAGED) {
          if (p.tma_y) fence_proxy_async_smem();
          named_bar_sync(1, kEpi * 32);
          if (!p.tma_y) {  // 16 bytes, eight features of a token, at a time
            const int chunks = p.wrows / 8;
            for (int i = etid; i < S::kTokRound * chunks; i += kEpi * 32) {
              const int tok = i / chunks, q = i - tok * chunks;
              const int m = tt * TOK + rd * S::kTokRound + tok, n = f0 + 8 * q;
              if (m < p.M && n < f1) {
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + (int64_t)m * p.N + n) =
                    *reinterpret_cast<const uint4*>(smem + S::kY + (q >> 3) * S::kYHalf + tok * 128 +
                                                    (((q & 7) ^ (tok & 7)) << 4));
              }
            }
          } else if (etid == 0) {
            for (int h = 0; h < p.wrows / 64; ++h) {
              const int f = f0 + h * 64, m = tt * TOK + rd * S::kTokRound;
              if (f < p.N && m < p.M) tma_store_2d(&ymap, smem + S::kY + h * S::kYHalf, f, m);
            }
            bulk_commit_group();
          }
        }
      }
    }
    if (STAGED && etid == 0) bulk_wait_group<0>();
  }

  // A wait ran out: of the copies asked for, those of stages whose barrier was
  // never armed cannot be waited for. They land within microseconds; nobody
  // leaves, or uses the ring, for a millisecond.
  if (*abort_flag) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }

  if constexpr (SPLIT) {
    // Every CTA's MMAs are done, so every ring is idle: here it takes this CTA's
    // sums [TOK][kRows + 4], and behind them the others' of its slice [CTA][slice][kRows + 4].
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    int* const mine = reinterpret_cast<int*>(smem);
    int* const theirs = mine + TOK * (kSumBytes / 4);
    static_assert(2 * TOK * kSumBytes <= (uint32_t)S::NS * S::kStage, "both in the ring");
    if (warp >= 3) {
      const int sub = warp & 3, g = lane >> 2, t = lane & 3;
      for (int c = ((warp - 3) >> 2) * 32; c < TOK; c += 64) {
        uint32_t r0[16], r1[16];
        const uint32_t acc = tmem + ((uint32_t)(sub * 32) << 16) + c;
        tmem_ld_16x256b_x4(acc, r0);
        tmem_ld_16x256b_x4(acc + (16u << 16), r1);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // token c + 8 (j / 2) + 2 t + j % 2, rows g, g + 8, g + 16, g + 24
          int* at = mine + (c + 8 * (j >> 1) + 2 * t + (j & 1)) * (kSumBytes / 4) + sub * 32 + g;
          const int e = 4 * (j >> 1) + (j & 1);
          at[0] = (int)r0[e];
          at[8] = (int)r0[e + 2];
          at[16] = (int)r1[e];
          at[24] = (int)r1[e + 2];
        }
      }
      fence_proxy_async_smem();
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < p.split; ++i) {
        const int to = (krank + i) % p.split;  // its slot for this CTA: the others in order
        const int at = krank < to ? krank : krank - 1;
        bulk_copy_s2cluster(dsmem_map(smem_u32(theirs) + at * slice * kSumBytes, to),
                            smem_u32(mine) + to * slice * kSumBytes, slice * kSumBytes, dsmem_map(smem_u32(sums), to));
      }
    }
    mbar_wait(sums, 0, p.status, 215, nullptr);
    if (p.pdl_x) pdl_wait_prior_grids();
    int wt, tt;
    gemm_unit(p, cid, wt, tt);
    const int f0 = wt * p.wrows, f1 = f0 + p.wrows < p.N ? f0 + p.wrows : p.N;
    const bool has_bias = p.bias_dtype != NSQ_DTYPE_NONE;
    for (int i = threadIdx.x; i < slice * kRows; i += kGemmThreads) {
      const int row = i % kRows, tok = i / kRows, n = f0 + row, m = tt * TOK + krank * slice + tok;
      if (n >= f1 || m >= p.M) continue;
      int sum = mine[(krank * slice + tok) * (kSumBytes / 4) + row];
      for (int r = 0; r < p.split - 1; ++r) sum += theirs[(r * slice + tok) * (kSumBytes / 4) + row];
      float v = (float)sum * p.xscale[m] * __ldg(p.wscale + n);
      if (has_bias) v += load_bias(p.bias, p.bias_dtype, n);
      static_cast<uint16_t*>(p.y)[(int64_t)m * p.N + n] = float_to_elem<BF16>(v);
    }
  }

  __syncthreads();
  tc_fence_before();
  if constexpr (CG == 2 || SPLIT) cluster_sync_all();  // SPLIT: every copy out of this CTA has landed
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) {
      tmem_dealloc_pair(tmem, S::kTmemCols);
    } else {
      tmem_dealloc(tmem, S::kTmemCols);
    }
  }
}

template <int CG, int TOK, bool BF16, bool STAGED, bool SPLIT = false>
cudaError_t launch_gemm(const CUtensorMap& xmap, const CUtensorMap& wmap, const CUtensorMap& ymap, const GemmParams& p,
                        cudaStream_t stream) {
  using S = GemmShape<CG, TOK>;
  auto kern = int8_gemm_kernel<CG, TOK, BF16, STAGED, SPLIT>;
  cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kern), S::kAlloc);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)p.num_w * p.num_t, most = num_sms() / CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(SPLIT ? units * p.split : CG * (units < most ? units : most)));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = S::kAlloc;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (CG == 2 || SPLIT) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = SPLIT ? p.split : 2;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.pdl_x) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, xmap, wmap, ymap, p);
}

template <int CG, int TOK>
int run_gemm(const Int8Args& a, int wrows, int split, cudaStream_t stream) {
  using S = GemmShape<CG, TOK>;
  const bool staged = split == 1 && a.N % 8 == 0, tma_y = staged && wrows % 64 == 0;
  CUtensorMap xmap, wmap, ymap;
  if (encode_tensor_map_2d(&xmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<int8_t*>(a.x), a.K, a.M, a.K, kBK,
                           S::kXRows, CU_TENSOR_MAP_SWIZZLE_128B) != CUDA_SUCCESS ||
      encode_tensor_map_2d(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<int8_t*>(a.w), a.K, a.N, a.K, kBK, wrows,
                           CU_TENSOR_MAP_SWIZZLE_128B) != CUDA_SUCCESS) {
    return NSQ_ECUDA;
  }
  ymap = xmap;
  if (tma_y && encode_tensor_map_2d(&ymap,
                                     a.y_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.y,
                                     a.N, a.M, (uint64_t)a.N * 2, 64, S::kTokRound,
                                     CU_TENSOR_MAP_SWIZZLE_128B) != CUDA_SUCCESS) {
    return NSQ_ECUDA;
  }
  GemmParams p{};
  p.xscale = a.xscale;
  p.wscale = a.wscale;
  p.bias = a.bias;
  p.bias_dtype = a.bias ? a.bias_dtype : NSQ_DTYPE_NONE;
  p.y = a.y;
  p.status = device_status_ptr();
  p.M = a.M;
  p.N = a.N;
  p.wrows = wrows;
  p.tma_y = tma_y;
  p.split = split;
  p.num_w = (a.N + CG * wrows - 1) / (CG * wrows);
  p.num_t = (a.M + TOK - 1) / TOK;
  p.num_kb = (a.K + kBK - 1) / kBK;
  p.num_st = (p.num_kb + kKps - 1) / kKps;
  p.pdl_x = a.after_quantize || pdl_enabled();
  p.withhold = test_withhold();
  if ((int64_t)p.num_w * p.num_t > 0x3FFFFFFF) return NSQ_ENOTSUP;
  cudaError_t e = cudaErrorInvalidValue;  // (pairs have no split form)
  if (split > 1) {
    if constexpr (CG == 1) {
      e = a.y_bf16 ? launch_gemm<1, TOK, true, false, true>(xmap, wmap, ymap, p, stream)
                   : launch_gemm<1, TOK, false, false, true>(xmap, wmap, ymap, p, stream);
    }
  } else if (staged) {
    e = a.y_bf16 ? launch_gemm<CG, TOK, true, true>(xmap, wmap, ymap, p, stream)
                 : launch_gemm<CG, TOK, false, true>(xmap, wmap, ymap, p, stream);
  } else {
    e = a.y_bf16 ? launch_gemm<CG, TOK, true, false>(xmap, wmap, ymap, p, stream)
                 : launch_gemm<CG, TOK, false, false>(xmap, wmap, ymap, p, stream);
  }
  return e == cudaSuccess ? NSQ_OK : NSQ_ECUDA;
}

}  // namespace

// The cheapest tile by an estimate in ns (measured on B200): for every wave of
// tiles the longer of a CTA's k-blocks (32, 64 or 128 tokens: 170, 205, 265
// each; CTA pairs of 256 x 256: 385) and its epilogue (900, 1300, 2150; 4000),
// once more the epilogue, and 6 us for a K split (cluster launch, exchange, no
// steady state of the ring: worth it for long K alone, 100 x 20000 -> 640 44 ->
// 13 us). Clusters of 4 at most, and 128 CTAs in them: more are not sure to run
// at once on 8 groups of 16 to 18 SMs. Rows of a tile: all that an even deal
// leaves.
int run_int8_gemm(const Int8Args& a, cudaStream_t stream) {
  const int64_t sms = num_sms(), kb = (a.K + kBK - 1) / kBK, num_st = (kb + kKps - 1) / kKps;
  auto estimate = [](int64_t waves, int64_t blocks, int64_t ns, int64_t epilogue) {
    return waves * (blocks * ns > epilogue ? blocks * ns : epilogue) + epilogue;
  };
  int64_t best = INT64_MAX;
  int tok_b = 0, rows_b = kRows, split_b = 1;
  for (int tok = 32; tok <= 128; tok *= 2) {
    const int64_t num_t = (a.M + tok - 1) / tok;
    const int64_t ns = tok == 32 ? 170 : tok == 64 ? 205 : 265, epilogue = tok == 32 ? 900 : tok == 64 ? 1300 : 2150;
    for (int split = 1; split <= 4 && split <= num_st; split *= 2) {
      // weight tiles that run at once
      const int64_t room = (split > 1 && sms > 128 ? 128 : sms) / (num_t * split);
      int64_t rows = kRows;
      if (room > 0) {
        const int64_t waves = (a.N + room * kRows - 1) / (room * kRows);
        rows = ((a.N + room * waves - 1) / (room * waves) + 7) / 8 * 8;
        if (rows < 32) rows = 32;
      }
      const int64_t tiles = num_t * ((a.N + rows - 1) / rows);
      if (split > 1 && (tiles * split > 128 || tiles * split > sms)) continue;
      const int64_t cost = estimate((tiles * split + sms - 1) / sms, (kb + split - 1) / split, ns, epilogue) +
                           (split > 1 ? 6000 : 0);
      if (cost < best) {
        best = cost;
        tok_b = tok;
        rows_b = (int)rows;
        split_b = split;
      }
    }
  }
  const int64_t pairs = (int64_t)((a.N + 255) / 256) * ((a.M + 255) / 256);
  if (estimate((pairs + sms / 2 - 1) / (sms / 2), kb, 385, 4000) < best) return run_gemm<2, 256>(a, kRows, 1, stream);
  return tok_b == 32   ? run_gemm<1, 32>(a, rows_b, split_b, stream)
         : tok_b == 64 ? run_gemm<1, 64>(a, rows_b, split_b, stream)
                       : run_gemm<1, 128>(a, rows_b, split_b, stream);
}

}  // namespace nsq
