// The 8-bit key/value cache: rows quantised as they are written, read back,
// and decode attention over the codes.
//
// The cache is a pool of pages; row (page, offset, head) holds head_dim codes
// and one fp32 scale:
//   s = max|row| / 127 (int8) or / 448 (e4m3), 1 where that is 0;
//   code = rint(row / s) or e4m3(row / s), nearest-even; value = code * s.
// A row that holds a NaN or an infinity gets a scale of that kind and reads
// back as NaN. Strides are free (head_dim is contiguous), so token-major and
// head-major pools both work.
#include "nsq_common.cuh"
#include "nsq_internal.h"
#include "nsq_rows8.cuh"

namespace nsq {

namespace {

struct KvWrite {
  KvCache c;
  const void *k, *v;
  int64_t k_stride[2], v_stride[2];  // token, head
  const int64_t* slots;
  int T;
  FastDiv head_div, page_div;
  DevStatus* status;
  bool pdl;
};

struct KvRead {
  KvCache c;
  void *k, *v;  // [T, kv_heads, head_dim]
  const int64_t* slots;
  int T;
  FastDiv head_div, page_div;
  DevStatus* status;
  bool pdl;
};

struct KvAttn : KvAttnArgs {
  int group, head_blocks, slot_heads;
  int least_log2;  // units of the smallest share
  int abreast;  // workers of a team: neighbouring items of a sequence (kv heads, blocks of query heads)
  int teams;  // in the grid
  FastDiv page_div, abreast_div;
  bool k_swap, v_swap;  // the tensor map has head before token
  float scale_log2;
  float* partial;
  int4* meta;
  DevStatus* status;
  bool pdl;
  bool withhold;  // failure-path test hook: the first worker's first stage never completes
};

// Records the first bad value in a device-side argument (tag 200 a written
// slot, 201 a read one, 202 a page, 203 a length) in the status word.
__device__ __forceinline__ void report(DevStatus* st, uint32_t where) {
  if (st != nullptr && atomicCAS(&st->code, 0u, (unsigned)NSQ_EINVAL) == 0u) {
    st->where = where;
    st->block = blockIdx.x;
  }
}

// Strides are below 2^32 elements (checked on the host).
__device__ __forceinline__ int64_t mul_wide(uint32_t a, int64_t stride) {
  return (int64_t)((uint64_t)a * (uint32_t)stride);
}

// ---------------------------------------------------------------------------
// Write and read
// ---------------------------------------------------------------------------

// Four codes (bytes of w) -> fp16 pairs (b0, b1) and (b2, b3), exact.
template <bool FP8>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FP8) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // 1024 + (code + 128) in the low mantissa bits, minus 1152
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = prmt(u, 0x64646464u, 0x4140), b = prmt(u, 0x64646464u, 0x4342);
    const __half2 c = __floats2half2_rn(1152.f, 1152.f);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), c);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), c);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// Two times eight elements of a row per lane, LPR lanes per row (LPR * 16 >=
// head_dim; LPR * 8 elements apart, so that the lanes of a row read and write
// whole sectors), k and v of one place together and several places at a time:
// the place is worked out once for 32 elements a lane, and the loads are in
// flight together. DRAM bounds both kernels, next the instructions (writing:
// 70% of the issue slots at 5 TB/s).
constexpr int kAtOnce = 2;

struct KvPlace {
  uint32_t page, off, tok, head;
  bool in;  // a place of the pool
};
template <typename P>
__device__ __forceinline__ KvPlace kv_place(const P& p, uint32_t row, uint32_t rows, uint32_t tag, bool tell) {
  KvPlace a;
  a.tok = fdiv(row, p.head_div);
  a.head = row - a.tok * (uint32_t)p.c.kv_heads;
  const int64_t slot = row < rows ? __ldg(p.slots + a.tok) : -1;
  a.in = slot >= 0 && slot < (int64_t)p.c.num_pages * p.c.page_size;
  if (!a.in && slot >= 0 && tell) report(p.status, tag);
  a.page = a.in ? fdiv((uint32_t)slot, p.page_div) : 0;
  a.off = a.in ? (uint32_t)slot - a.page * (uint32_t)p.c.page_size : 0;
  return a;
}
__device__ __forceinline__ int64_t kv_at(const KvPlace& a, const int64_t (&stride)[3]) {
  return mul_wide(a.page, stride[0]) + mul_wide(a.off, stride[1]) + mul_wide(a.head, stride[2]);
}

template <bool FP8, bool BF16, int LPR>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvWrite p) {
  if (p.pdl) pdl_wait_prior_grids();
  const int sub = threadIdx.x % LPR;
  const uint32_t rows = (uint32_t)p.T * (uint32_t)p.c.kv_heads;
  const bool in_row[2] = {sub * 8 < p.c.head_dim, (LPR + sub) * 8 < p.c.head_dim};
  const uint32_t step = gridDim.x * (256 / LPR);
  // whole warps stay in the loop: the shuffles below are all lanes'
  for (uint32_t r0 = blockIdx.x * (256 / LPR) + (threadIdx.x & ~31u) / LPR; r0 < rows; r0 += kAtOnce * step) {
    KvPlace a[kAtOnce];
    uint4 x[kAtOnce][2][2];  // [place][k, v][8 elements]
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t r = r0 + (threadIdx.x & 31) / LPR + i * step;
      a[i] = kv_place(p, r, rows, 200, sub == 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int64_t at = j ? a[i].tok * p.v_stride[0] + a[i].head * p.v_stride[1]
                             : a[i].tok * p.k_stride[0] + a[i].head * p.k_stride[1];
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(j ? p.v : p.k) + at) + sub;
#pragma unroll
        for (int c = 0; c < 2; ++c) x[i][j][c] = in_row[c] && r < rows ? __ldg(src + c * LPR) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t m = abs_max2(abs_max2(0, x[i][j][0]), x[i][j][1]);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!a[i].in) continue;
        const float s = row_scale<FP8>(abs_max_value<BF16>(m));
        const RowDiv dv(s);
        uint8_t* dst = j ? p.c.v + kv_at(a[i], p.c.v_stride) : p.c.k + kv_at(a[i], p.c.k_stride);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (in_row[c]) reinterpret_cast<uint2*>(dst)[c * LPR + sub] = row_codes8<FP8, BF16>(dv, x[i][j][c]);
        }
        if (sub == 0) *(j ? p.c.vs + kv_at(a[i], p.c.vs_stride) : p.c.ks + kv_at(a[i], p.c.ks_stride)) = s;
      }
    }
  }
}

// Four codes times s, as four elements.
template <bool FP8, bool BF16>
__device__ __forceinline__ uint2 values4(uint32_t w, float s) {
  uint32_t h[2], o[2];
  codes_to_f16<FP8>(w, h[0], h[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    if constexpr (BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * s, f.y * s);
      o[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(f.x * s, f.y * s);
      o[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return make_uint2(o[0], o[1]);
}

// The inverse: code * s rounded once to the output type. Rows of a negative
// or out-of-range slot read as zero.
template <bool FP8, bool BF16, int LPR>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvRead p) {
  if (p.pdl) pdl_wait_prior_grids();
  const int sub = threadIdx.x % LPR;
  const bool in_row[2] = {sub * 8 < p.c.head_dim, (LPR + sub) * 8 < p.c.head_dim};
  if (!in_row[0]) return;
  const uint32_t rows = (uint32_t)p.T * (uint32_t)p.c.kv_heads;
  const uint32_t step = gridDim.x * (256 / LPR);
  for (uint32_t r0 = blockIdx.x * (256 / LPR) + threadIdx.x / LPR; r0 < rows; r0 += kAtOnce * step) {
    KvPlace a[kAtOnce];
    uint2 c[kAtOnce][2][2];  // [place][k, v][8 codes]
    float s[kAtOnce][2];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) a[i] = kv_place(p, r0 + i * step, rows, 201, sub == 0);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        c[i][j][0] = c[i][j][1] = make_uint2(0, 0);
        s[i][j] = 0.f;
        if (a[i].in) {
          const uint8_t* src = j ? p.c.v + kv_at(a[i], p.c.v_stride) : p.c.k + kv_at(a[i], p.c.k_stride);
          c[i][j][0] = reinterpret_cast<const uint2*>(src)[sub];
          if (in_row[1]) c[i][j][1] = reinterpret_cast<const uint2*>(src)[LPR + sub];
          s[i][j] = *(j ? p.c.vs + kv_at(a[i], p.c.vs_stride) : p.c.ks + kv_at(a[i], p.c.ks_stride));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t r = r0 + i * step;
      if (r >= rows) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(j ? p.v : p.k) + (int64_t)r * p.c.head_dim);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!in_row[h]) continue;
          const uint2 lo = values4<FP8, BF16>(c[i][j][h].x, s[i][j]), hi = values4<FP8, BF16>(c[i][j][h].y, s[i][j]);
          dst[h * LPR + sub] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Decode attention
// ---------------------------------------------------------------------------
//
// One query token per sequence: out[h] = sum_t p[t] v[t] / sum_t p[t],
// p[t] = exp2(s[t] - m), s[t] = scale * log2(e) * q . k[t], m the running
// maximum. Bound by reading the codes once; so
//   * every warp works alone on its share of the tokens: it keeps a ring of
//     32-token stages in shared memory, filled ahead by TMA (one box per 16
//     tokens of a page and head) or, where pages are not multiples of 16
//     tokens, by 16-byte asynchronous copies; the ring runs on from one
//     sequence and head to the next, and no warp waits for another;
//   * mma.m16n8k16 with 16 tokens as rows for q . k and 16 dims as rows for
//     p . v; the query heads that share the kv head are the 8 columns. The
//     codes are read in the swizzled tile without bank conflicts (ldmatrix for
//     k, 16-byte reads for v) and become fp16 in registers, exactly;
//   * q enters the MMA as fp16: fp16 as it is, bf16 scaled per head by a power
//     of two that takes its largest near the end of fp16's range, exact for
//     every element within 2^-31 of that. Scores, maxima and sums are fp32;
//   * the fp16 weights of p . v are p * vs relative to a reference m' of their
//     own, log2 of their largest less 12: the largest lies in [2^12, 2^15], so
//     one down to 2^-26 of it keeps fp16's 11 bits (off by 2^-11 of itself at
//     most) and smaller ones are off by 2^-37 of the largest. fp16 because the
//     codes are exact in it and the MMA wants one type; it is what bounds the
//     accuracy. The denominator is summed in fp32 from unrounded terms. At the
//     end the accumulator is multiplied by exp2(m' - m). Both references follow
//     lazily, when a score passes m by 8 or a weight passes 2^15: rescaling and
//     the maximum over the warp are rare, and fp16 and fp32 have the room;
//   * work is cut into units of 32 tokens of one item (sequence, kv head) and
//     dealt evenly to the warps on the device, from seq_lens: long and ragged
//     batches fill the machine alike. Warps are dealt to in teams of up to 32, a
//     warp for each kv head, which walk the same tokens side by side: in a
//     token-major pool they read whole rows of memory between them (48 x 8192,
//     8 kv heads of 128: 146 us, on their own 178). A warp's range covers whole
//     items and at most two cut ones; those go to the workspace as fp32
//     partials, and a second kernel joins them in order. Where no sequence can
//     hold more than 128 tokens an item is one unit: nothing is cut and one
//     launch does.
// Measured (8 kv heads of 128, 4 query heads each, e4m3, bf16 q, the join
// included): 48 x 8192 tokens 146 us, 5.7 TB/s; 64 x 2048 58 us, 4.7 TB/s;
// 1 x 131001 60 us; 1 x 2048 10.5 us; 1 x 40 (2 kv heads of 64, int8, fp16 q)
// 6.6 us. Of the 58 us 2 pass before the first copy is issued, 43 are the
// stream at the rate of a plain copy, about 7 the last warps of an even deal
// (their rates differ by 10%) and 4 the join with its launch.

constexpr int kAttnWarps = 4;
constexpr int kTile = 32;  // tokens of a stage
constexpr int kWhole = 4;  // stages of an item that is not cut
constexpr int kHeads = 8;  // query heads of an item: the columns of an MMA

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kNoMax = -3e38f;  // below every score: exp2(x - kNoMax) is 0 for a masked x, and nothing is NaN

constexpr float kLift = 12.f;    // log2 of the weight that sets a reference
constexpr float kLeast = 126.f;  // mm is at least m - kLeast, so that weight_factor stays in fp32's range
// 2^(m - mm): what turns exp2(x - m) * vs into a weight relative to mm (0 while there is none)
__device__ __forceinline__ float weight_factor(float m, float mm) { return mm == kNoMax ? 0.f : ex2(m - mm); }
// acc / sum * 2^(mm - m): the output of a head whose weights of v were taken
// relative to mm and whose denominator relative to m (0 for an empty row). The
// sum of n terms goes first and the power in two steps, so that nothing on
// the way leaves fp32's range where the output does not.
__device__ __forceinline__ float finish(float acc, float sum, float mm, float m) {
  if (sum == 0.f) return 0.f;
  const float half = ex2(0.5f * (mm - m));
  return acc / sum * half * half;
}
__device__ __forceinline__ float head_lse(float sum, float m) {
  return sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.69314718055994531f;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// Asynchronous copies to shared memory; with bytes = 0 the place is zeroed and nothing is read.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// One arrival on the barrier when this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Tokens a sequence holds: n of seq_lens clamped to what its page-table row can name.
__device__ __forceinline__ int seq_tokens(const KvAttn& p, int n, bool tell) {
  if (n < 0 || n > p.capacity) {
    if (tell) report(p.status, 203);
    n = n < 0 ? 0 : p.capacity;
  }
  return n;
}
// a / b; the 32-bit division takes a fraction of the other's time
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// Units of an item: its stages, or 1 where items are not cut.
__device__ __forceinline__ int item_units(const KvAttn& p, int n) {
  return n <= kTile || p.meta == nullptr ? 1 : (n + kTile - 1) / kTile;
}

// A warp's ring: stages of 32 tokens, k then v, each as two 16-token tiles of
// HALVES x 16 rows of RB bytes (swizzled in RB-byte rows as TMA does), the 64
// scales and a mask of the tokens to attend to.
constexpr int kScaleBytes = 272;
template <int DP>
struct AttnShape {
  static constexpr int RB = DP < 128 ? DP : 128;  // bytes of a tile row
  static constexpr int HALVES = DP / RB;
  static constexpr int kTileBytes = 16 * DP;
  static constexpr int kStage = 4 * kTileBytes;
  static constexpr int kStages = DP == 64 ? 4 : 2;
  static constexpr int kScale = kAttnWarps * kStages * kStage;
  static constexpr int kBar = kScale + kAttnWarps * kStages * kScaleBytes;
  static constexpr int kAlloc = kBar + kAttnWarps * kStages * 8 + 1024;
  static constexpr int kCtas = 227 * 1024 / (kAlloc + 1024);
  static constexpr int kPerSm = kCtas < 3 ? kCtas : 3;
};

// A worker's place: stage s (of 32 tokens) of item (b, kh), in the segment of
// `cnt` units from unit tu that ends before stage s_end; `left` units to go,
// the segment's included.
struct Cursor {
  int b, kh, n, nu, tu, cnt, s, s_end;
  long long left;
  __device__ __forceinline__ void segment() {
    cnt = (long long)(nu - tu) < left ? nu - tu : (int)left;
    s = tu;
    s_end = nu == 1 && n > kTile ? (n + kTile - 1) / kTile : tu + cnt;
  }
  // the next item (there is one: left > cnt)
  __device__ __forceinline__ void next(const KvAttn& p, int kh_n) {
    left -= cnt;
    tu = 0;
    kh += p.abreast;
    if (kh >= kh_n) {
      kh -= kh_n;
      ++b;
      n = seq_tokens(p, __ldg(p.seq_lens + b), false);
      nu = item_units(p, n);
    }
    segment();
  }
};

// Place of 16-byte chunk c of tile row r
template <int RB>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)(r * RB + ((c ^ (RB == 128 ? (r & 7) : ((r >> 1) & 3))) << 4));
}
// Token of MMA row i (of 16): the identity, or for 64-byte rows bits 0 and 1
// exchanged, so that the v reads of a warp fall into different banks.
template <int RB>
__device__ __forceinline__ int row_token(int i) {
  return RB == 128 ? i : (i & 12) | ((i & 1) << 1) | ((i >> 1) & 1);
}

template <int DP, bool FP8, bool BF16, bool TMA>
__global__ void __launch_bounds__(kAttnWarps * 32, AttnShape<DP>::kPerSm) kv_attn_kernel(
    const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const KvAttn p) {
  using S = AttnShape<DP>;
  constexpr int RB = S::RB, HALVES = S::HALVES;
  constexpr int KCH = RB / 16;     // 16-byte chunks of a tile row
  constexpr int MT = DP / 16;      // 16-dim tiles of the output
  constexpr int VW = RB / 32;      // words of a v row per lane and half
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ long long s_scan[kAttnWarps];
  __shared__ long long s_excl[kAttnWarps * 32];  // units ahead of each thread's sequences

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBar) + warp * S::kStages;
  const uint32_t ring = smem_u32(smem) + warp * S::kStages * S::kStage;
  const uint32_t ring_sc = smem_u32(smem) + S::kScale + warp * S::kStages * kScaleBytes;  // scales, mask
  if (p.pdl) pdl_wait_prior_grids();
  const int vpt = (p.B + kAttnWarps * 32 - 1) / (kAttnWarps * 32);  // sequences of a thread
  const int n_first = tid * vpt < p.B ? __ldg(p.seq_lens + tid * vpt) : 0;  // on its way during the set-up
  // a phase: the lanes' copies, and one arrival of lane 0 (TMA: with the bytes)
  if (lane < S::kStages) mbar_init(&full[lane], 33 + (p.withhold && tid == 0 && blockIdx.x == 0));
  fence_barrier_init();
  if (TMA && tid == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_launch_dependents();  // the join's blocks may queue up behind this grid's; they wait for its end

  // ---- deal the units: each warp is a worker, each team of workers has its share of the batch's total ----
  const int kh_n = p.c.kv_heads * p.head_blocks;
  const int rows_n = kh_n / p.abreast;  // rows of items that a team works on side by side
  long long mine = 0;
  for (int i = 0; i < vpt; ++i) {
    const int b = tid * vpt + i;
    if (b >= p.B) break;
    const int n = seq_tokens(p, i == 0 ? n_first : __ldg(p.seq_lens + b), blockIdx.x == 0);
    mine += (long long)item_units(p, n) * rows_n;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  long long total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  s_excl[tid] = before + incl - mine;
  // dealt so that every worker has a share, an item's teams are neighbours,
  // and the first workers are one to a block
  const long long most = total >> p.least_log2 > 1 ? total >> p.least_log2 : 1;
  const int teams = most < p.teams ? (int)most : p.teams;
  const int me = warp * gridDim.x + blockIdx.x, team = fdiv(me, p.abreast_div);
  __syncthreads();  // the last one: from here on every warp is on its own
  if (team >= teams) return;
  // the first `extra` teams have share + 1 units, the others share
  const long long share = quotient(total, teams);
  const int extra = (int)(total - share * teams);
  const long long u0 = share * team + (team < extra ? team : extra);
  Cursor cur;  // what is worked on
  {
    int lo = -1;  // last thread with s_excl <= u0
#pragma unroll
    for (int i = 0; i < kAttnWarps; ++i) lo += __popc(__ballot_sync(0xffffffffu, s_excl[32 * i + lane] <= u0));
    long long rel = u0 - s_excl[lo];
    cur.b = lo * vpt;
    for (;;) {
      cur.n = seq_tokens(p, __ldg(p.seq_lens + cur.b), false);
      cur.nu = item_units(p, cur.n);
      const long long nb = (long long)cur.nu * rows_n;
      if (rel < nb) break;
      rel -= nb;
      ++cur.b;
    }
    const int row = (int)quotient(rel, cur.nu);
    cur.kh = row * p.abreast + me - team * p.abreast;
    cur.tu = (int)(rel - (long long)row * cur.nu);
    cur.left = share + (team < extra ? 1 : 0);
    cur.segment();
  }
  Cursor ahead = cur;  // what is being fetched

  // Page of token tok of the sequence in `at` as its table has it, -1 past its
  // end. Used through pool_page: the wait for the load is there.
  auto page_of = [&](const Cursor& at, int tok, int& off) {
    int page = -1;
    off = 0;
    if (tok < at.n) {
      const uint32_t pi = fdiv((uint32_t)tok, p.page_div);
      off = tok - (int)pi * p.c.page_size;
      page = __ldg(p.table + at.b * p.table_stride + pi);
    }
    return page;
  };
  // The page, or -1 if it is not one of the pool (recorded for a token that the
  // sequence holds): such tokens are never read.
  auto pool_page = [&](int page, bool held) {
    if ((uint32_t)page < (uint32_t)p.c.num_pages) return page;
    if (held) report(p.status, 202);
    return -1;
  };
  // TMA: lane j holds the page of 16-token tile 32 k + j of the item being
  // fetched, for the batch k in use (pg_a) and the one after (pg_b), and that
  // of tile j of the next item (pg_n).
  int off_a = 0, pg_a = -1, pg_b = -1, pg_n = -1;
  bool more = true;  // stages to fetch
  auto tile_page = [&](const Cursor& at, int j) {
    int off;
    return page_of(at, 16 * j, off);
  };
  auto look_ahead = [&]() {  // pg_b and pg_n for the segment that `ahead` enters
    const int k = (2 * ahead.s) & ~31;
    pg_b = tile_page(ahead, k + 32 + lane);
    if (ahead.left > ahead.cnt) {
      Cursor nx = ahead;
      nx.next(p, kh_n);
      pg_n = tile_page(nx, lane);
    }
  };
  if constexpr (TMA) {
    pg_a = tile_page(ahead, ((2 * ahead.s) & ~31) + lane);
  }
  // looked: pg_b and pg_n are those of the segment, read after its second stage
  // (before, if they are needed): the ring's first stages go first
  bool entering = true, looked = false;

  // this lane's scale (lanes 0..15 of k, 16..31 of v) of the first token of page 0, for the head in `ahead`
  const float* sc_base = nullptr;
  uint32_t sc_page = 0, sc_tok = 0;
  int off = 0;  // offset in its page of the next stage's first token (TMA)
  auto enter = [&]() {  // `ahead` has entered a segment
    const int head = ahead.kh / p.head_blocks;
    const bool is_k = lane < 16;
    sc_page = (uint32_t)(is_k ? p.c.ks_stride[0] : p.c.vs_stride[0]);
    sc_tok = (uint32_t)(is_k ? p.c.ks_stride[1] : p.c.vs_stride[1]);
    sc_base = (is_k ? p.c.ks : p.c.vs) + head * (is_k ? p.c.ks_stride[2] : p.c.vs_stride[2]);
    if constexpr (TMA) {
      sc_base += (uint64_t)(lane & 15) * sc_tok;
      const int tok = ahead.s * kTile;
      off = tok - (int)fdiv((uint32_t)tok, p.page_div) * p.c.page_size;
    }
  };
  enter();

  auto fill = [&](int slot) {  // starts the copies of stage `ahead` and moves on
    const uint32_t dst = ring + slot * S::kStage;
    const int left = ahead.n - ahead.s * kTile;  // tokens from the stage's first to the end
    const int head = ahead.kh / p.head_blocks;
    int pg[2], of[2];  // page and offset: TMA, of a tile's first token; else of this lane's token
    if constexpr (TMA) {
      if (!entering && (ahead.s & 15) == 0) {
        pg_a = pg_b;
        pg_b = tile_page(ahead, 2 * ahead.s + 32 + lane);
      }
    } else {
      pg_a = pool_page(page_of(ahead, ahead.s * kTile + lane, off_a), lane < left);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (TMA) {
        pg[h] = pool_page(__shfl_sync(0xffffffffu, pg_a, (2 * ahead.s + h) & 31), 16 * h < left);
        of[h] = off;
        off = off + 16 == p.c.page_size ? 0 : off + 16;
      } else {
        pg[h] = __shfl_sync(0xffffffffu, pg_a, 16 * h + (lane & 15));
        of[h] = __shfl_sync(0xffffffffu, off_a, 16 * h + (lane & 15));
      }
    }
    if constexpr (TMA) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[slot], ((pg[0] >= 0) + (pg[1] >= 0)) * 2 * S::kTileBytes);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (pg[h] < 0) continue;
#pragma unroll
          for (int half = 0; half < HALVES; ++half) {
            const uint32_t at = dst + h * S::kTileBytes + half * 16 * RB;
            const int cd = half * RB;
            tma_load_4d(at, &kmap, &full[slot], cd, p.k_swap ? head : of[h], p.k_swap ? of[h] : head, pg[h]);
            tma_load_4d(at + 2 * S::kTileBytes, &vmap, &full[slot], cd, p.v_swap ? head : of[h],
                        p.v_swap ? of[h] : head, pg[h]);
          }
        }
      }
    } else {
      const uint8_t* kb = p.c.k + head * p.c.k_stride[2];
      const uint8_t* vb = p.c.v + head * p.c.v_stride[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll 4
        for (int x = lane; x < 16 * HALVES * KCH; x += 32) {
          const int row = (x / KCH) & 15, c = x % KCH, half = x / (16 * KCH);
          const int pr = __shfl_sync(0xffffffffu, pg_a, 16 * h + row);
          const uint32_t orow = __shfl_sync(0xffffffffu, off_a, 16 * h + row);
          const int d = half * RB + 16 * c;
          const bool ok = pr >= 0 && d < p.c.head_dim;
          const uint32_t at = dst + h * S::kTileBytes + half * 16 * RB + tile_at<RB>(row, c);
          const int64_t ko = mul_wide(pr, p.c.k_stride[0]) + mul_wide(orow, p.c.k_stride[1]) + d;
          const int64_t vo = mul_wide(pr, p.c.v_stride[0]) + mul_wide(orow, p.c.v_stride[1]) + d;
          cp_async16(at, ok ? kb + ko : p.c.k, ok ? 16 : 0);
          cp_async16(at + 2 * S::kTileBytes, ok ? vb + vo : p.c.v, ok ? 16 : 0);
        }
      }
    }
    // the scales, and which tokens there are
    uint32_t there = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = pg[h] >= 0 && 16 * h + (lane & 15) < left;
      const float* src = sc_base + (uint64_t)(uint32_t)pg[h] * sc_page + (uint64_t)(uint32_t)of[h] * sc_tok;
      cp_async4(ring_sc + slot * kScaleBytes + h * 128 + lane * 4, in ? src : p.c.ks, in ? 4 : 0);
      there |= (__ballot_sync(0xffffffffu, in) & 0xffffu) << (16 * h);
    }
    if (lane == 0) {
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(ring_sc + slot * kScaleBytes + 256), "r"(there) : "memory");
      if constexpr (!TMA) mbar_arrive(&full[slot]);
    }
    cp_async_arrive(&full[slot]);
    __syncwarp();  // the mask is the warp's own: seen by all lanes from here on
    if (TMA && !looked && (!entering || ahead.s + 1 == ahead.s_end || (ahead.s & 15) == 15)) {
      look_ahead();
      looked = true;
    }
    entering = false;
    if (++ahead.s == ahead.s_end) {
      more = ahead.left > ahead.cnt;
      if (more) {
        ahead.next(p, kh_n);
        entering = true;
        looked = false;
        pg_a = pg_n;
        enter();
      }
    }
  };

  // places in a tile: ldmatrix rows of k, and this lane's chunk of the four tokens of v
  const int krow = row_token<RB>(lane & 15);
  uint32_t v_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row_token<RB>(2 * t + (i & 1) + 8 * (i >> 1));
    v_at[i] = RB == 128 ? tile_at<RB>(r, g) : tile_at<RB>(r, g >> 1) + 8 * (g & 1);
  }

  uint32_t filled = 0, done = 0;  // stages
  for (; filled < S::kStages && more; ++filled) fill(filled % S::kStages);

  for (bool first = true;; first = false) {
    // ---- one segment of item (b, kh) ----
    const int b = cur.b;
    const int head = cur.kh / p.head_blocks;
    const int hb0 = (cur.kh - head * p.head_blocks) * kHeads;  // first query head of this block within the group
    // q as the B operand: lane (g, t) holds head g, dims 16 j + 4 t + 0..3 of every j
    uint32_t qf[MT][2];
    float sc[2];  // score scale of heads 2t, 2t + 1
    const int hl = hb0 + g;
    const uint16_t* qrow = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] +
                           (int64_t)(head * p.group + (hl < p.group ? hl : 0)) * p.q_stride[1];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int d = 16 * j + 4 * t;
      uint2 x = make_uint2(0, 0);
      if (hl < p.group && d < p.c.head_dim) x = __ldg(reinterpret_cast<const uint2*>(qrow + d));
      qf[j][0] = x.x;
      qf[j][1] = x.y;
    }
    if constexpr (BF16) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m = fmaxf(m, fabsf(elem_to_float<BF16>((uint16_t)qf[j][i])));
          m = fmaxf(m, fabsf(elem_to_float<BF16>((uint16_t)(qf[j][i] >> 16))));
        }
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // 2^-e takes the largest to [2^14, 2^15) (where it is below 2^-100 to [1, 2),
      // so that the score's scale 2^e stays normal), in two steps so that
      // neither factor leaves fp32's range
      int e = m > 0.f && m <= 3.4e38f ? ilogbf(m) : 0;
      if (e > -100) e -= 14;
      const float f1 = exp2f((float)(-e / 2)), f2 = exp2f((float)(-e - (-e / 2)));
#pragma unroll
      for (int j = 0; j < MT; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          qf[j][i] = pack_f16(elem_to_float<BF16>((uint16_t)qf[j][i]) * f1 * f2,
                              elem_to_float<BF16>((uint16_t)(qf[j][i] >> 16)) * f1 * f2);
        }
      }
      const float s = p.scale_log2 / f1 / f2;
      sc[0] = __shfl_sync(0xffffffffu, s, (2 * t) * 4);
      sc[1] = __shfl_sync(0xffffffffu, s, (2 * t + 1) * 4);
    } else {
      sc[0] = sc[1] = p.scale_log2;
    }

    float o[MT][4];
    // references m and m' (kNoMax: no term yet), 2^(m - m'), denominators (this lane's tokens)
    float mx[2], mv[2], vf[2], l[2];
#pragma unroll
    for (int j = 0; j < MT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    mx[0] = mx[1] = mv[0] = mv[1] = kNoMax;
    vf[0] = vf[1] = l[0] = l[1] = 0.f;

    auto step = [&](int slot) {
      const uint32_t kt = ring + slot * S::kStage, vt = kt + 2 * S::kTileBytes, st = ring_sc + slot * kScaleBytes;
      float s[2][4];
      const uint32_t there = __float_as_uint(lds_f32(st + 256));  // the tokens to attend to
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.f;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
#pragma unroll
          for (int c = 0; c < KCH; c += 2) {
            uint32_t r[4], a[4];
            ldmatrix_x4(kt + h * S::kTileBytes + half * 16 * RB + tile_at<RB>(krow, c + (lane >> 4)), r);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              codes_to_f16<FP8>(r[2 * j], a[0], a[2]);
              codes_to_f16<FP8>(r[2 * j + 1], a[1], a[3]);
              mma_16816<false>(s[h], a, qf[half * KCH + c + j][0], qf[half * KCH + c + j][1]);
            }
          }
        }
      }
      // scores x, relative to the reference m their exponentials
      float vs[2][2];
      bool over = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int tok = row_token<RB>(g) + 8 * r;
          const float ks = lds_f32(st + h * 128 + tok * 4);
          vs[h][r] = lds_f32(st + h * 128 + 64 + tok * 4);
#pragma unroll
          for (int e = 0; e < 2; ++e) s[h][2 * r + e] *= ks * sc[e];
        }
      }
      if (there != 0xffffffffu) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if ((there >> (16 * h + row_token<RB>(g) + 8 * r)) & 1) continue;
            s[h][2 * r] = s[h][2 * r + 1] = -INFINITY;
          }
        }
      }
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(fmaxf(s[0][e], s[0][2 + e]), fmaxf(s[1][e], s[1][2 + e]));
        over |= top[e] > mx[e] + 8.f;
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float a = top[e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
          if (a > mx[e]) {
            l[e] *= ex2(mx[e] - a);
            mx[e] = a;
            vf[e] = weight_factor(a, mv[e]);
          }
        }
      }
      float wt[2][4];
      over = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float big = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float x = ex2(s[h][2 * r + e] - mx[e]);
            l[e] += x;
            wt[h][2 * r + e] = x * (vs[h][r] * vf[e]);
            big = fmaxf(big, wt[h][2 * r + e]);
          }
        }
        over |= big > 32768.f || mx[e] - mv[e] > kLeast;  // the latter, too, while there is no reference
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < 2; ++r) v = fmaxf(v, s[h][2 * r + e] + lg2(vs[h][r]));
          }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
          v = fmaxf(v - kLift, mx[e] - kLeast);  // scales so small (subnormal ones are 0 to lg2) need no finer reference
          if (v > mv[e]) {
            const float f = ex2(mv[e] - v);
            mv[e] = v;
            vf[e] = weight_factor(mx[e], v);
#pragma unroll
            for (int j = 0; j < MT; ++j) o[j][e] *= f, o[j][2 + e] *= f;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              wt[h][2 * r + e] = ex2(s[h][2 * r + e] - mx[e]) * (vs[h][r] * vf[e]);
            }
          }
        }
      }
      uint32_t pb[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 2; ++r) pb[h][r] = movmatrix_trans(pack_f16(wt[h][2 * r], wt[h][2 * r + 1]));
      }
      // dims 2j, 2j + 1 of this lane's 16 (or 8) are rows g, g + 8 of output tile j
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t part = (there >> (16 * h)) & 0xffffu;
        if (part == 0) continue;
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          uint32_t v[4][VW];
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const uint32_t at = vt + h * S::kTileBytes + half * 16 * RB + v_at[i2];
            if constexpr (VW == 2) {
              const uint2 y = lds64(at);
              v[i2][0] = y.x, v[i2][1] = y.y;
            } else {
              const uint4 y = lds128(at);
              v[i2][0] = y.x, v[i2][1] = y.y, v[i2][2] = y.z, v[i2][3] = y.w;
            }
          }
          if (part != 0xffffu) {  // codes of tokens not held may be NaN, which a weight of 0 does not stop
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
              if (!((part >> row_token<RB>(2 * t + (i2 & 1) + 8 * (i2 >> 1))) & 1)) {
#pragma unroll
                for (int j = 0; j < VW; ++j) v[i2][j] = 0;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            uint32_t a[4], c[4];
            codes_to_f16<FP8>(prmt(v[0][j], v[1][j], 0x5140), a[0], a[1]);
            codes_to_f16<FP8>(prmt(v[2][j], v[3][j], 0x5140), a[2], a[3]);
            codes_to_f16<FP8>(prmt(v[0][j], v[1][j], 0x7362), c[0], c[1]);
            codes_to_f16<FP8>(prmt(v[2][j], v[3][j], 0x7362), c[2], c[3]);
            mma_16816<false>(o[half * (RB / 16) + 2 * j], a, pb[h][0], pb[h][1]);
            mma_16816<false>(o[half * (RB / 16) + 2 * j + 1], c, pb[h][0], pb[h][1]);
          }
        }
      }
    };

    for (; cur.s < cur.s_end; ++cur.s, ++done) {
      const int slot = done % S::kStages;
      const bool ok = mbar_wait(&full[slot], (done / S::kStages) & 1, p.status, 204, nullptr);
      if (!__all_sync(0xffffffffu, ok)) {  // recorded; the copies in flight land before the block can end
        for (; done < filled; ++done) {
          mbar_wait(&full[done % S::kStages], (done / S::kStages) & 1, nullptr, 0, nullptr);
        }
        return;
      }
      step(slot);
      __syncwarp();
      if (more) {
        fill(slot);
        ++filled;
      }
    }

    // ---- the segment's result: lane (g, t) holds heads 2t, 2t + 1 and the dims of its chunk ----
    const bool opens = cur.tu == 0, closes = cur.tu + cur.cnt == cur.nu;
    const bool whole = opens && closes;
    const long long slot = 2 * (long long)me + (first ? 0 : 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
      const int h = 2 * t + e;
      if (hb0 + h >= p.group) continue;
      const float m = mx[e], mm = mv[e], sum = l[e];
      const int64_t row = (int64_t)b * p.H + head * p.group + hb0 + h;
      float* ws = whole ? nullptr : p.partial + (slot * p.slot_heads + h) * (DP + 4);
      if (g == 0) {
        if (whole) {
          if (p.lse != nullptr) p.lse[row] = head_lse(sum, m);
        } else {
          *reinterpret_cast<float4*>(ws) = make_float4(m, mm, sum, 0.f);
        }
      }
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        const int d0 = half * RB + g * (RB / 8);
#pragma unroll
        for (int c = 0; c < RB / 64; ++c) {  // 8 dims at a time
          float y[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[2 * j] = o[half * (RB / 16) + 4 * c + j][e];
            y[2 * j + 1] = o[half * (RB / 16) + 4 * c + j][2 + e];
          }
          if (whole) {
            if (d0 + 8 * c < p.c.head_dim) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                w[j] = (uint32_t)float_to_elem<BF16>(finish(y[2 * j], sum, mm, m)) |
                       ((uint32_t)float_to_elem<BF16>(finish(y[2 * j + 1], sum, mm, m)) << 16);
              }
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.c.head_dim + d0 + 8 * c) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            *reinterpret_cast<float4*>(ws + 4 + d0 + 8 * c) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(ws + 8 + d0 + 8 * c) = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      }
    }
    // the worker that opens an item says whether it is cut, and then which slot
    // it used and which workers follow
    if (whole && p.meta != nullptr && lane == 0) p.meta[b * kh_n + cur.kh] = make_int4(-1, 0, 0, 0);
    if (opens && !closes && lane == 0) {
      // the item's last unit, and the team whose share holds it
      const long long unit = u0 + share + (team < extra ? 1 : 0) - cur.left + cur.nu - 1;
      const long long longer = extra * (share + 1);
      const int last = (int)(unit < longer ? quotient(unit, share + 1) : extra + quotient(unit - longer, share));
      p.meta[b * kh_n + cur.kh] = make_int4(last - team + 1, (int)slot, me, 0);
    }
    if (cur.left == cur.cnt) return;
    cur.next(p, kh_n);
  }
}

// Joins the partials of cut items: the slot that the opening worker named and
// the first slots of the workers after it, always in the same order, so
// results do not depend on timing. A pair (query head, item) is a warp's, or,
// from more than kJoinWarp partials on, all warps' of its block; with PAIRS =
// 1 (few pairs) a block has 32 dims of one pair. Consecutive pairs are different items,
// so one long item is spread over blocks.
constexpr int kJoinWarp = 16;
template <int DP, bool BF16, int PAIRS>
__global__ void __launch_bounds__(PAIRS == 1 ? 256 : 32 * PAIRS) kv_attn_join_kernel(const KvAttn p, int items) {
  constexpr int kJoinThreads = PAIRS == 1 ? 256 : 32 * PAIRS;
  // threads that share a partial's row (or 32 dims of it), four dims each
  constexpr int LANES = PAIRS == 1 ? 8 : DP / 4;
  constexpr int KG = kJoinThreads / LANES;        // partials read side by side
  constexpr int V4 = DP > 128 ? DP / 128 : 1;     // four-dim pieces of a row per lane, in the one-warp form
  constexpr int64_t kRow = DP + 4;
  __shared__ float4 s_part[KG][LANES];
  __shared__ float s_w[kJoinThreads], s_red[3][kJoinThreads / 32];
  pdl_wait_prior_grids();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kh_n = p.c.kv_heads * p.head_blocks;
  const int64_t slot_row = p.slot_heads * kRow;
  // item and query head (of its block) of a pair; partials to join (0: none)
  auto look = [&](int pair, int& item, int& h, int4& me) -> int {
    h = pair / items;
    item = pair - h * items;
    if (h >= p.slot_heads || ((item % kh_n) % p.head_blocks) * kHeads + h >= p.group) return 0;
    me = __ldg(p.meta + item);
    // a worker whose wait ran out leaves what it should have written as it was:
    // nothing that the grid cannot have written is followed
    const int workers = p.teams * p.abreast;
    const bool in_grid = me.x <= p.teams && (uint32_t)me.y < 2u * (uint32_t)workers && (uint32_t)me.z < (uint32_t)workers;
    return me.x > 0 && in_grid && me.z + (me.x - 1) * p.abreast < workers ? me.x : 0;
  };
  auto store = [&](int item, int h, int d4, float4 acc, float sum, float mm, float m) {
    const int b = item / kh_n, kh = item - b * kh_n;
    const int head = kh / p.head_blocks;
    const int64_t row = (int64_t)b * p.H + head * p.group + (kh - head * p.head_blocks) * kHeads + h;
    if (4 * d4 < p.c.head_dim) {
      const uint32_t lo = (uint32_t)float_to_elem<BF16>(finish(acc.x, sum, mm, m)) |
                          ((uint32_t)float_to_elem<BF16>(finish(acc.y, sum, mm, m)) << 16);
      const uint32_t hi = (uint32_t)float_to_elem<BF16>(finish(acc.z, sum, mm, m)) |
                          ((uint32_t)float_to_elem<BF16>(finish(acc.w, sum, mm, m)) << 16);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.c.head_dim + 4 * d4) = make_uint2(lo, hi);
    }
    if (d4 == 0 && p.lse != nullptr) p.lse[row] = head_lse(sum, m);
  };

  int item, h;
  int4 me;
  const int count = look(blockIdx.x * PAIRS + (PAIRS == 1 ? 0 : warp), item, h, me);
  if (PAIRS > 1 && count > 0 && count <= kJoinWarp) {
    auto part = [&](int k) {
      return p.partial + (k == 0 ? (int64_t)me.y : 2 * ((int64_t)me.z + k * p.abreast)) * slot_row + h * kRow;
    };
    float4 x0 = make_float4(kNoMax, kNoMax, 0.f, 0.f);
    if (lane < count) x0 = *reinterpret_cast<const float4*>(part(lane));
    float4 x[kJoinWarp][V4];  // all in flight at once
#pragma unroll
    for (int k = 0; k < kJoinWarp; ++k) {
#pragma unroll
      for (int v = 0; v < V4; ++v) {
        x[k][v] = k < count && lane + 32 * v < LANES
                      ? *reinterpret_cast<const float4*>(part(k) + 4 + 4 * (lane + 32 * v))
                      : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float m = x0.x, mm = x0.y;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    }
    m = __shfl_sync(0xffffffffu, m, 0);
    mm = __shfl_sync(0xffffffffu, mm, 0);
    float sum = x0.z * ex2(x0.x - m);
    const float w0 = ex2(x0.y - mm);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float4 acc[V4];
#pragma unroll
    for (int v = 0; v < V4; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kJoinWarp; ++k) {
      const float f = __shfl_sync(0xffffffffu, w0, k);
#pragma unroll
      for (int v = 0; v < V4; ++v) {
        if (k < count) {
          acc[v].x = fmaf(x[k][v].x, f, acc[v].x);
          acc[v].y = fmaf(x[k][v].y, f, acc[v].y);
          acc[v].z = fmaf(x[k][v].z, f, acc[v].z);
          acc[v].w = fmaf(x[k][v].w, f, acc[v].w);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V4; ++v) {
      if (lane + 32 * v < LANES) store(item, h, lane + 32 * v, acc[v], sum, mm, m);
    }
  }
  if (PAIRS > 1 && !__syncthreads_or(count > kJoinWarp)) return;

  for (int i = 0; i < PAIRS; ++i) {
    int item, h;
    int4 me;
    const int count = look(blockIdx.x * PAIRS + i, item, h, me);
    if (count == 0 || (PAIRS > 1 && count <= kJoinWarp)) continue;
    auto part = [&](int k) {
      return p.partial + (k == 0 ? (int64_t)me.y : 2 * ((int64_t)me.z + k * p.abreast)) * slot_row + h * kRow;
    };
    const int d = tid % LANES + (PAIRS == 1 ? blockIdx.y * LANES : 0), kg = tid / LANES;
    // the first kJoinThreads partials; with one pair a block their rows are on
    // their way before the maxima are known (1 x 32768, 8 kv heads: 26.3 -> 23.6 us)
    const float4 none = make_float4(kNoMax, kNoMax, 0.f, 0.f);
    const float4 head = tid < count ? *reinterpret_cast<const float4*>(part(tid)) : none;
    constexpr int kRows = PAIRS == 1 ? kJoinThreads / KG : 1;
    float4 rows[kRows];
    if constexpr (PAIRS == 1) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int k = kg + j * KG;
        rows[j] = k < count ? *reinterpret_cast<const float4*>(part(k) + 4 + 4 * d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    // the maxima over all partials
    float m = head.x, mm = head.y;
    for (int k = tid + kJoinThreads; k < count; k += kJoinThreads) {
      const float4 x = *reinterpret_cast<const float4*>(part(k));
      m = fmaxf(m, x.x);
      mm = fmaxf(mm, x.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    }
    __syncthreads();  // the item before is done with the shared arrays
    if ((tid & 31) == 0) {
      s_red[0][tid >> 5] = m;
      s_red[1][tid >> 5] = mm;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) {
      m = fmaxf(m, s_red[0][i]);
      mm = fmaxf(mm, s_red[1][i]);
    }
    // weights of kJoinThreads partials at a time, then their sum
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < count; k0 += kJoinThreads) {
      const int here = count - k0 < kJoinThreads ? count - k0 : kJoinThreads;
      if (k0 > 0) __syncthreads();
      if (tid < here) {
        const float4 x = k0 == 0 ? head : *reinterpret_cast<const float4*>(part(k0 + tid));
        sum += x.z * ex2(x.x - m);
        s_w[tid] = ex2(x.y - mm);
      }
      __syncthreads();
      auto add = [&](int k, float4 x) {
        const float f = s_w[k];
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z);
        acc.w = fmaf(x.w, f, acc.w);
      };
      if (PAIRS == 1 && k0 == 0) {
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          if (kg + j * KG < here) add(kg + j * KG, rows[j]);
        }
      } else {
#pragma unroll 8
        for (int k = kg; k < here; k += KG) add(k, *reinterpret_cast<const float4*>(part(k0 + k) + 4 + 4 * d));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) s_red[2][tid >> 5] = sum;
    s_part[kg][tid % LANES] = acc;
    __syncthreads();
    if (kg == 0) {
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < kJoinThreads / 32; ++i) sum += s_red[2][i];
#pragma unroll
      for (int i = 1; i < KG; ++i) {
        const float4 x = s_part[i][tid % LANES];
        acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
      }
      store(item, h, d, acc, sum, mm, m);
    }
  }
}

template <typename F, typename... P>
cudaError_t launch(F kern, dim3 grid, int threads, int smem, cudaStream_t stream, bool pdl, const P&... p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p...);
}

struct AttnPlan {
  int dp, head_blocks, ctas, slot_heads, abreast;
  int64_t units;  // of the longest item
  bool cut;       // an item can span workers: the join kernel and its workspace are needed
};

AttnPlan attn_plan(int64_t B, int group, int kv_heads, int head_dim, int64_t capacity, int sms) {
  AttnPlan a{};
  a.dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  // more than 8 query heads of a kv head are several items, which read the same
  // codes at about the same time (16 columns in one item took 44 us where two
  // items take 34: 16 x 4096, 4 kv heads of 96, 12 query heads each)
  a.head_blocks = (group + kHeads - 1) / kHeads;
  const int per_sm = a.dp == 64 ? AttnShape<64>::kPerSm : a.dp == 128 ? AttnShape<128>::kPerSm : AttnShape<256>::kPerSm;
  const int64_t units = capacity <= kWhole * kTile ? 1 : (capacity + kTile - 1) / kTile;
  const int64_t items = B * kv_heads * a.head_blocks;
  const int64_t most = (int64_t)sms * per_sm;
  a.ctas = (int)(items > most / units ? most : items * units);
  a.cut = units > 1;
  for (int i = 1; i <= 32; ++i) {
    if (kv_heads * a.head_blocks % i == 0) a.abreast = i;
  }
  a.units = units;
  a.slot_heads = group < kHeads ? group : kHeads;
  return a;
}

// The codes as a 4-D tensor (head_dim, token and head in the order of their
// strides, page); a box is 16 tokens of one head. False where a tensor map
// cannot hold them: one whose pages, tokens or heads are the same memory (a
// stride of 0, as of an expanded tensor) is among these. A stride of a dimension
// of size 1 is 0 as well, but never used: the map gets 16 for it.
bool encode_pool(CUtensorMap* map, const KvCache& c, uint8_t* base, const int64_t (&stride)[3], bool* swap) {
  const int size[3] = {c.num_pages, c.page_size, c.kv_heads};
  for (int i = 0; i < 3; ++i) {
    if (stride[i] == 0 && size[i] > 1) return false;
  }
  *swap = stride[2] < stride[1];
  const uint64_t tok = stride[1] ? (uint64_t)stride[1] : 16, head = stride[2] ? (uint64_t)stride[2] : 16,
                 page = stride[0] ? (uint64_t)stride[0] : 16;
  const uint32_t rb = c.head_dim <= 64 ? 64 : 128;
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)(*swap ? c.kv_heads : c.page_size),
                            (uint64_t)(*swap ? c.page_size : c.kv_heads), (uint64_t)c.num_pages};
  const uint64_t strides[3] = {*swap ? head : tok, *swap ? tok : head, page};
  const uint32_t box[4] = {rb, *swap ? 1u : 16u, *swap ? 16u : 1u, 1u};
  return encode_tensor_map_4d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, dims, strides, box,
                              rb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B) == CUDA_SUCCESS;
}

template <int DP, bool FP8, bool BF16>
cudaError_t run_attn(KvAttn p, const AttnPlan& a, cudaStream_t stream) {
  using S = AttnShape<DP>;
  CUtensorMap kmap{}, vmap{};
  // whole 16-token tiles per page, and strides the tensor map can hold (else the copies of 16 bytes)
  const bool tma = p.c.page_size % 16 == 0 && encode_pool(&kmap, p.c, p.c.k, p.c.k_stride, &p.k_swap) &&
                   encode_pool(&vmap, p.c, p.c.v, p.c.v_stride, &p.v_swap);
  auto go = [&](auto kern) {
    const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kern), S::kAlloc);
    return e != cudaSuccess
               ? e
               : launch(kern, dim3(a.ctas), kAttnWarps * 32, S::kAlloc, stream, p.pdl, kmap, vmap, p);
  };
  const cudaError_t e =
      tma ? go(kv_attn_kernel<DP, FP8, BF16, true>) : go(kv_attn_kernel<DP, FP8, BF16, false>);
  if (e != cudaSuccess || !a.cut) return e;
  const int items = p.B * p.c.kv_heads * p.head_blocks;
  const int64_t pairs = (int64_t)items * p.slot_heads;
  // more partials an item than a warp takes, on average: blocks for 32 dims of a pair
  if ((int64_t)items * kJoinWarp < (int64_t)a.ctas * kAttnWarps && a.units > 2 * kJoinWarp) {
    return launch(kv_attn_join_kernel<DP, BF16, 1>, dim3(pairs, DP / 32), 256, 0, stream, true, p, items);
  }
  return launch(kv_attn_join_kernel<DP, BF16, 4>, dim3((pairs + 3) / 4), 128, 0, stream, true, p, items);
}

template <int DP>
cudaError_t run_attn_t(const KvAttn& p, const AttnPlan& a, bool fp8, bool bf16, cudaStream_t stream) {
  if (fp8) return bf16 ? run_attn<DP, true, true>(p, a, stream) : run_attn<DP, true, false>(p, a, stream);
  return bf16 ? run_attn<DP, false, true>(p, a, stream) : run_attn<DP, false, false>(p, a, stream);
}

int grid_rows(int64_t rows, int lpr) {
  // a row per group of lanes until every SM has its blocks, then up to kAtOnce
  const int64_t want = (rows * lpr + 255) / 256, cap = (int64_t)num_sms() * 8;
  const int64_t deep = (want + kAtOnce - 1) / kAtOnce;
  return (int)(want < 1 ? 1 : want <= cap ? want : deep > cap ? deep : cap);
}

}  // namespace

cudaError_t launch_kv_write(const KvCache& c, const void* k, const int64_t* k_stride, const void* v,
                            const int64_t* v_stride, const int64_t* slots, int T, bool fp8, bool bf16,
                            cudaStream_t stream) {
  const int lpr = c.head_dim <= 64 ? 4 : c.head_dim <= 128 ? 8 : 16;
  const dim3 grid(grid_rows((int64_t)T * c.kv_heads, lpr));
  const KvWrite p{c, k, v, {k_stride[0], k_stride[1]}, {v_stride[0], v_stride[1]}, slots, T,
                  make_fastdiv((uint32_t)c.kv_heads), make_fastdiv((uint32_t)c.page_size), device_status_ptr(),
                  pdl_enabled()};
  auto go = [&](auto k4, auto k8, auto k16) {
    return launch(lpr == 4 ? k4 : lpr == 8 ? k8 : k16, grid, 256, 0, stream, p.pdl, p);
  };
#define NSQ_KV_GO(F, B) go(kv_write_kernel<F, B, 4>, kv_write_kernel<F, B, 8>, kv_write_kernel<F, B, 16>)
  if (fp8) return bf16 ? NSQ_KV_GO(true, true) : NSQ_KV_GO(true, false);
  return bf16 ? NSQ_KV_GO(false, true) : NSQ_KV_GO(false, false);
#undef NSQ_KV_GO
}

cudaError_t launch_kv_read(const KvCache& c, const int64_t* slots, int T, void* k, void* v, bool fp8, bool bf16,
                           cudaStream_t stream) {
  const int lpr = c.head_dim <= 64 ? 4 : c.head_dim <= 128 ? 8 : 16;
  const dim3 grid(grid_rows((int64_t)T * c.kv_heads, lpr));
  const KvRead p{c, k, v, slots, T, make_fastdiv((uint32_t)c.kv_heads), make_fastdiv((uint32_t)c.page_size),
                 device_status_ptr(), pdl_enabled()};
  auto go = [&](auto k4, auto k8, auto k16) {
    return launch(lpr == 4 ? k4 : lpr == 8 ? k8 : k16, grid, 256, 0, stream, p.pdl, p);
  };
#define NSQ_KV_GO(F, B) go(kv_read_kernel<F, B, 4>, kv_read_kernel<F, B, 8>, kv_read_kernel<F, B, 16>)
  if (fp8) return bf16 ? NSQ_KV_GO(true, true) : NSQ_KV_GO(true, false);
  return bf16 ? NSQ_KV_GO(false, true) : NSQ_KV_GO(false, false);
#undef NSQ_KV_GO
}

// Workspace: per worker two partial slots ([heads][head_dim + 4] fp32 each: two
// references, the denominator, a pad, the accumulator), then one int4 per item:
// its partials (-1: not cut), the first one's slot, and the worker of that slot;
// the others are the first slots of its place in the teams after. Its size is
// for all SMs of the device: SMs kept free for others (which may change from
// one call to the next, and during one) only make the grid of a launch smaller.
static size_t attn_slot_bytes(const AttnPlan& a) {
  return (size_t)a.ctas * kAttnWarps * 2 * a.slot_heads * (a.dp + 4) * sizeof(float);
}

size_t kv_attn_workspace(int64_t B, int group, int kv_heads, int head_dim, int64_t capacity) {
  const AttnPlan a = attn_plan(B, group, kv_heads, head_dim, capacity, device_sms());
  return a.cut ? attn_slot_bytes(a) + (size_t)B * kv_heads * a.head_blocks * sizeof(int4) : 0;
}

cudaError_t launch_kv_attn(const KvAttnArgs& args, bool fp8, bool bf16, void* ws, cudaStream_t stream) {
  const int group = args.H / args.c.kv_heads;
  const AttnPlan a = attn_plan(args.B, group, args.c.kv_heads, args.c.head_dim, args.capacity, num_sms());
  KvAttn p{args};
  p.group = group;
  p.head_blocks = a.head_blocks;
  p.page_div = make_fastdiv((uint32_t)args.c.page_size);
  p.scale_log2 = args.scale * 1.4426950408889634f;
  p.slot_heads = a.slot_heads;
  p.least_log2 = a.cut ? 1 : 0;
  p.abreast = a.abreast;
  p.abreast_div = make_fastdiv((uint32_t)a.abreast);
  p.teams = a.ctas * kAttnWarps / a.abreast;
  p.partial = a.cut ? static_cast<float*>(ws) : nullptr;
  p.meta = a.cut ? reinterpret_cast<int4*>(static_cast<uint8_t*>(ws) + attn_slot_bytes(a)) : nullptr;
  p.status = device_status_ptr();
  p.pdl = pdl_enabled();
  p.withhold = test_withhold();
  return a.dp == 64    ? run_attn_t<64>(p, a, fp8, bf16, stream)
         : a.dp == 128 ? run_attn_t<128>(p, a, fp8, bf16, stream)
                       : run_attn_t<256>(p, a, fp8, bf16, stream);
}

}  // namespace nsq
