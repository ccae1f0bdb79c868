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
  int group, head_blocks;
  FastDiv page_div;
  float scale_log2;
  float* partial;
  int4* meta;
  DevStatus* status;
  bool pdl;
};

// Records the first bad value in a device-side argument (tag 200 a written
// slot, 201 a read one, 202 a page, 203 a length) in the status word.
__device__ __forceinline__ void report(DevStatus* st, uint32_t where) {
  if (st != nullptr && atomicCAS(&st->code, 0u, (unsigned)NSQ_EINVAL) == 0u) {
    st->where = where;
    st->block = blockIdx.x;
  }
}

// ---------------------------------------------------------------------------
// Write and read
// ---------------------------------------------------------------------------

// Eight elements of a row per lane, LPR lanes per row (LPR * 8 >= head_dim):
// one 16-byte load, a shuffle maximum, one 8-byte store. Bound by DRAM.
template <bool FP8, bool BF16, int LPR>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvWrite p) {
  if (p.pdl) pdl_wait_prior_grids();
  const int sub = threadIdx.x % LPR;
  const uint32_t rows = (uint32_t)p.T * (uint32_t)p.c.kv_heads;
  const bool in_row = sub * 8 < p.c.head_dim;
  for (uint32_t r0 = (blockIdx.x * 256 + threadIdx.x) / LPR; r0 < 2 * rows; r0 += gridDim.x * (256 / LPR)) {
    const bool isv = r0 >= rows;
    const uint32_t r = isv ? r0 - rows : r0;
    const int64_t tok = fdiv(r, p.head_div);
    const int head = (int)(r - (uint32_t)tok * (uint32_t)p.c.kv_heads);
    const int64_t slot = __ldg(p.slots + tok);
    if (slot < 0) continue;  // a padded token
    if (slot >= (int64_t)p.c.num_pages * p.c.page_size) {
      if (sub == 0) report(p.status, 200);
      continue;
    }
    const int64_t page = fdiv((uint32_t)slot, p.page_div);
    const int64_t off = slot - page * p.c.page_size;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (in_row) {
      const uint16_t* src = static_cast<const uint16_t*>(isv ? p.v : p.k) +
                            tok * (isv ? p.v_stride[0] : p.k_stride[0]) + head * (isv ? p.v_stride[1] : p.k_stride[1]);
      raw = __ldg(reinterpret_cast<const uint4*>(src + sub * 8));
    }
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = elem_to_float<BF16>((uint16_t)(w[i / 2] >> (16 * (i & 1))));
      m = nan_max(m, fabsf(x[i]));
    }
    // the lanes of a row are converged here: whole rows leave the loop together
    const uint32_t lanes = LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u) << (threadIdx.x & 31 & ~(LPR - 1));
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) m = nan_max(m, __shfl_xor_sync(lanes, m, o));
    const float s = row_scale<FP8>(m);
    const RowDiv dv(s);
    uint32_t c0 = 0, c1 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c0 |= (uint32_t)row_code<FP8>(dv(x[i])) << (8 * i);
      c1 |= (uint32_t)row_code<FP8>(dv(x[i + 4])) << (8 * i);
    }
    if (in_row) {
      uint8_t* dst = (isv ? p.c.v : p.c.k) +
                     (isv ? page * p.c.v_stride[0] + off * p.c.v_stride[1] + head * p.c.v_stride[2]
                          : page * p.c.k_stride[0] + off * p.c.k_stride[1] + head * p.c.k_stride[2]);
      *reinterpret_cast<uint2*>(dst + sub * 8) = make_uint2(c0, c1);
    }
    if (sub == 0) {
      float* sd = (isv ? p.c.vs : p.c.ks) +
                  (isv ? page * p.c.vs_stride[0] + off * p.c.vs_stride[1] + head * p.c.vs_stride[2]
                       : page * p.c.ks_stride[0] + off * p.c.ks_stride[1] + head * p.c.ks_stride[2]);
      *sd = s;
    }
  }
}

template <bool FP8>
__device__ __forceinline__ float code_value(uint8_t c) {
  if constexpr (FP8) {
    return static_cast<float>(*reinterpret_cast<const __nv_fp8_e4m3*>(&c));
  } else {
    return (float)(int8_t)c;
  }
}

// The inverse: code * s rounded once to the output type. Rows of a negative
// or out-of-range slot read as zero.
template <bool FP8, bool BF16, int LPR>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvRead p) {
  if (p.pdl) pdl_wait_prior_grids();
  const int sub = threadIdx.x % LPR;
  if (sub * 8 >= p.c.head_dim) return;
  const uint32_t rows = (uint32_t)p.T * (uint32_t)p.c.kv_heads;
  for (uint32_t r0 = (blockIdx.x * 256 + threadIdx.x) / LPR; r0 < 2 * rows; r0 += gridDim.x * (256 / LPR)) {
    const bool isv = r0 >= rows;
    const uint32_t r = isv ? r0 - rows : r0;
    const int64_t tok = fdiv(r, p.head_div);
    const int head = (int)(r - (uint32_t)tok * (uint32_t)p.c.kv_heads);
    const int64_t slot = __ldg(p.slots + tok);
    uint32_t o[4] = {0, 0, 0, 0};
    if (slot >= 0) {
      if (slot >= (int64_t)p.c.num_pages * p.c.page_size) {
        if (sub == 0) report(p.status, 201);
      } else {
        const int64_t page = fdiv((uint32_t)slot, p.page_div);
        const int64_t off = slot - page * p.c.page_size;
        const uint8_t* src = (isv ? p.c.v : p.c.k) +
                             (isv ? page * p.c.v_stride[0] + off * p.c.v_stride[1] + head * p.c.v_stride[2]
                                  : page * p.c.k_stride[0] + off * p.c.k_stride[1] + head * p.c.k_stride[2]);
        const float s = *((isv ? p.c.vs : p.c.ks) +
                          (isv ? page * p.c.vs_stride[0] + off * p.c.vs_stride[1] + head * p.c.vs_stride[2]
                               : page * p.c.ks_stride[0] + off * p.c.ks_stride[1] + head * p.c.ks_stride[2]));
        const uint2 c = *reinterpret_cast<const uint2*>(src + sub * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t word = i < 2 ? c.x : c.y;
          const float a = code_value<FP8>((uint8_t)(word >> (16 * (i & 1)))) * s;
          const float b = code_value<FP8>((uint8_t)(word >> (16 * (i & 1) + 8))) * s;
          o[i] = (uint32_t)float_to_elem<BF16>(a) | ((uint32_t)float_to_elem<BF16>(b) << 16);
        }
      }
    }
    uint16_t* dst = static_cast<uint16_t*>(isv ? p.v : p.k) + (int64_t)r * p.c.head_dim + sub * 8;
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---------------------------------------------------------------------------
// Decode attention
// ---------------------------------------------------------------------------
//
// One query token per sequence: out[h] = sum_t p[t] v[t] / sum_t p[t],
// p[t] = exp2(s[t] - m), s[t] = scale * log2(e) * q . k[t], m the running
// maximum. Bound by reading the codes once; so
//   * a warp takes 16 tokens at a time and reads their codes from global
//     memory straight into the registers that are the A operands of
//     mma.m16n8k16 (rows = tokens for q . k, rows = dims for p . v), the query
//     heads that share the kv head being the 8 columns. The order of the k
//     index within an MMA is free, so 16 consecutive bytes per lane are used
//     as they come; no shared memory, no barriers, in the loop;
//   * codes become fp16 exactly; q is scaled per head by a power of two into
//     fp16's range, exact for fp16 and for every bf16 within 2^-14 of the
//     head's largest. Scores, maxima and sums are fp32;
//   * the scale of v is folded into the exponent: the fp16 weights of p . v
//     are exp2(s + log2(vs) - m'), with a maximum m' of their own, so that
//     they use fp16's range whatever the scales are (half-ulp 2^-12 each); the
//     denominator is summed in fp32 from unrounded terms. At the end the
//     accumulator is multiplied by exp2(m' - m);
//   * work is cut into units of 64 tokens of one (sequence, kv head) and dealt
//     evenly to the CTAs on the device, from seq_lens: long and ragged batches
//     fill the machine alike. A CTA's range covers whole items and at most two
//     cut ones; those go to the workspace as fp32 partials, and a second small
//     kernel joins them in order.

constexpr int kAttnWarps = 4;
constexpr int kUnit = 16 * kAttnWarps;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// acc * 2^(mm - m) / sum: the output of a head whose weights of v were taken
// relative to mm and whose denominator relative to m (0 for an empty row; no
// term with a scale above 0 leaves mm at -inf and acc at 0 or NaN).
__device__ __forceinline__ float finish(float acc, float sum, float mm, float m) {
  if (sum == 0.f) return 0.f;
  return acc * (mm == -INFINITY ? 0.f : ex2(mm - (m == -INFINITY ? 0.f : m))) / sum;
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

__device__ __forceinline__ uint4 ld_stream16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Tokens a sequence holds: seq_lens clamped to what its page-table row can name.
__device__ __forceinline__ int seq_tokens(const KvAttn& p, int b, bool tell) {
  int n = __ldg(p.seq_lens + b);
  if (n < 0 || n > p.capacity) {
    if (tell) report(p.status, 203);
    n = n < 0 ? 0 : p.capacity;
  }
  return n;
}
__device__ __forceinline__ int item_units(int n) { return n == 0 ? 1 : (n + kUnit - 1) / kUnit; }

// One warp's 16 tokens. k[r]: row r = token g + 8r, 16-byte chunks of 64 dims;
// v[i]: tokens 2t, 2t+1, 2t+8, 2t+9, dims [g * DP / 8, + DP / 8).
template <int DP>
struct KvTile {
  uint4 k[2][DP / 64];
  uint32_t v[4][DP / 32];
  float ks[2], vs[2];
  bool in[2];  // token g + 8r is held
};

template <int DP, int NT, bool FP8, bool BF16, bool PAGE16>
__global__ void __launch_bounds__(kAttnWarps * 32, DP * NT <= 128 ? 3 : 2) kv_attn_kernel(const KvAttn p) {
  constexpr int KC = DP / 64;      // 16-byte chunks of a K row per lane
  constexpr int VW = DP / 32;      // words of a V row per lane
  constexpr int MT = DP / 16;      // 16-dim tiles of the output
  constexpr int HEADS = 8 * NT;
  __shared__ float s_o[kAttnWarps][HEADS][DP];
  __shared__ float s_m[kAttnWarps][HEADS], s_mv[kAttnWarps][HEADS], s_l[kAttnWarps][HEADS];
  __shared__ long long s_scan[kAttnWarps];
  __shared__ long long s_start[2];  // first unit's sequence, and its index within it

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  if (p.pdl) pdl_wait_prior_grids();

  // ---- deal the units: this CTA takes [u0, u1) of the batch's total ----
  const int kh_n = p.c.kv_heads * p.head_blocks;
  const int vpt = (p.B + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
  long long mine = 0;
  for (int i = 0; i < vpt; ++i) {
    const int b = tid * vpt + i;
    if (b < p.B) mine += (long long)item_units(seq_tokens(p, b, blockIdx.x == 0)) * kh_n;
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
  // (to no more CTAs than units, so that the CTAs of a cut item are neighbours)
  const long long ctas = total < (long long)gridDim.x ? total : (long long)gridDim.x;
  const bool idle = blockIdx.x >= ctas;
  long long u = idle ? total : total * blockIdx.x / ctas;
  const long long u1 = idle ? total : total * (blockIdx.x + 1) / ctas;
  const long long excl = before + incl - mine;
  if (u >= excl && u < excl + mine) {
    long long rel = u - excl;
    int b = tid * vpt;
    for (;;) {
      const long long nb = (long long)item_units(seq_tokens(p, b, false)) * kh_n;
      if (rel < nb) break;
      rel -= nb;
      ++b;
    }
    s_start[0] = b;
    s_start[1] = rel;
  }
  if (p.meta != nullptr && tid == 0) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  if (u >= u1) return;
  int b = (int)s_start[0];
  int n = seq_tokens(p, b, false);
  int nu = item_units(n);
  int kh = (int)(s_start[1] / nu);
  int tu = (int)(s_start[1] - (long long)kh * nu);

  for (bool first = true; u < u1; first = false) {
    // ---- one segment: units [tu, tu + cnt) of item (b, kh) ----
    const int cnt = (int)((long long)(nu - tu) < u1 - u ? (long long)(nu - tu) : u1 - u);
    const int head = kh / p.head_blocks;
    const int hb0 = (kh - head * p.head_blocks) * HEADS;  // first query head of this block within the group
    const uint8_t* kbase = p.c.k + head * p.c.k_stride[2];
    const uint8_t* vbase = p.c.v + head * p.c.v_stride[2];
    const float* ksbase = p.c.ks + head * p.c.ks_stride[2];
    const float* vsbase = p.c.vs + head * p.c.vs_stride[2];

    // q as the B operand: lane (g, t) holds head g, dims c * 64 + 16 t + 0..15
    uint32_t qf[NT][KC][8];
    float sc[NT][2];  // score scale of heads 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int hl = hb0 + nt * 8 + g;
      const uint16_t* qrow = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] +
                             (int64_t)(head * p.group + (hl < p.group ? hl : 0)) * p.q_stride[1];
      uint32_t raw[KC][8];
      float m = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const bool in = hl < p.group && c * 64 + t * 16 < p.c.head_dim;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 x = in ? __ldg(reinterpret_cast<const uint4*>(qrow + c * 64 + t * 16 + h * 8))
                             : make_uint4(0, 0, 0, 0);
          raw[c][4 * h] = x.x, raw[c][4 * h + 1] = x.y, raw[c][4 * h + 2] = x.z, raw[c][4 * h + 3] = x.w;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          m = fmaxf(m, fabsf(elem_to_float<BF16>((uint16_t)raw[c][i])));
          m = fmaxf(m, fabsf(elem_to_float<BF16>((uint16_t)(raw[c][i] >> 16))));
        }
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // the largest lands in [1, 2): e = its exponent, applied in two steps so
      // that neither factor leaves fp32's range
      int e = m > 0.f && m <= 3.4e38f ? ilogbf(m) : 0;
      const float f1 = exp2f((float)(-e / 2)), f2 = exp2f((float)(-e - (-e / 2)));
#pragma unroll
      for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          qf[nt][c][i] = pack_f16(elem_to_float<BF16>((uint16_t)raw[c][i]) * f1 * f2,
                                  elem_to_float<BF16>((uint16_t)(raw[c][i] >> 16)) * f1 * f2);
        }
      }
      const float s = p.scale_log2 / f1 / f2;
      sc[nt][0] = __shfl_sync(0xffffffffu, s, (2 * t) * 4);
      sc[nt][1] = __shfl_sync(0xffffffffu, s, (2 * t + 1) * 4);
    }

    float o[MT][NT][4];
    float mx[NT][2], mv[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < MT; ++j) o[j][nt][0] = o[j][nt][1] = o[j][nt][2] = o[j][nt][3] = 0.f;
      mx[nt][0] = mx[nt][1] = mv[nt][0] = mv[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    const int32_t* table = p.table + b * p.table_stride;
    // Page of this warp's tile in unit i (PAGE16: the whole tile lies in one
    // page; otherwise lane j < 16 looks up token j). A masked token or a page
    // outside the pool gives -1: nothing of it is read.
    auto lookup = [&](int i, int& page, int& off) {
      const int tok = (tu + i) * kUnit + warp * 16 + (PAGE16 ? 0 : (lane & 15));
      page = -1;
      off = 0;
      if (i < cnt && tok < n) {
        const uint32_t pi = fdiv((uint32_t)tok, p.page_div);
        off = tok - (int)pi * p.c.page_size;
        page = __ldg(table + pi);
        if ((uint32_t)page >= (uint32_t)p.c.num_pages) {
          report(p.status, 202);
          page = -1;
        }
      }
    };
    auto load = [&](KvTile<DP>& x, int i, int page, int off) {
      const int t0 = (tu + i) * kUnit + warp * 16;
      auto place = [&](int j, int64_t& pg, int64_t& of) -> bool {
        if constexpr (PAGE16) {
          pg = page;
          of = off + j;
        } else {
          pg = __shfl_sync(0xffffffffu, page, j);
          of = __shfl_sync(0xffffffffu, off, j);
        }
        return pg >= 0 && t0 + j < n;
      };
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        int64_t pg, of;
        const bool in = place(g + 8 * r, pg, of);
        const uint8_t* row = kbase + pg * p.c.k_stride[0] + of * p.c.k_stride[1];
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const int d = c * 64 + t * 16;
          x.k[r][c] = in && d < p.c.head_dim ? ld_stream16(row + d) : make_uint4(0, 0, 0, 0);
        }
        x.ks[r] = in ? __ldg(ksbase + pg * p.c.ks_stride[0] + of * p.c.ks_stride[1]) : 0.f;
        x.vs[r] = in ? __ldg(vsbase + pg * p.c.vs_stride[0] + of * p.c.vs_stride[1]) : 0.f;
        x.in[r] = in;
      }
#pragma unroll
      for (int i2 = 0; i2 < 4; ++i2) {
        int64_t pg, of;
        const bool in = place(2 * t + (i2 & 1) + 8 * (i2 >> 1), pg, of);
        const uint8_t* row = vbase + pg * p.c.v_stride[0] + of * p.c.v_stride[1];
        const int d0 = g * (DP / 8);
        if constexpr (VW == 2) {
          const uint2 y = in && d0 < p.c.head_dim ? ld_stream8(row + d0) : make_uint2(0, 0);
          x.v[i2][0] = y.x, x.v[i2][1] = y.y;
        } else {
#pragma unroll
          for (int h = 0; h < VW / 4; ++h) {
            const uint4 y = in && d0 + 16 * h < p.c.head_dim ? ld_stream16(row + d0 + 16 * h) : make_uint4(0, 0, 0, 0);
            x.v[i2][4 * h] = y.x, x.v[i2][4 * h + 1] = y.y, x.v[i2][4 * h + 2] = y.z, x.v[i2][4 * h + 3] = y.w;
          }
        }
      }
    };
    auto step = [&](const KvTile<DP>& x) {
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint32_t w0[4] = {x.k[0][c].x, x.k[0][c].y, x.k[0][c].z, x.k[0][c].w};
        const uint32_t w1[4] = {x.k[1][c].x, x.k[1][c].y, x.k[1][c].z, x.k[1][c].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a[4];
          codes_to_f16<FP8>(w0[w], a[0], a[2]);
          codes_to_f16<FP8>(w1[w], a[1], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<false>(s[nt], a, qf[nt][c][2 * w], qf[nt][c][2 * w + 1]);
        }
      }
      const float lv0 = lg2(x.vs[0]), lv1 = lg2(x.vs[1]);
      uint32_t pb[NT][2];
      bool grew = false;
      float sv[NT][4], m_new[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[nt][e] = x.in[0] ? s[nt][e] * (x.ks[0] * sc[nt][e]) : -INFINITY;
          s[nt][2 + e] = x.in[1] ? s[nt][2 + e] * (x.ks[1] * sc[nt][e]) : -INFINITY;
          sv[nt][e] = s[nt][e] + lv0;
          sv[nt][2 + e] = s[nt][2 + e] + lv1;
          float a = fmaxf(s[nt][e], s[nt][2 + e]), v = fmaxf(sv[nt][e], sv[nt][2 + e]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
          }
          if (a > mx[nt][e]) {
            l[nt][e] *= ex2(mx[nt][e] - a);
            mx[nt][e] = a;
          }
          m_new[nt][e] = fmaxf(mv[nt][e], v);
          grew |= m_new[nt][e] > mv[nt][e];
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f0 = m_new[nt][0] > mv[nt][0] ? ex2(mv[nt][0] - m_new[nt][0]) : 1.f;
          const float f1 = m_new[nt][1] > mv[nt][1] ? ex2(mv[nt][1] - m_new[nt][1]) : 1.f;
          mv[nt][0] = m_new[nt][0];
          mv[nt][1] = m_new[nt][1];
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            o[j][nt][0] *= f0, o[j][nt][2] *= f0;
            o[j][nt][1] *= f1, o[j][nt][3] *= f1;
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // a maximum of -inf (nothing unmasked yet): every term is exp2(-inf) = 0
        const float a0 = mx[nt][0] == -INFINITY ? 0.f : mx[nt][0], a1 = mx[nt][1] == -INFINITY ? 0.f : mx[nt][1];
        const float v0 = mv[nt][0] == -INFINITY ? 0.f : mv[nt][0], v1 = mv[nt][1] == -INFINITY ? 0.f : mv[nt][1];
        l[nt][0] += ex2(s[nt][0] - a0) + ex2(s[nt][2] - a0);
        l[nt][1] += ex2(s[nt][1] - a1) + ex2(s[nt][3] - a1);
        pb[nt][0] = movmatrix_trans(pack_f16(ex2(sv[nt][0] - v0), ex2(sv[nt][1] - v1)));
        pb[nt][1] = movmatrix_trans(pack_f16(ex2(sv[nt][2] - v0), ex2(sv[nt][3] - v1)));
      }
      // dims 2j, 2j + 1 of this lane's DP / 8 are rows g, g + 8 of tile j
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        uint32_t a[4], c[4];
        codes_to_f16<FP8>(prmt(x.v[0][j], x.v[1][j], 0x5140), a[0], a[1]);
        codes_to_f16<FP8>(prmt(x.v[2][j], x.v[3][j], 0x5140), a[2], a[3]);
        codes_to_f16<FP8>(prmt(x.v[0][j], x.v[1][j], 0x7362), c[0], c[1]);
        codes_to_f16<FP8>(prmt(x.v[2][j], x.v[3][j], 0x7362), c[2], c[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816<false>(o[2 * j][nt], a, pb[nt][0], pb[nt][1]);
          mma_16816<false>(o[2 * j + 1][nt], c, pb[nt][0], pb[nt][1]);
        }
      }
    };

    // The next tile's codes are in flight while this one is used, and the
    // page of the one after is looked up.
    {
      KvTile<DP> x0, x1;
      int pg, of;
      lookup(0, pg, of);
      load(x0, 0, pg, of);
      lookup(1, pg, of);
      for (int i = 0; i < cnt; i += 2) {
        load(x1, i + 1, pg, of);
        lookup(i + 2, pg, of);
        step(x0);
        if (i + 1 >= cnt) break;
        load(x0, i + 2, pg, of);
        lookup(i + 3, pg, of);
        step(x1);
      }
    }

    // ---- join the warps ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
        const int h = nt * 8 + 2 * t + e;
        if (g == 0) {
          s_m[warp][h] = mx[nt][e];
          s_mv[warp][h] = mv[nt][e];
          s_l[warp][h] = l[nt][e];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          s_o[warp][h][g * (DP / 8) + 2 * j] = o[j][nt][e];
          s_o[warp][h][g * (DP / 8) + 2 * j + 1] = o[j][nt][2 + e];
        }
      }
    }
    __syncthreads();
    const bool whole = cnt == nu;
    const int slot = 2 * blockIdx.x + (first ? 0 : 1);
    const int heads = p.group - hb0 < HEADS ? p.group - hb0 : HEADS;
    for (int i = tid; i < heads * DP; i += kAttnWarps * 32) {
      const int h = i / DP, d = i - h * DP;
      float m = -INFINITY, mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        m = fmaxf(m, s_m[w][h]);
        mm = fmaxf(mm, s_mv[w][h]);
      }
      const float m0 = m == -INFINITY ? 0.f : m, mm0 = mm == -INFINITY ? 0.f : mm;
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        acc += s_o[w][h][d] * ex2(s_mv[w][h] - mm0);
        sum += s_l[w][h] * ex2(s_m[w][h] - m0);
      }
      if (whole) {
        const int64_t row = (int64_t)b * p.H + head * p.group + hb0 + h;
        if (d < p.c.head_dim) {
          const float y = finish(acc, sum, mm, m);
          static_cast<uint16_t*>(p.out)[row * p.c.head_dim + d] = float_to_elem<BF16>(y);
        }
        if (d == 0 && p.lse != nullptr) p.lse[row] = sum == 0.f ? -INFINITY : (m0 + log2f(sum)) * 0.69314718055994531f;
      } else {
        float* ws = p.partial + (int64_t)slot * HEADS * (DP + 4) + h * (DP + 4);
        ws[4 + d] = acc;
        if (d == 0) {
          ws[0] = m;
          ws[1] = mm;
          ws[2] = sum;
        }
      }
    }
    // the CTA that opens a cut item says which slot it used and which CTA closes the item
    if (!whole && tu == 0 && tid == 0) {
      const int last = (int)(((u + nu) * ctas + total - 1) / total) - 1;
      p.meta[blockIdx.x] = make_int4(b * kh_n + kh, slot, last, 0);
    }
    __syncthreads();  // the next segment reuses the shared arrays

    u += cnt;
    tu = 0;
    if (++kh == kh_n && u < u1) {
      kh = 0;
      ++b;
      n = seq_tokens(p, b, false);
      nu = item_units(n);
    }
  }
}

// Joins the partials of cut items, one CTA per (opening CTA, query head): its
// slot, then the first slots of the CTAs after it up to the one that closes
// the item, always in that order, so results do not depend on timing.
constexpr int kJoinThreads = 256;
template <int DP, int NT, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) kv_attn_join_kernel(const KvAttn p) {
  constexpr int HEADS = 8 * NT;
  constexpr int KG = kJoinThreads / DP;  // groups of threads that share the partials out
  constexpr int64_t kRow = DP + 4, kSlot = (int64_t)HEADS * kRow;
  __shared__ float s_part[KG][DP], s_m[KG], s_mv[KG], s_l[KG];
  pdl_wait_prior_grids();
  const int4 me = p.meta[blockIdx.x];
  if (me.x < 0) return;
  const int kh_n = p.c.kv_heads * p.head_blocks;
  const int b = me.x / kh_n, kh = me.x - b * kh_n;
  const int head = kh / p.head_blocks, h = blockIdx.y;
  const int hq = (kh - head * p.head_blocks) * HEADS + h;
  if (hq >= p.group) return;
  const int count = me.z - (int)blockIdx.x + 1;
  const int d = threadIdx.x % DP, kg = threadIdx.x / DP;
  const float* ws = p.partial + h * kRow;
  float m = -INFINITY, mm = -INFINITY, acc = 0.f, sum = 0.f;
#pragma unroll 4
  for (int k = kg; k < count; k += KG) {
    const float* x = ws + (k == 0 ? me.y : 2 * ((int64_t)blockIdx.x + k)) * kSlot;
    const float mk = x[0], mmk = x[1], lk = x[2], ok = x[4 + d];
    const float mn = fmaxf(m, mk), mmn = fmaxf(mm, mmk);
    const float z = mn == -INFINITY ? 0.f : mn, zz = mmn == -INFINITY ? 0.f : mmn;
    acc = acc * ex2(mm - zz) + ok * ex2(mmk - zz);
    sum = sum * ex2(m - z) + lk * ex2(mk - z);
    m = mn;
    mm = mmn;
  }
  s_part[kg][d] = acc;
  if (d == 0) {
    s_m[kg] = m;
    s_mv[kg] = mm;
    s_l[kg] = sum;
  }
  __syncthreads();
  if (kg != 0) return;
#pragma unroll
  for (int k = 1; k < KG; ++k) {
    const float mn = fmaxf(m, s_m[k]), mmn = fmaxf(mm, s_mv[k]);
    const float z = mn == -INFINITY ? 0.f : mn, zz = mmn == -INFINITY ? 0.f : mmn;
    acc = acc * ex2(mm - zz) + s_part[k][d] * ex2(s_mv[k] - zz);
    sum = sum * ex2(m - z) + s_l[k] * ex2(s_m[k] - z);
    m = mn;
    mm = mmn;
  }
  const int64_t row = (int64_t)b * p.H + head * p.group + hq;
  if (d < p.c.head_dim) {
    static_cast<uint16_t*>(p.out)[row * p.c.head_dim + d] = float_to_elem<BF16>(finish(acc, sum, mm, m));
  }
  if (d == 0 && p.lse != nullptr) {
    p.lse[row] = sum == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(sum)) * 0.69314718055994531f;
  }
}

template <typename F, typename P>
cudaError_t launch(F kern, dim3 grid, int threads, cudaStream_t stream, bool pdl, const P& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

struct AttnPlan {
  int dp, nt, head_blocks, ctas;
  bool cut;  // an item can span CTAs: the join kernel and its workspace are needed
};

AttnPlan attn_plan(int64_t B, int group, int kv_heads, int head_dim, int64_t capacity) {
  AttnPlan a{};
  a.dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  a.nt = group <= 8 || a.dp == 256 ? 1 : 2;
  a.head_blocks = (group + 8 * a.nt - 1) / (8 * a.nt);
  const int64_t units = capacity <= kUnit ? 1 : (capacity + kUnit - 1) / kUnit;
  const int64_t items = B * kv_heads * a.head_blocks;
  const int64_t most = (int64_t)num_sms() * (a.dp * a.nt <= 128 ? 3 : 2);
  a.ctas = (int)(items > most / units ? most : items * units);
  a.cut = units > 1;
  return a;
}

template <int DP, int NT, bool FP8, bool BF16>
cudaError_t run_attn(KvAttn p, const AttnPlan& a, cudaStream_t stream) {
  cudaError_t e = p.c.page_size % 16 == 0
                      ? launch(kv_attn_kernel<DP, NT, FP8, BF16, true>, dim3(a.ctas), kAttnWarps * 32, stream, p.pdl, p)
                      : launch(kv_attn_kernel<DP, NT, FP8, BF16, false>, dim3(a.ctas), kAttnWarps * 32, stream, p.pdl, p);
  if (e != cudaSuccess || !a.cut) return e;
  // programmatic launch: its blocks are resident by the time the partials are written
  return launch(kv_attn_join_kernel<DP, NT, BF16>, dim3(a.ctas, p.group < 8 * NT ? p.group : 8 * NT), kJoinThreads,
                stream, true, p);
}

template <int DP, int NT>
cudaError_t run_attn_t(const KvAttn& p, const AttnPlan& a, bool fp8, bool bf16, cudaStream_t stream) {
  if (fp8) return bf16 ? run_attn<DP, NT, true, true>(p, a, stream) : run_attn<DP, NT, true, false>(p, a, stream);
  return bf16 ? run_attn<DP, NT, false, true>(p, a, stream) : run_attn<DP, NT, false, false>(p, a, stream);
}

int grid_rows(int64_t rows, int lpr) {
  const int64_t want = (rows * lpr + 255) / 256, cap = (int64_t)num_sms() * 16;
  return (int)(want < 1 ? 1 : want > cap ? cap : want);
}

}  // namespace

cudaError_t launch_kv_write(const KvCache& c, const void* k, const int64_t* k_stride, const void* v,
                            const int64_t* v_stride, const int64_t* slots, int T, bool fp8, bool bf16,
                            cudaStream_t stream) {
  const int lpr = c.head_dim <= 64 ? 8 : c.head_dim <= 128 ? 16 : 32;
  const dim3 grid(grid_rows(2 * (int64_t)T * c.kv_heads, lpr));
  const KvWrite p{c, k, v, {k_stride[0], k_stride[1]}, {v_stride[0], v_stride[1]}, slots, T,
                  make_fastdiv((uint32_t)c.kv_heads), make_fastdiv((uint32_t)c.page_size), device_status_ptr(),
                  pdl_enabled()};
  auto go = [&](auto k8, auto k16, auto k32) {
    return launch(lpr == 8 ? k8 : lpr == 16 ? k16 : k32, grid, 256, stream, p.pdl, p);
  };
#define NSQ_KV_GO(F, B) go(kv_write_kernel<F, B, 8>, kv_write_kernel<F, B, 16>, kv_write_kernel<F, B, 32>)
  if (fp8) return bf16 ? NSQ_KV_GO(true, true) : NSQ_KV_GO(true, false);
  return bf16 ? NSQ_KV_GO(false, true) : NSQ_KV_GO(false, false);
#undef NSQ_KV_GO
}

cudaError_t launch_kv_read(const KvCache& c, const int64_t* slots, int T, void* k, void* v, bool fp8, bool bf16,
                           cudaStream_t stream) {
  const int lpr = c.head_dim <= 64 ? 8 : c.head_dim <= 128 ? 16 : 32;
  const dim3 grid(grid_rows(2 * (int64_t)T * c.kv_heads, lpr));
  const KvRead p{c, k, v, slots, T, make_fastdiv((uint32_t)c.kv_heads), make_fastdiv((uint32_t)c.page_size),
                 device_status_ptr(), pdl_enabled()};
  auto go = [&](auto k8, auto k16, auto k32) {
    return launch(lpr == 8 ? k8 : lpr == 16 ? k16 : k32, grid, 256, stream, p.pdl, p);
  };
#define NSQ_KV_GO(F, B) go(kv_read_kernel<F, B, 8>, kv_read_kernel<F, B, 16>, kv_read_kernel<F, B, 32>)
  if (fp8) return bf16 ? NSQ_KV_GO(true, true) : NSQ_KV_GO(true, false);
  return bf16 ? NSQ_KV_GO(false, true) : NSQ_KV_GO(false, false);
#undef NSQ_KV_GO
}

// Workspace: per CTA two partial slots ([heads][head_dim + 4] fp32 each: two
// maxima, the denominator, a pad, the accumulator), then one int4: the item
// that the CTA opens without closing it (or -1), its slot, the closing CTA.
size_t kv_attn_workspace(int64_t B, int group, int kv_heads, int head_dim, int64_t capacity) {
  const AttnPlan a = attn_plan(B, group, kv_heads, head_dim, capacity);
  if (!a.cut) return 0;
  return (size_t)a.ctas * (2 * (size_t)8 * a.nt * (a.dp + 4) * 4 + sizeof(int4));
}

cudaError_t launch_kv_attn(const KvAttnArgs& args, bool fp8, bool bf16, void* ws, cudaStream_t stream) {
  const int group = args.H / args.c.kv_heads;
  const AttnPlan a = attn_plan(args.B, group, args.c.kv_heads, args.c.head_dim, args.capacity);
  KvAttn p{args};
  p.group = group;
  p.head_blocks = a.head_blocks;
  p.page_div = make_fastdiv((uint32_t)args.c.page_size);
  p.scale_log2 = args.scale * 1.4426950408889634f;
  const size_t slots = (size_t)a.ctas * 2 * 8 * a.nt * (a.dp + 4) * sizeof(float);
  p.partial = a.cut ? static_cast<float*>(ws) : nullptr;
  p.meta = a.cut ? reinterpret_cast<int4*>(static_cast<uint8_t*>(ws) + slots) : nullptr;
  p.status = device_status_ptr();
  p.pdl = pdl_enabled();
  if (a.dp == 64) return a.nt == 1 ? run_attn_t<64, 1>(p, a, fp8, bf16, stream) : run_attn_t<64, 2>(p, a, fp8, bf16, stream);
  if (a.dp == 128) {
    return a.nt == 1 ? run_attn_t<128, 1>(p, a, fp8, bf16, stream) : run_attn_t<128, 2>(p, a, fp8, bf16, stream);
  }
  return run_attn_t<256, 1>(p, a, fp8, bf16, stream);
}

}  // namespace nsq
