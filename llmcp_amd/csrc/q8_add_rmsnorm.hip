// q8_add_rmsnorm.hip -- the residual's addition, RMSNorm and the Q8_1 of its
// rows in one pass.
//
// s = x + r (rounded to the rows' type), rstd = f32(1 / sqrt(sum s^2 / H +
// eps)), y = (s * rstd) * w' in f32, rounded to the type, and per 32 values
// of y as stored the quantizer's arithmetic.  The squares of f32 values are
// exact in f64 and are summed there: the error of any order of the sum lies
// about 2^29 below f32's rounding, so a tree gives the same rstd as a serial
// sum but for one row in some 10^8, and no step of a quantizer hangs on how
// the row is split over lanes.  (The f64 work is a multiply and an add per
// value of a row that is bound by memory.)  Measured in bf16, H = 2560, sum, norm
// and Q8_1 out: one row 3.9 us (the latency of two passes over the workgroup),
// 4096 rows 19.2 us for 96 MB (5.0 TB/s; a copy reaches 5.3; 20.7 with the
// loads one by one and the sum by LDS permutes).
#include "q8_kernels.h"

#include <algorithm>

#include "q8_device.h"
#include "q8_gemv.h"

namespace llmcp_q8 {
namespace {

struct AddNormArgs {
  const void *x, *r, *w;
  int64_t ldx, ldr, lds, ldy;
  void *s, *y;  // y may be null
  int8_t *q;    // Q8_1 rows, dense, or null
  float *qs;
  float eps;
  int32_t zero_centered, h;
  int32_t ax, ar, as, ay;  // rows take vector accesses
};

// Eight values of a row.
template <bool BF16>
__device__ __forceinline__ void load8(float (&v)[8], const void *p, int64_t i, int aligned) {
  if (BF16 && aligned == 2) {
    const uint4 b = *(const uint4 *)((const uint16_t *)p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = bf16_to_float(word(b, k) & 0xffffu);
      v[2 * k + 1] = bf16_to_float(word(b, k) >> 16);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float4 f = load_act4(p, i + 4 * k, BF16, aligned != 0);
    v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
  }
}

// Eight values as they are in memory, 16 B aligned: no conversion, so that the
// loads behind one go out before it has come.
template <bool BF16>
struct Raw8 {
  uint4 b[BF16 ? 1 : 2];
  __device__ __forceinline__ void load(const void *p, int64_t i) {
    const uint4 *const at = (const uint4 *)((const uint8_t *)p + i * (BF16 ? 2 : 4));
#pragma unroll
    for (int k = 0; k < (BF16 ? 1 : 2); ++k) b[k] = at[k];
  }
  __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (BF16) v[k] = bf16_to_float(k & 1 ? word(b[0], k / 2) >> 16 : word(b[0], k / 2) & 0xffffu);
      else v[k] = __uint_as_float(word(b[k / 4], k % 4));
    }
  }
};

// Stores eight values, rounding v to what is stored.
template <bool BF16>
__device__ __forceinline__ void store8(float (&v)[8], void *p, int64_t i, int aligned) {
  if (BF16) {
    uint16_t b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      b[k] = float_to_bf16(v[k]);
      v[k] = bf16_to_float(b[k]);
    }
    if (!p) return;
    uint16_t *const to = (uint16_t *)p + i;
    if (aligned == 2) {
      *(uint4 *)to = make_uint4(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16,
                                b[4] | (uint32_t)b[5] << 16, b[6] | (uint32_t)b[7] << 16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) to[k] = b[k];
    }
  } else {
    if (!p) return;
    float *const to = (float *)p + i;
    if (aligned) {
      *(float4 *)to = make_float4(v[0], v[1], v[2], v[3]);
      *(float4 *)(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) to[k] = v[k];
    }
  }
}

// v of the lane that CTRL names, 0 where there is none, added.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const int2 b = __builtin_bit_cast(int2, v);
  const int2 o = make_int2(__builtin_amdgcn_update_dpp(0, b.x, CTRL, 0xf, 0xf, true),
                           __builtin_amdgcn_update_dpp(0, b.y, CTRL, 0xf, 0xf, true));
  return v + __builtin_bit_cast(double, o);
}

// A workgroup per row; thread t holds values 8 (t + i * threads) .. + 7 for
// i < VPT in registers from the loads to the stores, so outputs may take the
// inputs' memory.  VEC: input rows and weight 16 B aligned, all their loads out
// together.
template <bool BF16, int VPT, bool VEC>
__global__ __launch_bounds__(1024) void add_rmsnorm_kernel(const AddNormArgs p) {
  __shared__ double part[16];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, threads = blockDim.x, vecs = p.h / 8;
  float v[VPT][8];
  double sum = 0.0;
  float w[VPT][8];
  if constexpr (VEC) {
    Raw8<BF16> x[VPT], r[VPT], g[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      // (past the row: the last values again, taken out below)
      const int e = min(t + i * threads, vecs - 1);
      x[i].load(p.x, row * p.ldx + 8 * e);
      r[i].load(p.r, row * p.ldr + 8 * e);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) g[i].load(p.w, 8 * min(t + i * threads, vecs - 1));
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[8];
      x[i].widen(v[i]);
      r[i].widen(f);
      g[i].widen(w[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = v[i][k] + f[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = min(t + i * threads, vecs - 1);
      float f[8];
      load8<BF16>(v[i], p.x, row * p.ldx + 8 * e, p.ax);
      load8<BF16>(f, p.r, row * p.ldr + 8 * e, p.ar);
      load8<BF16>(w[i], p.w, 8 * e, 1);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = v[i][k] + f[k];
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = t + i * threads;
    if (e < vecs) {
      store8<BF16>(v[i], p.s, row * p.lds + 8 * e, p.as);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += (double)v[i][k] * (double)v[i][k];
  }
  sum = dpp_add<0x111>(sum);  // row_shr:1, 2, 4, 8
  sum = dpp_add<0x112>(sum);
  sum = dpp_add<0x114>(sum);
  sum = dpp_add<0x118>(sum);
  sum = dpp_add<0x142>(sum);  // row_bcast:15, 31: the whole sum in lane 63
  sum = dpp_add<0x143>(sum);
  if ((t & 63) == 63) part[t >> 6] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < threads / 64; ++i) sum += part[i];
  const float rstd = (float)(1.0 / sqrt(sum / (double)p.h + (double)p.eps));
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = t + i * threads;
    const bool live = e < vecs;  // alike in the four lanes of a block
    if (live) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float ww = p.zero_centered ? w[i][k] + 1.0f : w[i][k];
        v[i][k] = (v[i][k] * rstd) * ww;
      }
      store8<BF16>(v[i], p.y, row * p.ldy + 8 * e, p.ay);
    }
    if (p.q) {
      // Q8_1 of a block of four lanes: quantize_block8 on eight values a lane
      float m = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[i][k]));
      m = fmaxf(m, dpp_f32<0xB1>(m));
      m = fmaxf(m, dpp_f32<0x4E>(m));
      const float s = div127(m);
      const bool zero = m == 0.0f, slow = !zero && !recip_in_range(s);
      float inv = zero ? 0.0f : recip_fast(s);
      if (__builtin_amdgcn_ballot_w64(slow)) inv = zero ? 0.0f : recip(s);
      uint32_t b[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        b[j] = round_byte(v[i][4 * j] * inv) | (round_byte(v[i][4 * j + 1] * inv) << 8) |
               (round_byte(v[i][4 * j + 2] * inv) << 16) | (round_byte(v[i][4 * j + 3] * inv) << 24);
      if (live) {
        *(uint2 *)(p.q + row * p.h + 8 * e) = make_uint2(b[0], b[1]);
        if ((t & 3) == 0) p.qs[row * (p.h / kBlock) + e / 4] = s;
      }
    }
  }
}

// 2: 16 B accesses of eight bf16 values, 1: of four values, 0: single ones.
int row_access(const void *p, int64_t ld, bool bf16) {
  if (bf16 && (uintptr_t)p % 16 == 0 && ld % 8 == 0) return 2;
  return (uintptr_t)p % (bf16 ? 8 : 16) == 0 && ld % 4 == 0 ? 1 : 0;
}

template <bool BF16>
hipError_t launch_add_rmsnorm_t(const AddNormArgs &a, int64_t m, hipStream_t s) {
  const int vecs = a.h / 8;
  const int threads = std::min(1024, (vecs + 63) / 64 * 64);
  const dim3 grid((unsigned)m), wg((unsigned)threads);
  const int most = BF16 ? 2 : 1;
  const bool vec = a.ax == most && a.ar == most && (uintptr_t)a.w % 16 == 0;
  const auto kernel = vec ? (vecs <= 1024   ? add_rmsnorm_kernel<BF16, 1, true>
                             : vecs <= 2048 ? add_rmsnorm_kernel<BF16, 2, true>
                                            : add_rmsnorm_kernel<BF16, 4, true>)
                          : (vecs <= 1024   ? add_rmsnorm_kernel<BF16, 1, false>
                             : vecs <= 2048 ? add_rmsnorm_kernel<BF16, 2, false>
                                            : add_rmsnorm_kernel<BF16, 4, false>);
  hipLaunchKernelGGL(kernel, grid, wg, 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_add_rmsnorm(const void *x, int64_t ldx, const void *r, int64_t ldr, bool bf16,
                              int64_t m, int64_t h, const void *w, float eps, bool zero_centered,
                              void *s, int64_t lds, void *y, int64_t ldy, int8_t *q, float *qs,
                              hipStream_t stream) {
  if (h > kAddNormMaxCols || m > 0xFFFFFFFFll / 1024) return hipErrorInvalidConfiguration;
  AddNormArgs a = {x, r, w, ldx, ldr, lds, ldy, s, y, q, qs, eps, zero_centered ? 1 : 0, (int32_t)h,
                   row_access(x, ldx, bf16), row_access(r, ldr, bf16), row_access(s, lds, bf16),
                   row_access(y, ldy, bf16)};
  return bf16 ? launch_add_rmsnorm_t<true>(a, m, stream) : launch_add_rmsnorm_t<false>(a, m, stream);
}

}  // namespace llmcp_q8
