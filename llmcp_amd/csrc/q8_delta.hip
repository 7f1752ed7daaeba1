// q8_delta.hip -- the gated delta rule: per value head a state S [key_dim,
// value_dim], and per row of a sequence
//   u = beta (v - a S^T k),  S = a S + k u^T,  o = scale S^T q,  a = exp(g).
#include <algorithm>

#include "q8_gemv.h"
#include "q8_mixer.h"

namespace llmcp_q8 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

struct DeltaArgs {
  DeltaLaunch l;
  int32_t slices;  // of a head's columns
};

__device__ __forceinline__ RowRange delta_range(const DeltaLaunch &l, int32_t s) {
  if (!l.starts) return {0, (int32_t)l.rows};
  return row_range(l.starts, s, (int32_t)l.rows);
}

// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// Row after row.  A workgroup has COLS columns of a head's state in registers:
// a thread 4 columns of every 1024 / COLS-th row.  S^T k and S^T q of the state
// before the row are summed together (o = a S^T q + (k . q) u), so a row
// takes one exchange between the waves.
template <bool BF16, int KD, int COLS>
__global__ __launch_bounds__(256) void delta_rows_kernel(const DeltaArgs p) {
  constexpr int PER = COLS / 4, GROUPS = 256 / PER, ROWS = KD / GROUPS;  // lanes a row
  constexpr int VALS = KD / 64;  // values of q and k per lane
  __shared__ float qk[4][2][KD];
  __shared__ __align__(16) float sums[2][4][2][COLS];
  const DeltaLaunch &l = p.l;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = threadIdx.x % PER * 4, r0 = threadIdx.x / PER;
  const int32_t slice = blockIdx.x % p.slices, sh = blockIdx.x / p.slices;
  const int32_t seq = sh / l.heads, head = sh - seq * l.heads;
  const int32_t key_head = head / (l.heads / l.key_heads);
  const RowRange range = delta_range(l, seq);
  const int64_t at = (int64_t)sh * KD * l.value_dim + slice * COLS + c;
  v4f s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    s[i] = l.state ? *(const v4f *)(l.state + at + (int64_t)(r0 + i * GROUPS) * l.value_dim)
                   : v4f{0, 0, 0, 0};
  auto load = [&](const HeadRows &x, int32_t row, float (&v)[VALS]) {
    const int64_t from = row * x.row_ld + key_head * x.head_ld + lane * VALS;
#pragma unroll
    for (int i = 0; i < VALS; ++i)
      v[i] = BF16 ? bf16_to_float(((const uint16_t *)x.data)[from + i]) : ((const float *)x.data)[from + i];
  };
  for (int32_t row = range.lo; row < range.hi; ++row) {
    float q[VALS], k[VALS];
    load(l.q, row, q);
    load(l.k, row, k);
    v4f v;
    const int64_t from = row * l.v.row_ld + head * l.v.head_ld + slice * COLS + c;
    if (BF16) {
      const v2u b = *(const v2u *)((const uint16_t *)l.v.data + from);
      v = v4f{bf16_to_float(b[0] & 0xffffu), bf16_to_float(b[0] >> 16),
              bf16_to_float(b[1] & 0xffffu), bf16_to_float(b[1] >> 16)};
    } else {
      v = *(const v4f *)((const float *)l.v.data + from);
    }
    const float a = expf(l.decay[row * l.decay_ld + head]), beta = l.beta[row * l.beta_ld + head];
    float kk = 0, qq = 0, kq = 0;
#pragma unroll
    for (int i = 0; i < VALS; ++i) {
      kk = __builtin_fmaf(k[i], k[i], kk);
      qq = __builtin_fmaf(q[i], q[i], qq);
      kq = __builtin_fmaf(k[i], q[i], kq);
      qk[wave][0][lane * VALS + i] = q[i];
      qk[wave][1][lane * VALS + i] = k[i];
    }
    kk = wave_sum(kk);
    qq = wave_sum(qq);
    kq = wave_sum(kq);
    const float rk = l.normalize ? 1.0f / sqrtf(kk + l.eps) : 1.0f;
    const float rq = l.scale * (l.normalize ? 1.0f / sqrtf(qq + l.eps) : 1.0f);
    __builtin_amdgcn_wave_barrier();
    v4f pk = v4f{0, 0, 0, 0}, pq = pk;
    float kr[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float qr = qk[wave][0][r0 + i * GROUPS];
      kr[i] = qk[wave][1][r0 + i * GROUPS];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pk[j] = __builtin_fmaf(s[i][j], kr[i], pk[j]);
        pq[j] = __builtin_fmaf(s[i][j], qr, pq[j]);
      }
    }
#pragma unroll
    for (int d = PER; d < 64; d *= 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pk[j] += __shfl_xor(pk[j], d);
        pq[j] += __shfl_xor(pq[j], d);
      }
    }
    float(*const sum)[2][COLS] = sums[row & 1];
    if (lane < PER) {
      *(v4f *)&sum[wave][0][c] = pk;
      *(v4f *)&sum[wave][1][c] = pq;
    }
    __syncthreads();  // (and the row before has been read: two buffers)
    pk = *(const v4f *)&sum[0][0][c];
    pq = *(const v4f *)&sum[0][1][c];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      pk = pk + *(const v4f *)&sum[w][0][c];
      pq = pq + *(const v4f *)&sum[w][1][c];
    }
    const v4f u = (v - pk * (a * rk)) * beta;
    const v4f o = pq * (a * rq) + u * (kq * rk * rq);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float kn = kr[i] * rk;
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = __builtin_fmaf(kn, u[j], a * s[i][j]);
    }
    if (r0 == 0) {
      const int64_t to = row * l.o.row_ld + head * l.o.head_ld + slice * COLS + c;
      if (BF16)
        *(v2u *)((uint16_t *)l.o.data + to) =
            v2u{float_to_bf16(o[0]) | (uint32_t)float_to_bf16(o[1]) << 16,
                float_to_bf16(o[2]) | (uint32_t)float_to_bf16(o[3]) << 16};
      else
        *(v4f *)((float *)l.o.data + to) = o;
    }
  }
  if (range.lo == range.hi && l.state == l.new_state) return;
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    *(v4f *)(l.new_state + at + (int64_t)(r0 + i * GROUPS) * l.value_dim) = s[i];
}

template <bool BF16, int KD, int COLS>
hipError_t launch_delta_rows(const DeltaLaunch &l, hipStream_t s) {
  const DeltaArgs a = {l, l.value_dim / COLS};
  const int64_t grid = (int64_t)l.sequences * l.heads * a.slices;
  if (grid > 0x7FFFFF) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((delta_rows_kernel<BF16, KD, COLS>), dim3((unsigned)grid), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <bool BF16, int KD>
hipError_t launch_delta_k(const DeltaLaunch &l, hipStream_t s) {
  if (l.value_dim % 32 || (int64_t)l.sequences * l.heads * l.value_dim < 256 * 32)
    return launch_delta_rows<BF16, KD, 16>(l, s);
  return launch_delta_rows<BF16, KD, 32>(l, s);
}

}  // namespace

hipError_t launch_delta(const DeltaLaunch &l, hipStream_t s) {
  if (l.key_dim == 128) return l.q.bf16 ? launch_delta_k<true, 128>(l, s) : launch_delta_k<false, 128>(l, s);
  if (l.key_dim == 64) return l.q.bf16 ? launch_delta_k<true, 64>(l, s) : launch_delta_k<false, 64>(l, s);
  return hipErrorInvalidConfiguration;
}

}  // namespace llmcp_q8
