// q8_cache.hip -- keys and values into the pages of a cache and back.
//
// A row x of one head is kept as bf16, or as int8 with one f32 scale: s =
// max|x| / 127, q = rne(x * (1 / s)).  One scale per row and head (and not
// per 32 values, as the linears' Q8_1 has it) factors out of a dot with a
// query and out of a probability times a value, so attention feeds the whole
// numbers q to the matrix cores without a rounding; it costs 4 B of 260.
//
// Bound by memory, one row by the latency of its row starts, length and page, each
// after the other. Measured: 4096 rows of 4 heads of 256, bf16 to Q8 and back 16.9 us
// (25 MB each way, 3.0 TB/s); one row in a replayed pair 5.1 to 7.5.
#include <algorithm>

#include "q8_gemv.h"
#include "q8_mixer.h"

namespace llmcp_q8 {
namespace {

struct KvArgs {
  HeadRows k, v;
  KvBatch b;
  KvPages c;
  int32_t rows;
  int32_t *err_flag;
};

// Where the slot of a row is, in units of rows of `dim` values of head 0: its
// page's first slot plus the slot within a head's; -1 without one.
__device__ __forceinline__ int64_t slot_of(const KvArgs &p, int32_t row, int lane, int32_t &seq) {
  seq = sequence_of(p.b.starts, p.b.sequences, row, lane);
  if (seq < 0) return -1;
  const RowRange r = row_range(p.b.starts, seq, p.rows);
  if (row < r.lo || row >= r.hi) {
    seq = -1;
    return -1;
  }
  const int32_t most = p.b.max_pages * p.c.page_size;
  const int64_t at = (int64_t)p.b.lengths[seq] - r.hi + row;
  if (at < 0 || at >= most) return -1;
  const int32_t index = (int32_t)at / p.c.page_size;
  const int32_t page = page_at(p.b, p.c, seq, index, p.err_flag);
  if (page < 0) return -1;
  return (int64_t)page * p.c.heads * p.c.page_size + ((int32_t)at - index * p.c.page_size);
}

template <bool BF16>
__device__ __forceinline__ void load_head8(float (&v)[8], const HeadRows &x, int64_t at) {
  if (BF16) {
    const uint4 b = *(const uint4 *)((const uint16_t *)x.data + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_to_float(word(b, i) & 0xffffu);
      v[2 * i + 1] = bf16_to_float(word(b, i) >> 16);
    }
  } else {
    const float4 a = *(const float4 *)((const float *)x.data + at);
    const float4 b = *(const float4 *)((const float *)x.data + at + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

__device__ __forceinline__ uint4 pack_bf16(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = float_to_bf16(v[2 * i]) | (uint32_t)float_to_bf16(v[2 * i + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A workgroup per row; thread t holds 8 values of a head of k or v, LANES =
// dim / 8 threads a head.
template <bool BF16, bool Q8, int LANES>
__global__ __launch_bounds__(256) void kv_write_kernel(const KvArgs p) {
  const int32_t row = blockIdx.x;
  int32_t seq;
  const int64_t slot = slot_of(p, row, threadIdx.x & 63, seq);
  if (slot < 0) return;
  const int vecs = p.c.heads * LANES;
  for (int i = threadIdx.x; i < 2 * vecs; i += blockDim.x) {
    const bool value = i >= vecs;
    const int j = value ? i - vecs : i, h = j / LANES, d = j % LANES * 8;
    const HeadRows &x = value ? p.v : p.k;
    float f[8];
    load_head8<BF16>(f, x, row * x.row_ld + h * x.head_ld + d);
    const int64_t to = slot + (int64_t)h * p.c.page_size;
    void *const out = value ? p.c.v : p.c.k;
    if constexpr (!Q8) {
      *(uint4 *)((uint16_t *)out + to * (LANES * 8) + d) = pack_bf16(f);
    } else {
      float m = 0.0f;
      bool odd = false;  // an infinity or NaN in the row
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m = fmaxf(m, fabsf(f[k]));
        odd |= !(fabsf(f[k]) < __builtin_inff());
      }
      if (odd) m = __builtin_inff();
      m = fmaxf(m, dpp_f32<0xB1>(m));   // lanes 1, 2, 7, 15 apart
      m = fmaxf(m, dpp_f32<0x4E>(m));
      m = fmaxf(m, dpp_f32<0x141>(m));
      if (LANES > 8) m = fmaxf(m, dpp_f32<0x140>(m));
      if (LANES > 16) m = fmaxf(m, __shfl_xor(m, 16));
      const bool live = m < __builtin_inff() && m >= 0x1p-118f;
      const float s = live ? div127(m) : m < 1.0f ? 0.0f : __builtin_nanf("");
      const float inv = live ? recip_fast(s) : 0.0f;
      uint32_t b[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float q[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) q[n] = live ? f[4 * k + n] * inv : 0.0f;
        b[k] = round_byte(q[0]) | round_byte(q[1]) << 8 | round_byte(q[2]) << 16 |
               round_byte(q[3]) << 24;
      }
      *(uint2 *)((int8_t *)out + to * (LANES * 8) + d) = make_uint2(b[0], b[1]);
      if (d == 0) (value ? p.c.vs : p.c.ks)[to] = s;
    }
  }
}

template <bool BF16, bool Q8, int LANES>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs p) {
  const int32_t row = blockIdx.x;
  int32_t seq;
  const int64_t slot = slot_of(p, row, threadIdx.x & 63, seq);
  if (seq < 0) return;
  const int vecs = p.c.heads * LANES;
  for (int i = threadIdx.x; i < 2 * vecs; i += blockDim.x) {
    const bool value = i >= vecs;
    const int j = value ? i - vecs : i, h = j / LANES, d = j % LANES * 8;
    const int64_t at = slot + (int64_t)h * p.c.page_size;
    const void *const in = value ? p.c.v : p.c.k;
    float f[8] = {};
    if (slot >= 0) {
      if constexpr (Q8) {
        const uint2 b = *(const uint2 *)((const int8_t *)in + at * (LANES * 8) + d);
        const float s = (value ? p.c.vs : p.c.ks)[at];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          f[k] = (float)(int8_t)((k < 4 ? b.x : b.y) >> (8 * (k & 3))) * s;
      } else {
        const HeadRows rows = {(void *)in, 0, 0, true};
        load_head8<true>(f, rows, at * (LANES * 8) + d);
      }
    }
    const HeadRows &y = value ? p.v : p.k;
    const int64_t to = row * y.row_ld + h * y.head_ld + d;
    if (BF16) {
      *(uint4 *)((uint16_t *)y.data + to) = pack_bf16(f);
    } else {
      *(float4 *)((float *)y.data + to) = make_float4(f[0], f[1], f[2], f[3]);
      *(float4 *)((float *)y.data + to + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
}

template <bool BF16, bool Q8, int LANES>
hipError_t launch_kv_t(const KvArgs &a, bool write, hipStream_t s) {
  const int threads = std::min(256, (2 * a.c.heads * LANES + 63) / 64 * 64);
  hipLaunchKernelGGL((write ? kv_write_kernel<BF16, Q8, LANES> : kv_read_kernel<BF16, Q8, LANES>),
                     dim3((unsigned)a.rows), dim3((unsigned)threads), 0, s, a);
  return hipGetLastError();
}

template <bool BF16, bool Q8>
hipError_t launch_kv_d(const KvArgs &a, bool write, hipStream_t s) {
  switch (a.c.dim) {
    case 64: return launch_kv_t<BF16, Q8, 8>(a, write, s);
    case 128: return launch_kv_t<BF16, Q8, 16>(a, write, s);
    case 256: return launch_kv_t<BF16, Q8, 32>(a, write, s);
    default: return hipErrorInvalidConfiguration;
  }
}

hipError_t launch_kv(const HeadRows &k, const HeadRows &v, int64_t rows, const KvBatch &b,
                     const KvPages &c, int32_t *err_flag, bool write, hipStream_t s) {
  if (rows < 1 || rows > kMaxMixerRows) return hipErrorInvalidConfiguration;
  const KvArgs a = {k, v, b, c, (int32_t)rows, err_flag};
  if (k.bf16) return c.q8 ? launch_kv_d<true, true>(a, write, s) : launch_kv_d<true, false>(a, write, s);
  return c.q8 ? launch_kv_d<false, true>(a, write, s) : launch_kv_d<false, false>(a, write, s);
}

}  // namespace

hipError_t launch_kv_write(const HeadRows &k, const HeadRows &v, int64_t rows, const KvBatch &b,
                           const KvPages &c, int32_t *err_flag, hipStream_t s) {
  return launch_kv(k, v, rows, b, c, err_flag, true, s);
}
hipError_t launch_kv_read(const HeadRows &k, const HeadRows &v, int64_t rows, const KvBatch &b,
                          const KvPages &c, int32_t *err_flag, hipStream_t s) {
  return launch_kv(k, v, rows, b, c, err_flag, false, s);
}

}  // namespace llmcp_q8
