// q8_delta.hip -- the gated delta rule: per value head a state S [key_dim,
// value_dim], and per row of a sequence
//   u = beta (v - a S^T k),  S = a S + k u^T,  o = scale S^T q,  a = exp(g).
//
// Few rows go one after another (delta_rows_kernel). Many bf16 rows go in chunks
// of 64: with G the running sum of g in the chunk, S0 the state before it, and
//   L_ij = beta_i exp(G_i - G_j) k_i . k_j  (j < i),      T = (I + L)^-1,
//   A_ij = exp(G_i - G_j) q_i . k_j         (j <= i),
// the chunk's u, outputs and state are
//   U = T diag(beta) (V - diag(exp G) K S0),
//   O = diag(exp G) Q S0 + A U,
//   S = exp(G_63) S0 + K^T diag(exp(G_63 - G)) U.
// T and A do not depend on the state: delta_chunk_kernel makes them for all
// chunks side by side. delta_scan_kernel then walks a sequence's chunks with
// 16 columns of a head's state per workgroup.
//
// States and sums are f32 on bf16 matrix instructions: rows of q and k are
// exact in bf16 (their norms, the scale and the decays multiply f32 results),
// and an f32 factor goes in as parts of 8 bits: three of S0 towards U and of U
// towards the state (exact products), two of what only reaches a bf16 output. T
// meets V - K S0 in f32 matrix instructions.
//
// Bound by the states' stream (few rows: 32 sequences of one row and 32 heads of 128 x
// 128 24 us for 135 MB), by latency of one row (4.2 us, 1.4 for every further
// one) and of a chunk in the scan (2.2 us: three exchanges between the waves, whose
// operands come from LDS). 4096 rows of 32 heads: 168 us, traced apart (which takes
// longer) 35 for T and A (three workgroups per CU) and 140 for the scan's 64 chunks,
// its 256 workgroups one per CU.
#include <stddef.h>

#include <algorithm>

#include "q8_gemv.h"
#include "q8_mixer.h"

namespace llmcp_q8 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
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

// ------------------------------------------------------------- chunks --

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

constexpr int kChunk = 64;

// What a chunk of a head leaves for the scan, each block in the order in which
// a wave's lanes take it as an operand.
struct ChunkData {
  v4f t[10][64];        // T diag(beta): block (w, t <= w) at w (w + 1) / 2 + t
  v4u a[6][2][64];      // A in two parts: 16 rows w by 32 columns s <= w / 2
  float k_in[kChunk];   // exp(G_i) over |k_i|
  float q_in[kChunk];   // exp(G_i) scale over |q_i|
  float k_out[kChunk];  // exp(G_63 - G_i) over |k_i|
  float decay[64];      // exp(G_63), for every lane
  int32_t odd[64];      // whether the chunk has to go row by row
};
static_assert(sizeof(ChunkData) % 256 == 0, "aligned");
__device__ constexpr int a_block(int w, int s) { return (w / 2) * 2 + (w % 2) + (w / 2) * s + (w / 2 ? (w % 2) : 0); }
static_assert(a_block(0, 0) == 0 && a_block(1, 0) == 1 && a_block(2, 0) == 2 && a_block(2, 1) == 3 &&
              a_block(3, 0) == 4 && a_block(3, 1) == 5, "blocks of A");

struct ChunkArgs {
  DeltaLaunch l;
  ChunkData *data;     // [chunks of the window][heads]
  int32_t first, count; // the window's chunks
  int32_t slices;
};

// A chunk of the call: its sequence, the chunk's number there and its rows.
struct Chunk {
  int32_t seq = -1, index = 0, row = 0, live = 0;
};

// Chunk number c, sequences in order, each in whole chunks.
__device__ __forceinline__ Chunk find_chunk(const DeltaLaunch &l, int32_t c, int lane) {
  Chunk r;
  int32_t sum = 0;
  for (int32_t at = 0; at < l.sequences; at += 64) {
    RowRange range = {0, 0};
    if (at + lane < l.sequences) range = delta_range(l, at + lane);
    int32_t incl = (range.hi - range.lo + kChunk - 1) / kChunk;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int32_t o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    const int n = __popcll(__builtin_amdgcn_ballot_w64(sum + incl <= c));
    if (n < 64) {
      r.seq = at + n;
      r.index = c - (n ? sum + __builtin_amdgcn_readlane(incl, n - 1) : sum);
      r.row = __builtin_amdgcn_readlane(range.lo, n) + r.index * kChunk;
      r.live = min(kChunk, __builtin_amdgcn_readlane(range.hi, n) - r.row);
      break;
    }
    sum += __builtin_amdgcn_readlane(incl, 63);
  }
  return r;
}

// Chunks of the sequences before s.
__device__ __forceinline__ int32_t chunks_before(const DeltaLaunch &l, int32_t s, int lane) {
  int32_t sum = 0;
  for (int32_t at = 0; at < s; at += 64) {
    if (at + lane < s) {
      const RowRange range = delta_range(l, at + lane);
      sum += (range.hi - range.lo + kChunk - 1) / kChunk;
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  return __builtin_amdgcn_readfirstlane(sum);
}

__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// The upper halves of two words: their leading 8 bits as bf16.
__device__ __forceinline__ uint32_t upper2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float below(float x) { return x - high_half(__float_as_uint(x)); }

// Four values as PARTS bf16 parts of 8 bits each.
template <int PARTS>
__device__ __forceinline__ void split4(v4f x, v2u (&part)[PARTS]) {
#pragma unroll
  for (int n = 0; n < PARTS; ++n) {
    part[n] = v2u{upper2(x[0], x[1]), upper2(x[2], x[3])};
    if (n + 1 < PARTS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = below(x[i]);
    }
  }
}

__device__ __forceinline__ v8bf join(v2u a, v2u b) {
  return __builtin_bit_cast(v8bf, v4u{a[0], a[1], b[0], b[1]});
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

// T and A of a chunk and head. The products K K^T and Q K^T are exact products
// in f32 sums; wave w has rows 16 w .. 16 w + 15 of both. The inverse goes
// by 16 x 16 blocks: those on the diagonal by substitution, a column per lane,
// then wave j has column j of the blocks below, T_ij = -T_ii sum L_ik T_kj, a
// result's registers being the next product's operand.
template <int KD>
__global__ __launch_bounds__(256) void delta_chunk_kernel(const ChunkArgs p) {
  constexpr int KS = KD / 32, LD = 68;
  // K's rows make room for T: 53.5 KB, three workgroups per CU
  __shared__ __align__(16) float lm[kChunk][LD], am[kChunk][LD], tm[kChunk][LD];
  v4u (*const kt)[KS][64] = (v4u (*)[KS][64])&tm[0][0];
  static_assert(sizeof(v4u) * 4 * KS * 64 <= sizeof(float) * kChunk * LD, "K's rows fit");
  __shared__ double run[kChunk];
  __shared__ float kn[kChunk], qn[kChunk], bt[kChunk];
  __shared__ int odd;
  const DeltaLaunch &l = p.l;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int32_t c = blockIdx.x / l.heads, head = blockIdx.x - c * l.heads;
  const int32_t key_head = head / (l.heads / l.key_heads);
  const Chunk ch = find_chunk(l, p.first + c, lane);
  if (ch.seq < 0) return;
  if (threadIdx.x == 0) odd = 0;
  __syncthreads();
  const int my = 16 * wave + col;
  v8bf kr[KS], qr[KS];
  {
    const bool live = my < ch.live;
    const int64_t row = ch.row + (live ? my : 0);
    float kk = 0, qq = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v4u a = *(const v4u *)((const uint16_t *)l.k.data + row * l.k.row_ld + key_head * l.k.head_ld + 32 * s + 8 * g);
      v4u b = *(const v4u *)((const uint16_t *)l.q.data + row * l.q.row_ld + key_head * l.q.head_ld + 32 * s + 8 * g);
      if (!live) a = v4u{0, 0, 0, 0}, b = a;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kk = __builtin_fmaf(low_half(a[i]), low_half(a[i]), kk);
        kk = __builtin_fmaf(high_half(a[i]), high_half(a[i]), kk);
        qq = __builtin_fmaf(low_half(b[i]), low_half(b[i]), qq);
        qq = __builtin_fmaf(high_half(b[i]), high_half(b[i]), qq);
      }
      kt[wave][s][lane] = a;
      kr[s] = __builtin_bit_cast(v8bf, a);
      qr[s] = __builtin_bit_cast(v8bf, b);
    }
    kk += __shfl_xor(kk, 16);
    qq += __shfl_xor(qq, 16);
    kk += __shfl_xor(kk, 32);
    qq += __shfl_xor(qq, 32);
    float k1 = 1.0f, q1 = l.scale;
    if (l.normalize) {
      k1 = 1.0f / sqrtf(kk + l.eps);
      q1 = l.scale * (1.0f / sqrtf(qq + l.eps));
    }
    if (!live) k1 = 0.0f, q1 = 0.0f;
    if (g == 0) {
      kn[my] = k1;
      qn[my] = q1;
      if (!finite(kk) || !finite(qq) || !finite(k1) || !finite(q1)) odd = 1;
    }
  }
  if (wave == 0) {
    const bool live = lane < ch.live;
    const int64_t row = ch.row + (live ? lane : 0);
    float d = live ? l.decay[row * l.decay_ld + head] : 0.0f;
    const float b = live ? l.beta[row * l.beta_ld + head] : 0.0f;
    // what decays below e^-10000 is nothing; the sum stays finite
    if (d < -1e4f) d = -1e4f;
    // Where decays grow the state, what is written over later still stands in exp(G)
    // and in T, times up to e to the sum of the rises, and has to cancel there: by
    // e at most (two bits), else row by row.
    const float rise = wave_sum(fmaxf(d, 0.0f));
    if (!finite(d) || !finite(b) || !(rise <= 1.0f)) odd = 1;
    double sum = (double)d;
#pragma unroll
    for (int n = 1; n < 64; n *= 2) {
      const double o = __shfl_up(sum, n);
      if (lane >= n) sum += o;
    }
    run[lane] = sum;
    bt[lane] = b;
  }
  __syncthreads();
  // rows 16 wave + 4 g + i by columns 16 t + col
  double gi[4];
  float bi[4], ki[4], qi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * wave + 4 * g + i;
    gi[i] = run[r];
    ki[i] = kn[r];
    qi[i] = qn[r];
    bi[i] = bt[r] * ki[i];
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t > wave) continue;
    v4f kk = v4f{0, 0, 0, 0}, qk = kk;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const v8bf b = __builtin_bit_cast(v8bf, kt[t][s][lane]);
      kk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr[s], b, kk, 0, 0, 0);
      qk = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qr[s], b, qk, 0, 0, 0);
    }
    const int j = 16 * t + col;
    const double gj = run[j];
    const float kj = kn[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * wave + 4 * g + i;
      const float e = j <= r ? expf((float)(gi[i] - gj)) : 0.0f;
      lm[r][j] = j < r ? (bi[i] * kj) * (e * kk[i]) : 0.0f;
      am[r][j] = j <= r ? (qi[i] * kj) * (e * qk[i]) : 0.0f;
    }
  }
  __syncthreads();
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == col ? 1.0f : 0.0f;
#pragma unroll
      for (int k = 0; k < i; ++k) v = __builtin_fmaf(-lm[16 * wave + i][16 * wave + k], x[k], v);
      x[i] = v;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((i >> 2) == g) tm[16 * wave + i][my] = x[i];
  }
  __syncthreads();
  if (wave < 3) {
    v4f tc[4];  // column `wave` of T's blocks: rows 4 g + i, column col
#pragma unroll
    for (int i = 0; i < 4; ++i) tc[0][i] = tm[16 * wave + 4 * g + i][my];
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int bi_ = wave + d;
      if (bi_ > 3) continue;
      v4f sum = v4f{0, 0, 0, 0}, out = sum;
#pragma unroll
      for (int k = 0; k < d; ++k) {
        const v4f a = *(const v4f *)&lm[16 * bi_ + col][16 * (wave + k) + 4 * g];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], tc[k][i], sum, 0, 0, 0);
      }
      const v4f a = *(const v4f *)&tm[16 * bi_ + col][16 * bi_ + 4 * g];
#pragma unroll
      for (int i = 0; i < 4; ++i) out = __builtin_amdgcn_mfma_f32_16x16x4f32(-a[i], sum[i], out, 0, 0, 0);
      tc[d] = out;
#pragma unroll
      for (int i = 0; i < 4; ++i) tm[16 * bi_ + 4 * g + i][my] = out[i];
    }
  }
  __syncthreads();
  ChunkData &to = p.data[(int64_t)c * l.heads + head];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t > wave) continue;
    v4f x = *(const v4f *)&tm[my][16 * t + 4 * g];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= bt[16 * t + 4 * g + i];
    to.t[wave * (wave + 1) / 2 + t][lane] = x;
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (s > wave / 2) continue;
    v2u part[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v4f x = v4f{0, 0, 0, 0};
      if (2 * s + h <= wave) x = *(const v4f *)&am[my][16 * (2 * s + h) + 4 * g];
      split4<2>(x, part[h]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
      to.a[a_block(wave, s)][n][lane] = v4u{part[0][n][0], part[0][n][1], part[1][n][0], part[1][n][1]};
  }
  if (wave == 0) {
    const double last = run[kChunk - 1];
    const float e = expf((float)run[lane]);
    to.k_in[lane] = e * kn[lane];
    to.q_in[lane] = e * qn[lane];
    to.k_out[lane] = expf((float)(last - run[lane])) * kn[lane];
    to.decay[lane] = expf((float)last);
    to.odd[lane] = odd;
  }
}

// Blocks of a sequence in an order in which consecutive ones are on one XCD (the
// hardware deals them out over 8), so that a head's slices share its operands in
// one L2.
__device__ __forceinline__ int32_t on_one_xcd(int32_t block, int32_t blocks) {
  const int32_t x = block % 8, each = blocks / 8, rest = blocks % 8;
  return x * each + min(x, rest) + block / 8;
}

// A sequence's chunks of the window, 16 columns of a head's state per
// workgroup of eight waves. Waves 0 to 3 carry the state: wave w has rows 16 w ..
// of the chunk's U and tiles of 16 key dims of the state. Waves 4 to 7 have the
// same rows of the outputs, and bring K's rows to LDS. Between the waves
// everything passes through LDS in the order of the lanes, since a result's
// registers (rows 4 g + i, column col) are a lane's part of the next product's
// operand when the summed index is taken in that order. What a phase takes from
// memory is asked for a phase or more ahead, as it comes (a conversion or a row's
// mask there would wait for it; rows past the chunk's last repeat that one, and
// what a wave needs no block of is another's again: as many loads on every path,
// so that a wait counts those after it right); what it takes from LDS, together.
template <int KD>
__global__ __launch_bounds__(512) void delta_scan_kernel(const ChunkArgs p) {
  constexpr int KS = KD / 32, TILES = KD / 16, TW = TILES / 4, KL = KD / 32;
  __shared__ __align__(16) uint8_t kl[2][kChunk * KD * 2];
  __shared__ __align__(16) v2u sp[3][TILES][64], up[2][4][64], uo[3][4][64];
  __shared__ __align__(16) v4f bl[4][64];
  __shared__ float red[2][4][2][16];
  __shared__ float red3[2][4][3];
  __shared__ int odd_v[2][16];  // columns with an infinity or NaN among the chunk's values or U
  const DeltaLaunch &l = p.l;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int which = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool carries = which < 4;
  const int wave = which & 3, t256 = threadIdx.x & 255;
  const int32_t seq = blockIdx.x / (l.heads * p.slices);
  const int32_t block = on_one_xcd(blockIdx.x - seq * (l.heads * p.slices), l.heads * p.slices);
  const int32_t head = block / p.slices, slice = block - head * p.slices, sh = seq * l.heads + head;
  const int32_t key_head = head / (l.heads / l.key_heads);
  const int32_t column = slice * 16 + col;
  const RowRange range = delta_range(l, seq);
  const int32_t chunks = (range.hi - range.lo + kChunk - 1) / kChunk;
  const int32_t base = chunks_before(l, seq, lane) - p.first;  // the first chunk's place in the window
  const int32_t from = max(0, -base), to = min(chunks, p.count - base);
  // (a sequence without rows hands its state on in the first window)
  if (from >= to && !(chunks == 0 && p.first == 0 && l.state != l.new_state)) return;
  const int64_t at = (int64_t)sh * KD * l.value_dim + column;
  const float *const before = from > 0 ? l.new_state : l.state;
  v4f state[TW];
#pragma unroll
  for (int t = 0; t < TW; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      state[t][i] = before && carries ? before[at + (int64_t)(16 * (TW * wave + t) + 4 * g + i) * l.value_dim] : 0.0f;
  }
  auto rows_of = [&](int32_t n) { return min(kChunk, range.hi - range.lo - n * kChunk); };
  // Places in a chunk are 32-bit lane offsets from the chunk's first row (rows
  // are less than 2^22 values apart).
  const uint32_t q_ld = 2 * (uint32_t)l.q.row_ld, k_ld = 2 * (uint32_t)l.k.row_ld,
                 v_ld = 2 * (uint32_t)l.v.row_ld, o_ld = 2 * (uint32_t)l.o.row_ld;
  auto row_at = [&](const HeadRows &x, int32_t n, int32_t h) {
    return (uint8_t *)x.data + 2 * ((int64_t)(range.lo + n * kChunk) * x.row_ld + (int64_t)h * x.head_ld);
  };
  auto data_of = [&](int32_t n) { return (const uint8_t *)(p.data + ((int64_t)(base + n) * l.heads + head)); };
  const int64_t data_step = (int64_t)l.heads * sizeof(ChunkData);
  constexpr uint32_t kA = offsetof(ChunkData, a), kKIn = offsetof(ChunkData, k_in),
                     kQIn = offsetof(ChunkData, q_in), kKOut = offsetof(ChunkData, k_out),
                     kDecay = offsetof(ChunkData, decay), kOdd = offsetof(ChunkData, odd);
  // K in LDS: 16 B of a row by a swizzle that spreads both ways it is read
  auto place = [](int r, int c) { return r * KD * 2 + ((c ^ ((r & 7) << 1 | (r >> 3 & 1))) & (KD / 8 - 1)) * 16; };
  if (threadIdx.x < 32) odd_v[threadIdx.x / 16][threadIdx.x % 16] = 0;
  __syncthreads();
  const int32_t first = min(from, max(to - 1, 0));

  if (carries) {
    uint16_t vb[4];
    v4f k_in = v4f{0, 0, 0, 0}, tr[4], k_out = k_in;
    int32_t odd_chunk = 0;
    float decay = 0.0f;
    const uint8_t *vp = row_at(l.v, first, head), *dp = data_of(first);
    const uint32_t v_full = (16 * wave + 4 * g) * v_ld + 2 * column;
    auto ask_v = [&](uint32_t last) {
      if (last == kChunk - 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) vb[i] = *(const uint16_t *)(vp + (v_full + i * v_ld));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vb[i] = *(const uint16_t *)(vp + (min(16u * wave + 4 * g + i, last) * v_ld + 2 * column));
      }
      k_in = *(const v4f *)(dp + kKIn + 64 * wave + 16 * g);
      odd_chunk = *(const int32_t *)(dp + kOdd + 4 * lane);
      decay = *(const float *)(dp + kDecay + 4 * lane);
    };
    auto ask_t = [&]() {
      const uint8_t *const tp = dp + wave * (wave + 1) / 2 * 1024 + lane * 16;
#pragma unroll
      for (int t = 0; t < 4; ++t) tr[t] = *(const v4f *)(tp + min(t, wave) * 1024);
      k_out = *(const v4f *)(dp + kKOut + 64 * wave + 16 * g);
    };
    auto keep_state = [&]() {
#pragma unroll
      for (int t = 0; t < TW; ++t) {
        v2u part[3];
        split4<3>(state[t], part);
#pragma unroll
        for (int n = 0; n < 3; ++n) sp[n][TW * wave + t][lane] = part[n];
      }
    };
    if (from < to) {
      ask_v(rows_of(from) - 1);
      ask_t();
    }
    keep_state();
    for (int32_t n = from; n < to; ++n) {
      const int32_t live = rows_of(n);
      const int buf = n & 1;
      bool bad = false;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = 16 * wave + 4 * g + i < live ? bf16_to_float(vb[i]) : 0.0f;
        bad |= !finite(v[i]);
      }
      if (bad) odd_v[buf][col] = 1;
      const bool odd_all = __builtin_amdgcn_readfirstlane(odd_chunk) != 0;
      const float decay_now = decay;
      __syncthreads();  // the state's parts, K's rows and the vote are there
      v2u kh[KS][2], sv[3][TILES];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          kh[s][h] = *(const v2u *)(kl[buf] + place(16 * wave + col, 4 * s + 2 * h + (g >> 1)) + (g & 1) * 8);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          sv[i][2 * s] = sp[i][2 * s][lane];
          sv[i][2 * s + 1] = sp[i][2 * s + 1][lane];
        }
      }
      // An infinity or NaN would reach rows before its own, by 0 times it: its
      // column (every column, if it is not in the values) goes row by row below.
      bool mine_odd = odd_all || odd_v[buf][col];
      __builtin_amdgcn_sched_barrier(0);
      // V - diag(k_in) K S0
      {
        v4f ks[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) ks[i] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
          for (int i = 0; i < 3; ++i)
            ks[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(kh[s][0], kh[s][1]),
                                                            join(sv[i][2 * s], sv[i][2 * s + 1]), ks[i], 0, 0, 0);
        }
        v4f x = (ks[2] + ks[1]) + ks[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf(-k_in[i], x[i], mine_odd ? 0.0f : v[i]);
        bl[wave][lane] = x;
      }
      __builtin_amdgcn_sched_barrier(0);
      // (the last chunk asks for itself again)
      if (n + 1 < to) {
        dp += data_step;
        vp += (int64_t)kChunk * v_ld;
      }
      ask_v(rows_of(min(n + 1, to - 1)) - 1);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      if (threadIdx.x < 16) odd_v[buf ^ 1][threadIdx.x] = 0;  // (set after the next barrier but one)
      // U
      {
        v4f b[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) b[t] = bl[t][lane];
        v4f u = v4f{0, 0, 0, 0}, u2 = u;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (t > wave) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i % 2 == 0) u = __builtin_amdgcn_mfma_f32_16x16x4f32(tr[t][i], b[t][i], u, 0, 0, 0);
            else u2 = __builtin_amdgcn_mfma_f32_16x16x4f32(tr[t][i], b[t][i], u2, 0, 0, 0);
          }
        }
        u = u + u2;
        v2u part[2], out[3];
        v4f x = u;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] *= k_out[i];
        split4<3>(x, out);
#pragma unroll
        for (int i = 0; i < 3; ++i) uo[i][wave][lane] = out[i];
        split4<2>(u, part);
#pragma unroll
        for (int i = 0; i < 2; ++i) up[i][wave][lane] = part[i];
        // (as would U where it left f32, parts of an infinity being none; x is not
        // finite where u is not)
        if (!finite((x[0] + x[1]) + (x[2] + x[3]))) odd_v[buf][col] = 1;
      }
      __builtin_amdgcn_sched_barrier(0);
      ask_t();
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      // the state after the chunk
      mine_odd |= odd_v[buf][col] != 0;
      v4f old[TW];
      {
        v4s kt[TW][2][2];
        v2u ol[3][4];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = 16 * (2 * s + h) + 4 * g + (col >> 2);
              kt[t][s][h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) v4s *)(kl[buf] + place(r, 2 * (TW * wave + t) + (col >> 1 & 1)) + (col & 1) * 8));
            }
          }
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            ol[i][2 * s] = uo[i][2 * s][lane];
            ol[i][2 * s + 1] = uo[i][2 * s + 1][lane];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        v4f sum[TW][3];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int t = 0; t < TW; ++t) {
            const v8s both = __builtin_shufflevector(kt[t][s][0], kt[t][s][1], 0, 1, 2, 3, 4, 5, 6, 7);
            const v8bf a = __builtin_bit_cast(v8bf, both);
#pragma unroll
            for (int i = 0; i < 3; ++i)
              sum[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, join(ol[i][2 * s], ol[i][2 * s + 1]),
                                                                  s ? sum[t][i] : v4f{0, 0, 0, 0}, 0, 0, 0);
          }
        }
#pragma unroll
        for (int t = 0; t < TW; ++t) {
          const v4f x = (sum[t][2] + sum[t][1]) + sum[t][0];
          old[t] = state[t];
#pragma unroll
          for (int i = 0; i < 4; ++i) state[t][i] = __builtin_fmaf(decay_now, state[t][i], x[i]);
        }
      }
      if (__builtin_amdgcn_ballot_w64(mine_odd)) {
        for (int32_t r = 0; r < live; ++r) {
          const int64_t rr = range.lo + n * kChunk + r;
          const uint16_t *const kp = (const uint16_t *)l.k.data + rr * l.k.row_ld + key_head * l.k.head_ld;
          const uint16_t *const qp = (const uint16_t *)l.q.data + rr * l.q.row_ld + key_head * l.q.head_ld;
          float k[TW][4], pk = 0, pq = 0, kk = 0, qq = 0, kq = 0;
#pragma unroll
          for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int x = 16 * (TW * wave + t) + 4 * g + i;
              const float qv = bf16_to_float(qp[x]);
              k[t][i] = bf16_to_float(kp[x]);
              pk = __builtin_fmaf(old[t][i], k[t][i], pk);
              pq = __builtin_fmaf(old[t][i], qv, pq);
              kk = __builtin_fmaf(k[t][i], k[t][i], kk);
              qq = __builtin_fmaf(qv, qv, qq);
              kq = __builtin_fmaf(k[t][i], qv, kq);
            }
          }
#pragma unroll
          for (int x = 16; x < 64; x *= 2) {
            pk += __shfl_xor(pk, x);
            pq += __shfl_xor(pq, x);
            kk += __shfl_xor(kk, x);
            qq += __shfl_xor(qq, x);
            kq += __shfl_xor(kq, x);
          }
          const int b = r & 1;
          if (g == 0) {
            red[b][wave][0][col] = pk;
            red[b][wave][1][col] = pq;
          }
          if (lane == 0) {
            red3[b][wave][0] = kk;
            red3[b][wave][1] = qq;
            red3[b][wave][2] = kq;
          }
          __syncthreads();
          pk = pq = kk = qq = kq = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            pk += red[b][w][0][col];
            pq += red[b][w][1][col];
            kk += red3[b][w][0];
            qq += red3[b][w][1];
            kq += red3[b][w][2];
          }
          const float rk = l.normalize ? 1.0f / sqrtf(kk + l.eps) : 1.0f;
          const float rq = l.scale * (l.normalize ? 1.0f / sqrtf(qq + l.eps) : 1.0f);
          const float a = expf(l.decay[rr * l.decay_ld + head]), beta = l.beta[rr * l.beta_ld + head];
          const float vv = bf16_to_float(((const uint16_t *)l.v.data)[rr * l.v.row_ld + head * l.v.head_ld + column]);
          const float u = (vv - pk * (a * rk)) * beta;
          const float o = pq * (a * rq) + u * (kq * rk * rq);
#pragma unroll
          for (int t = 0; t < TW; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) old[t][i] = __builtin_fmaf(k[t][i] * rk, u, a * old[t][i]);
          }
          if (wave == 0 && g == 0 && mine_odd)
            ((uint16_t *)l.o.data)[rr * l.o.row_ld + head * l.o.head_ld + column] = float_to_bf16(o);
        }
#pragma unroll
        for (int t = 0; t < TW; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) state[t][i] = mine_odd ? old[t][i] : state[t][i];
        }
      }
      keep_state();
    }
#pragma unroll
    for (int t = 0; t < TW; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        l.new_state[at + (int64_t)(16 * (TW * wave + t) + 4 * g + i) * l.value_dim] = state[t][i];
    }
    return;
  }

  // ---- waves 4 to 7
  v2u q[KS][2];
  v4u kv[KL], ar[2][2];
  v4f q_in = v4f{0, 0, 0, 0};
  int32_t odd_chunk = 0;
  const uint8_t *qp = row_at(l.q, first, key_head), *kp = row_at(l.k, first, key_head), *dp = data_of(first);
  uint8_t *op = row_at(l.o, first, head);
  constexpr int PER = KD / 8, EACH = 256 / PER;  // threads a row of K, rows at a time
  const uint32_t q_full = (16 * wave + col) * q_ld + 8 * g, k_full = t256 / PER * k_ld + 16 * (t256 % PER);
  auto ask_q = [&](uint32_t last) {
    const uint8_t *const x = qp + (last == kChunk - 1 ? q_full : min(16u * wave + col, last) * q_ld + 8 * g);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) q[s][h] = *(const v2u *)(x + 64 * s + 32 * h);
    }
  };
  auto ask_k = [&](uint32_t last) {
    if (last == kChunk - 1) {
#pragma unroll
      for (int i = 0; i < KL; ++i) kv[i] = *(const v4u *)(kp + i * EACH * k_ld + k_full);
    } else {
#pragma unroll
      for (int i = 0; i < KL; ++i)
        kv[i] = *(const v4u *)(kp + (min((uint32_t)(i * EACH + t256 / PER), last) * k_ld + 16 * (t256 % PER)));
    }
  };
  auto keep_k = [&](int32_t n) {
    const int32_t live = rows_of(n);
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int r = i * EACH + t256 / PER;
      *(v4u *)(kl[n & 1] + place(r, t256 % PER)) = r < live ? kv[i] : v4u{0, 0, 0, 0};
    }
  };
  auto ask_a = [&]() {
    const uint8_t *const x = dp + kA + a_block(wave, 0) * 2048 + lane * 16;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ar[s][i] = *(const v4u *)(x + min(s, wave / 2) * 2048 + i * 1024);
    }
    q_in = *(const v4f *)(dp + kQIn + 64 * wave + 16 * g);
    odd_chunk = *(const int32_t *)(dp + kOdd + 4 * lane);
  };
  if (from < to) {
    ask_k(rows_of(from) - 1);
    ask_q(rows_of(from) - 1);
    ask_a();
    keep_k(from);
    if (from + 1 < to) kp += (int64_t)kChunk * k_ld;
    ask_k(rows_of(min(from + 1, to - 1)) - 1);
  }
  for (int32_t n = from; n < to; ++n) {
    const int32_t live = rows_of(n);
    const int buf = n & 1;
    const uint32_t last_next = rows_of(min(n + 1, to - 1)) - 1;
    __syncthreads();
    v2u sv[2][TILES];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) sv[i][t] = sp[i][t][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    v4f qs[2];
    qs[0] = qs[1] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qs[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(q[s][0], q[s][1]), join(sv[i][2 * s], sv[i][2 * s + 1]), qs[i], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (n + 1 < to) qp += (int64_t)kChunk * q_ld;
    ask_q(last_next);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    if (n + 1 < to) keep_k(n + 1);  // (the other buffer was read for the last time a chunk ago)
    if (n + 2 < to) kp += (int64_t)kChunk * k_ld;
    ask_k(rows_of(min(n + 2, to - 1)) - 1);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    const int odd_here = odd_v[buf][col];
    v2u ul[2][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ul[i][t] = up[i][t][lane];
    }
    __builtin_amdgcn_sched_barrier(0);
    v4f o = v4f{0, 0, 0, 0}, o2 = o;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > wave / 2) continue;
      const v8bf u0 = join(ul[0][2 * s], ul[0][2 * s + 1]), u1 = join(ul[1][2 * s], ul[1][2 * s + 1]);
      const v8bf a0 = __builtin_bit_cast(v8bf, ar[s][0]), a1 = __builtin_bit_cast(v8bf, ar[s][1]);
      o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, u0, o, 0, 0, 0);
      o2 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, u1, o2, 0, 0, 0);
      o2 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, u0, o2, 0, 0, 0);
    }
    o = o + o2;
    const v4f q0 = qs[0] + qs[1];
    const bool mine_odd = (__builtin_amdgcn_readfirstlane(odd_chunk) != 0) | (odd_here != 0);
    // (rows past the last are out of the buffer's range, without a branch)
    const auto to_o = __builtin_amdgcn_make_buffer_rsrc(op, 0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * wave + 4 * g + i;
      const uint32_t off = r < live && !mine_odd ? (uint32_t)r * o_ld + 2 * column : 0xffffff00u;
      __builtin_amdgcn_raw_buffer_store_b16(float_to_bf16(__builtin_fmaf(q_in[i], q0[i], o[i])), to_o, off, 0, 0);
    }
    op += (int64_t)kChunk * o_ld;
    if (n + 1 < to) dp += data_step;
    ask_a();
    if (__builtin_amdgcn_ballot_w64(mine_odd)) {
      for (int32_t r = 0; r < live; ++r) __syncthreads();  // (with the rows of the other waves)
    }
  }
}

template <bool BF16, int KD>
hipError_t launch_delta_k(const DeltaLaunch &l, hipStream_t s) {
  if (l.value_dim % 32 || (int64_t)l.sequences * l.heads * l.value_dim < 256 * 32)
    return launch_delta_rows<BF16, KD, 16>(l, s);
  return launch_delta_rows<BF16, KD, 32>(l, s);
}

// Chunks of all sequences, at most, and those of one window: what the
// workspace holds at a time (up to 192 MiB, a chunk of all heads at least).
int64_t delta_chunks(const DeltaLaunch &l) {
  return l.rows / kChunk + std::min<int64_t>(l.sequences, l.rows);
}
int64_t delta_window(const DeltaLaunch &l) {
  const int64_t fit = (192ll << 20) / ((int64_t)sizeof(ChunkData) * l.heads);
  return std::max<int64_t>(1, std::min(delta_chunks(l), fit));
}

template <int KD>
hipError_t launch_delta_chunks(const DeltaLaunch &l, void *workspace, hipStream_t s) {
  const int64_t total = delta_chunks(l), window = delta_window(l);
  ChunkArgs a = {l, (ChunkData *)workspace, 0, 0, l.value_dim / 16};
  const int64_t scan = (int64_t)l.sequences * l.heads * a.slices;
  if (window * l.heads > 0x7FFFFF || scan > 0x7FFFFF) return hipErrorInvalidConfiguration;
  for (int64_t first = 0; first < total; first += window) {
    a.first = (int32_t)first;
    a.count = (int32_t)std::min(window, total - first);
    hipLaunchKernelGGL((delta_chunk_kernel<KD>), dim3((unsigned)(a.count * l.heads)), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((delta_scan_kernel<KD>), dim3((unsigned)scan), dim3(512), 0, s, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

// Chunks from a mean of 10 rows per sequence on where the scan's workgroups are
// resident at once, of 16 where they are not. Measured on 32 heads of 128 x 128, us
// of 8 / 12 / 16 / 24 rows one after another against in chunks: one sequence 15 /
// 20 / 25 / 34 against 15 for all; 8 sequences 29 / 40 / 51 / 72 against 51; 32
// sequences 84 / 119 / 155 / 235 against 172. (f32 rows always go one after another:
// their products would not be exact in bf16.)
bool delta_chunked(const DeltaLaunch &l) {
  const int64_t least = (int64_t)l.sequences * l.heads * (l.value_dim / 16) <= cu_count() ? 10 : 16;
  return l.q.bf16 && l.rows >= least * l.sequences;
}

int64_t delta_workspace(const DeltaLaunch &l) {
  return delta_chunked(l) ? delta_window(l) * l.heads * (int64_t)sizeof(ChunkData) : 0;
}

hipError_t launch_delta(const DeltaLaunch &l, void *workspace, hipStream_t s) {
  if (delta_chunked(l)) {
    if (!workspace) return hipErrorInvalidConfiguration;
    return l.key_dim == 128 ? launch_delta_chunks<128>(l, workspace, s)
           : l.key_dim == 64 ? launch_delta_chunks<64>(l, workspace, s)
                             : hipErrorInvalidConfiguration;
  }
  if (l.key_dim == 128) return l.q.bf16 ? launch_delta_k<true, 128>(l, s) : launch_delta_k<false, 128>(l, s);
  if (l.key_dim == 64) return l.q.bf16 ? launch_delta_k<true, 64>(l, s) : launch_delta_k<false, 64>(l, s);
  return hipErrorInvalidConfiguration;
}

}  // namespace llmcp_q8
