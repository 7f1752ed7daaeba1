// q8_attention.hip -- attention of a chunk of new rows per sequence over the
// pages of a key/value cache.
//
// The products are taken transposed: scores S^T = K Q^T (keys by rows) and
// O^T += V^T P^T, so that a lane holds all of one row's statistics (running
// maximum, sum, and the factor its accumulator is scaled by), and the scores
// of a lane are, in order, its part of the next product's operand: P never
// leaves the registers.  Of f32 rows q and p are taken as three bf16 parts of 8
// bits each, whose products are exact.  Q8 keys and values go in as whole numbers, the
// key's scale multiplying the score and the value's the probability.
//
// The rows of a tile are the sequence's rows with the query heads of one kv
// head side by side: row i * group + g is head g of the group of row i, so
// keys and values are read once for the group.
#include <algorithm>

#include "q8_gemv.h"
#include "q8_mixer.h"

namespace llmcp_q8 {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

struct AttnArgs {
  HeadRows q, o;
  KvBatch b;
  KvPages c;
  float scale2;  // scale * log2(e)
  int32_t rows, group, tiles, splits;
  float *part;   // [unit][split][16] rows of dim + 4: the sum, maximum, total
  int32_t *err_flag;
};

constexpr int kTileRows = 16;   // rows of a tile
constexpr int kBlockKeys = 32;  // keys of a wave's step
constexpr int kWaves = 4;

// The tile that a unit is.
struct Unit {
  int32_t seq = -1, head = 0;
  int32_t lo = 0, n = 0;     // the sequence's rows
  int32_t row = 0;           // first packed row of the tile
  int32_t keys = 0;          // slots the sequence has
  int32_t seen = 0;          // keys that the tile's last row sees
  int64_t first = 0;         // position of the sequence's first row
};

// Unit u of the call, of `tiles` at most for each kv head: kv heads outermost,
// then sequences, then tiles of `tile` packed rows.  Every wave finds it by itself,
// the sequences' tiles summed over lanes.
__device__ __forceinline__ Unit find_unit(const AttnArgs &p, int32_t u, int32_t tile, int lane) {
  Unit r;
  r.head = u / p.tiles;
  u -= r.head * p.tiles;
  int32_t sum = 0, before = 0;
  for (int32_t at = 0; at < p.b.sequences; at += 64) {
    const int32_t s = at + lane;
    RowRange range = {0, 0};
    int32_t length = 0;
    if (s < p.b.sequences) {
      range = row_range(p.b.starts, s, p.rows);
      length = p.b.lengths[s];
    }
    int32_t incl = ((range.hi - range.lo) * p.group + tile - 1) / tile;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int32_t o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    const int n = __popcll(__builtin_amdgcn_ballot_w64(sum + incl <= u));
    if (n < 64) {
      r.seq = at + n;
      before = n ? sum + __builtin_amdgcn_readlane(incl, n - 1) : sum;
      r.lo = __builtin_amdgcn_readlane(range.lo, n);
      r.n = __builtin_amdgcn_readlane(range.hi, n) - r.lo;
      length = __builtin_amdgcn_readlane(length, n);
      r.first = (int64_t)length - r.n;
      r.keys = min(max(length, 0), p.b.max_pages * p.c.page_size);
      break;
    }
    sum += __builtin_amdgcn_readlane(incl, 63);
  }
  if (r.seq < 0) return r;
  r.row = (u - before) * tile;
  const int32_t last = min(r.row + tile, r.n * p.group) - 1;
  r.seen = (int32_t)min(max(r.first + last / p.group + 1, (int64_t)0), (int64_t)r.keys);
  return r;
}

// Keys per part of a unit whose tile sees `seen`, whole steps of a workgroup.
__device__ __forceinline__ int32_t part_keys(int32_t seen, int32_t splits) {
  constexpr int32_t step = kWaves * kBlockKeys;
  return ((seen + splits - 1) / splits + step - 1) / step * step;
}

// f32 as three bf16 parts, the sum exactly x (parts of an infinity or NaN: itself).
__device__ __forceinline__ void split3(float x, uint32_t (&part)[3]) {
  const uint32_t b = __float_as_uint(x);
  const bool odd = (b & 0x7f800000u) == 0x7f800000u;
  part[0] = b >> 16;
  if (odd && (b & 0x7fffffu)) part[0] |= 0x40u;
  const float r = x - __uint_as_float(b & 0xffff0000u);
  const uint32_t rb = __float_as_uint(r);
  part[1] = odd ? 0 : rb >> 16;
  const float t = r - __uint_as_float(rb & 0xffff0000u);
  part[2] = odd ? 0 : __float_as_uint(t) >> 16;
}

// Eight int8 values (two dwords) as bf16, exact.
__device__ __forceinline__ v8bf widen8(uint32_t a, uint32_t b) {
  v4u w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t d = i < 2 ? a : b;
    const int sh = i % 2 * 16;
    const float lo = (float)(int8_t)(d >> sh), hi = (float)(int8_t)(d >> (sh + 8));
    w[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
  return __builtin_bit_cast(v8bf, w);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return float_to_bf16(lo) | (uint32_t)float_to_bf16(hi) << 16;
}

__device__ __forceinline__ float exp2_f32(float x) { return __builtin_amdgcn_exp2f(x); }

// The lowest -inf stands for 0, so that -inf - (-inf) never is.
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// Tiles of 16 rows: a decode step's, or a short chunk's.  Each wave takes
// every fourth step of 32 keys of the workgroup's part by itself, with its own
// statistics and accumulator; they meet at the end.  K goes from memory to the
// operand's registers, V through LDS (written row by row, read
// transposed), each wave in its own 64 * D bytes.
template <int D, bool Q8, int PARTS>
__global__ __launch_bounds__(256, 2) void attention_few_kernel(const AttnArgs p) {
  constexpr int STEPS = D / 32, DT = D / 16;
  constexpr int CHUNKS = D / 8;                // 16 B of bf16 in a row
  constexpr int VL = Q8 ? D / 32 : D / 16;     // loads of 16 B per lane for 32 rows of V
  __shared__ __align__(16) uint8_t tile_lds[kWaves][64 * D];
  __shared__ float stat[kWaves][2][kTileRows];
  __shared__ __align__(16) float scale_lds[kWaves][2][kBlockKeys];
  __shared__ float odd_lds[kWaves][Q8 ? 1 : kBlockKeys * kTileRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const Unit u = find_unit(p, blockIdx.x / p.splits, kTileRows, lane);
  if (u.seq < 0) return;
  const int32_t split = blockIdx.x % p.splits;
  const int32_t step_keys = part_keys(u.seen, p.splits);
  const int32_t k_lo = split * step_keys, k_hi = min(u.seen, k_lo + step_keys);
  const int32_t parts = max(1, step_keys ? (u.seen + step_keys - 1) / step_keys : 0);
  if (split >= parts) return;

  // this lane's row of the tile
  const int32_t packed = u.row + col;
  const bool live = packed < u.n * p.group;
  const int32_t i_row = live ? packed / p.group : 0;
  const int32_t head = u.head * p.group + (live ? packed - i_row * p.group : 0);
  const int32_t sees = live ? (int32_t)min(max(u.first + i_row + 1, (int64_t)0), (int64_t)u.keys) : 0;
  // the fewest keys that a row of the tile sees
  const int32_t all_see = (int32_t)min(max(u.first + u.row / p.group + 1, (int64_t)0), (int64_t)u.keys);

  v8bf q[PARTS][STEPS];
  {
    const int64_t at = (int64_t)(u.lo + i_row) * p.q.row_ld + (int64_t)head * p.q.head_ld;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      // the key's values that this lane's operand holds in step s
      const int d = Q8 ? s / 2 * 64 + g * 16 + s % 2 * 8 : s * 32 + g * 8;
      if constexpr (PARTS == 1) {
        v4u w = *(const v4u *)((const uint16_t *)p.q.data + at + d);
        if (!live) w = v4u{0, 0, 0, 0};
        q[0][s] = __builtin_bit_cast(v8bf, w);
      } else {
        v4f f[2] = {*(const v4f *)((const float *)p.q.data + at + d),
                    *(const v4f *)((const float *)p.q.data + at + d + 4)};
        v4u w[3];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a[3], b[3];
          split3(live ? f[k / 2][k % 2 * 2] : 0.0f, a);
          split3(live ? f[k / 2][k % 2 * 2 + 1] : 0.0f, b);
#pragma unroll
          for (int n = 0; n < 3; ++n) w[n][k] = a[n] | b[n] << 16;
        }
#pragma unroll
        for (int n = 0; n < PARTS; ++n) q[n][s] = __builtin_bit_cast(v8bf, w[n]);
      }
    }
  }

  float m = -__builtin_inff(), l = 0.0f;
  v4f acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = v4f{0, 0, 0, 0};
  uint8_t *const lds = tile_lds[wave];

  for (int32_t k0 = k_lo + wave * kBlockKeys; k0 < k_hi; k0 += kWaves * kBlockKeys) {
    // lane k (and k + 32): the row of key k0 + k in the cache, -1 for none
    int32_t slot = -1;
    {
      const int32_t key = k0 + (lane & 31);
      if (key < k_hi) {
        const int32_t index = key / p.c.page_size;
        const int32_t page = page_at(p.b, p.c, u.seq, index, p.err_flag);
        if (page >= 0)
          slot = (page * p.c.heads + u.head) * p.c.page_size + (key - index * p.c.page_size);
      }
    }
    const uint32_t valid = (uint32_t)__builtin_amdgcn_ballot_w64(slot >= 0);
    const int32_t at = max(slot, 0);  // (a row of the cache for those without one)
    if (Q8) {
      if (lane < 32) {
        scale_lds[wave][0][lane] = p.c.ks[at] * p.scale2;
        scale_lds[wave][1][lane] = p.c.vs[at];
      }
    }
    // V on its way
    v4u vr[VL];
    bool has[VL];
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      constexpr int PER = Q8 ? D / 16 : D / 8;  // lanes a row
      const int r = i * (64 / PER) + lane / PER;
      const int32_t row = __shfl(at, r);
      has[i] = valid >> r & 1;
      vr[i] = *(const v4u *)((const uint8_t *)p.c.v + (int64_t)row * (Q8 ? D : 2 * D) + lane % PER * 16);
    }
    // scores
    v4f s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int32_t row = __shfl(at, 16 * t + col);
      s[t] = v4f{0, 0, 0, 0};
      if constexpr (Q8) {
        v4u w[D / 64];
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
          w[k] = *(const v4u *)((const int8_t *)p.c.k + (int64_t)row * D + k * 64 + g * 16);
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
          const v8bf a = widen8(w[k / 2][k % 2 * 2], w[k / 2][k % 2 * 2 + 1]);
#pragma unroll
          for (int n = 0; n < PARTS; ++n)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[n][k], s[t], 0, 0, 0);
        }
      } else {
        v4u w[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
          w[k] = *(const v4u *)((const uint16_t *)p.c.k + (int64_t)row * D + k * 32 + g * 8);
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
#pragma unroll
          for (int n = 0; n < PARTS; ++n)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[k]), q[n][k],
                                                           s[t], 0, 0, 0);
        }
      }
    }
    // scaled, masked; their maximum
    float vs[2][4];
    const bool edge = k0 + kBlockKeys > all_see || valid != 0xffffffffu;
    float top = -__builtin_inff();
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      v4f ks = v4f{p.scale2, p.scale2, p.scale2, p.scale2}, vv = v4f{1, 1, 1, 1};
      if (Q8) {
        ks = *(const v4f *)&scale_lds[wave][0][16 * t + 4 * g];
        vv = *(const v4f *)&scale_lds[wave][1][16 * t + 4 * g];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 16 * t + 4 * g + i;
        s[t][i] = s[t][i] * ks[i];
        vs[t][i] = vv[i];
        if (edge && !(k0 + k < sees && (valid >> k & 1))) {
          s[t][i] = -__builtin_inff();
          vs[t][i] = 0.0f;
        }
        top = fmaxf(top, s[t][i]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m_new = fmaxf(m, top), mf = finite_max(m_new);
    const float alpha = exp2_f32(m - mf);
    m = m_new;
    l *= alpha;
    float pr[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = exp2_f32(s[j / 4][j % 4] - mf);
      l += e;
      // (a masked key's e is 0 and its scale too, whatever the cache holds)
      pr[j] = Q8 ? e * vs[j / 4][j % 4] : e;
    }
    v8bf pb[PARTS];
    {
      v4u w[3];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (PARTS == 1) {
          w[0][k] = pack2(pr[2 * k], pr[2 * k + 1]);
        } else {
          uint32_t a[3], b[3];
          split3(pr[2 * k], a);
          split3(pr[2 * k + 1], b);
#pragma unroll
          for (int n = 0; n < 3; ++n) w[n][k] = a[n] | b[n] << 16;
        }
      }
#pragma unroll
      for (int n = 0; n < PARTS; ++n) pb[n] = __builtin_bit_cast(v8bf, w[n]);
    }
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] = acc[t] * alpha;
    }
    // V to LDS, rows without a key as zeros; pairs of chunks swapped by row, so
    // that the transposed reads of four rows meet different banks
    bool odd = false;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      constexpr int PER = Q8 ? D / 16 : D / 8;
      const int r = i * (64 / PER) + lane / PER, c = lane % PER;
      const int swap = 2 * (r & (CHUNKS / 2 - 1) & 7);
      if (!has[i]) vr[i] = v4u{0, 0, 0, 0};
      if constexpr (Q8) {
        *(v8bf *)(lds + r * 2 * D + ((2 * c) ^ swap) * 16) = widen8(vr[i][0], vr[i][1]);
        *(v8bf *)(lds + r * 2 * D + ((2 * c + 1) ^ swap) * 16) = widen8(vr[i][2], vr[i][3]);
      } else {
        if (edge) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool lo = (vr[i][k] & 0x7f80u) == 0x7f80u, hi = (vr[i][k] & 0x7f800000u) == 0x7f800000u;
            odd |= lo || hi;
            vr[i][k] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
          }
        }
        *(v4u *)(lds + r * 2 * D + (c ^ swap) * 16) = vr[i];
      }
    }
    __builtin_amdgcn_wave_barrier();
    if (!Q8 && edge && __builtin_amdgcn_ballot_w64(odd)) {
      // An infinity or NaN among values that some rows may not see: 0 times it
      // is NaN, so it stays out of the product and is added key by key, to the
      // rows that see it.
#pragma unroll
      for (int j = 0; j < 8; ++j)
        odd_lds[wave][(16 * (j / 4) + 4 * g + j % 4) * kTileRows + col] = pr[j];
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int k = 0; k < kBlockKeys; ++k) {
        if (!(valid >> k & 1)) continue;
        const int32_t row = __builtin_amdgcn_readlane(at, k);
        const float pk = odd_lds[wave][k * kTileRows + col];
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const v2u w = *(const v2u *)((const uint16_t *)p.c.v + (int64_t)row * D + 16 * t + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = bf16_to_float(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
            if (!(fabsf(v) < __builtin_inff()) && k0 + k < sees) acc[t][i] += pk * v;
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      // four keys of 16 columns per 16 lanes: rows 4 g .. 4 g + 3 of each half
      v4s half[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int r = 16 * n + 4 * g + (col >> 2);
        const int swap = 2 * (r & (CHUNKS / 2 - 1) & 7);
        const int c = 2 * t + (col >> 1 & 1);
        half[n] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4s *)(lds + r * 2 * D + (c ^ swap) * 16 + (col & 1) * 8));
      }
      typedef short v8s __attribute__((ext_vector_type(8)));
      const v8s both = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      const v8bf a = __builtin_bit_cast(v8bf, both);
#pragma unroll
      for (int n = 0; n < PARTS; ++n)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[n], acc[t], 0, 0, 0);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // the four waves' sums meet
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) {
    stat[wave][0][col] = m;
    stat[wave][1][col] = l;
  }
  float *const mine = (float *)lds;
#pragma unroll
  for (int t = 0; t < DT; ++t) *(v4f *)(mine + col * D + ((4 * t + g) ^ col) * 4) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < kTileRows * (D / 4); i += 256) {
    const int r = i / (D / 4), c = i % (D / 4);
    const int32_t pk = u.row + r;
    if (pk >= u.n * p.group) break;
    float top = stat[0][0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, stat[w][0][r]);
    const float mf = finite_max(top);
    v4f sum = v4f{0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_f32(stat[w][0][r] - mf);
      total += f * stat[w][1][r];
      sum = sum + *(const v4f *)((const float *)tile_lds[w] + r * D + (c ^ r) * 4) * f;
    }
    if (parts > 1) {
      float *const to = p.part + (int64_t)(blockIdx.x * kTileRows + r) * (D + 4);
      *(v4f *)(to + 4 * c) = sum;
      if (c == 0) {
        to[D] = top;
        to[D + 1] = total;
      }
    } else {
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      sum = sum * inv;
      const int32_t row = pk / p.group, h = u.head * p.group + pk - row * p.group;
      const int64_t to = (int64_t)(u.lo + row) * p.o.row_ld + (int64_t)h * p.o.head_ld + 4 * c;
      if (p.o.bf16) *(v2u *)((uint16_t *)p.o.data + to) = v2u{pack2(sum[0], sum[1]), pack2(sum[2], sum[3])};
      else *(v4f *)((float *)p.o.data + to) = sum;
    }
  }
}

// The parts of the units whose keys were split, joined in order.
template <int D>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs p) {
  const Unit u = find_unit(p, blockIdx.x, kTileRows, threadIdx.x & 63);
  if (u.seq < 0) return;
  const int32_t step_keys = part_keys(u.seen, p.splits);
  const int32_t parts = step_keys ? (u.seen + step_keys - 1) / step_keys : 0;
  if (parts <= 1) return;
  const float *const from = p.part + (int64_t)blockIdx.x * p.splits * kTileRows * (D + 4);
  for (int i = threadIdx.x; i < kTileRows * (D / 4); i += 256) {
    const int r = i / (D / 4), c = i % (D / 4);
    const int32_t pk = u.row + r;
    if (pk >= u.n * p.group) break;
    float top = -__builtin_inff();
    for (int32_t s = 0; s < parts; ++s) top = fmaxf(top, from[(int64_t)(s * kTileRows + r) * (D + 4) + D]);
    const float mf = finite_max(top);
    v4f sum = v4f{0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll 4
    for (int32_t s = 0; s < parts; ++s) {
      const float *const at = from + (int64_t)(s * kTileRows + r) * (D + 4);
      const float f = exp2_f32(at[D] - mf);
      total += f * at[D + 1];
      sum = sum + *(const v4f *)(at + 4 * c) * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    sum = sum * inv;
    const int32_t row = pk / p.group, h = u.head * p.group + pk - row * p.group;
    const int64_t to = (int64_t)(u.lo + row) * p.o.row_ld + (int64_t)h * p.o.head_ld + 4 * c;
    if (p.o.bf16) *(v2u *)((uint16_t *)p.o.data + to) = v2u{pack2(sum[0], sum[1]), pack2(sum[2], sum[3])};
    else *(v4f *)((float *)p.o.data + to) = sum;
  }
}

template <int D, bool Q8>
hipError_t launch_attention_d(const AttnArgs &a, bool bf16, int32_t units, hipStream_t s) {
  const dim3 grid((unsigned)(units * a.splits)), wg(64 * kWaves);
  if (bf16) hipLaunchKernelGGL((attention_few_kernel<D, Q8, 1>), grid, wg, 0, s, a);
  else hipLaunchKernelGGL((attention_few_kernel<D, Q8, 3>), grid, wg, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL((attention_join_kernel<D>), dim3((unsigned)units), wg, 0, s, a);
  return hipGetLastError();
}

}  // namespace

AttentionPlan attention_plan(int64_t rows, int32_t heads, const KvBatch &b, const KvPages &c) {
  AttentionPlan plan;
  const int64_t group = heads / c.heads;
  plan.tiles = (int32_t)(rows * group / kTileRows + std::min<int64_t>(b.sequences, rows));
  const int64_t units = (int64_t)plan.tiles * c.heads;
  const int64_t steps = ((int64_t)b.max_pages * c.page_size + kWaves * kBlockKeys - 1) / (kWaves * kBlockKeys);
  plan.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({steps, 2048 / units, 64}));
  if (plan.splits > 1) plan.part_floats = units * plan.splits * kTileRows * (c.dim + 4);
  return plan;
}

hipError_t launch_attention(const HeadRows &q, const HeadRows &o, int64_t rows, int32_t heads,
                            const KvBatch &b, const KvPages &c, float scale, const AttentionPlan &plan,
                            float *part, int32_t *err_flag, hipStream_t s) {
  const int64_t units = (int64_t)plan.tiles * c.heads;
  if (rows < 1 || units < 1 || units * plan.splits > 0x7FFFFF || (plan.splits > 1 && !part))
    return hipErrorInvalidConfiguration;
  AttnArgs a = {q, o, b, c, (float)((double)scale * 1.4426950408889634), (int32_t)rows,
                heads / c.heads, plan.tiles, plan.splits, part, err_flag};
  switch (c.dim) {
    case 64: return c.q8 ? launch_attention_d<64, true>(a, q.bf16, (int32_t)units, s)
                         : launch_attention_d<64, false>(a, q.bf16, (int32_t)units, s);
    case 128: return c.q8 ? launch_attention_d<128, true>(a, q.bf16, (int32_t)units, s)
                          : launch_attention_d<128, false>(a, q.bf16, (int32_t)units, s);
    case 256: return c.q8 ? launch_attention_d<256, true>(a, q.bf16, (int32_t)units, s)
                          : launch_attention_d<256, false>(a, q.bf16, (int32_t)units, s);
    default: return hipErrorInvalidConfiguration;
  }
}

}  // namespace llmcp_q8
