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
//
// A probability (of a Q8 value, times its scale) of a bf16 row is rounded to bf16
// before it meets the values: a rounding per weight of the sum next to the
// result's own, half again on the result's error; with two parts a prompt of 4096
// rows takes 304 us instead of 262, chunks 225 instead of 190, single rows 4 % more.
//
// Measured, a whole call: 32 sequences of one row, 16 heads over 4 of 256, 1.2 to 8
// thousand Q8 keys 93 to 101 us (307 MB, 3.3 TB/s), bf16 keys 160; one row over 2048
// bf16 keys 12.8; 4096 rows over themselves 262 (520 TFLOP/s); two chunks of 512
// rows of 32 heads over 8 of 128 over 8192 Q8 keys 190; 1024 f32 rows over
// themselves, 16 heads over 4 of 256, 160.
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
  int32_t snake;  // attention_many: order of the units
  float *part;    // [unit][split][tile rows] rows of dim + 4: the sum, maximum, total
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

// The pages of a sequence from one on, a lane each: a load and its wait for 64 of
// them.
struct PageWindow {
  int32_t pages = -1, from = -64;
};

// The cache's row of key k0 + lane (of KEYS; -1 for none), or (WHOLE: a page is a
// multiple of KEYS) of key k0; there are keys up to k_hi.
template <int KEYS, bool WHOLE>
__device__ __forceinline__ int32_t slot_of_key(const AttnArgs &p, const Unit &u, int32_t k_hi, int lane,
                                               int32_t k0, PageWindow &w) {
  const int32_t end = max(min(k0 + KEYS, k_hi) - 1, 0) / p.c.page_size;
  if (end >= w.from + 64) {
    w.from = k0 / p.c.page_size;
    w.pages = p.b.table[(int64_t)u.seq * p.b.max_pages + min(w.from + lane, p.b.max_pages - 1)];
  }
  const int32_t key = WHOLE ? k0 : k0 + (lane & (KEYS - 1));
  const int32_t index = min(key, max(k_hi - 1, 0)) / p.c.page_size;
  const int32_t page = WHOLE ? __builtin_amdgcn_readlane(w.pages, index - w.from) : __shfl(w.pages, index - w.from);
  int32_t slot = -1;
  if (key < k_hi) {
    if ((uint32_t)page < (uint32_t)p.c.pages)
      slot = (page * p.c.heads + u.head) * p.c.page_size + (key - index * p.c.page_size);
    else if (page != -1)
      *p.err_flag = 1;
  }
  return WHOLE ? __builtin_amdgcn_readfirstlane(slot) : slot;
}

// Which of a step's keys there are.
template <int KEYS, bool WHOLE>
__device__ __forceinline__ uint64_t keys_of(int32_t slot, int32_t k0, int32_t k_hi) {
  constexpr uint64_t all = KEYS == 64 ? ~0ull : (1ull << 32) - 1;
  if (!WHOLE) return __builtin_amdgcn_ballot_w64(slot >= 0) & all;
  const int32_t n = k_hi - k0;
  return slot < 0 || n <= 0 ? 0 : n >= KEYS ? all : (1ull << n) - 1;
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
template <int D, bool Q8, int PARTS, bool WHOLE>
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
  PageWindow window;

  for (int32_t k0 = k_lo + wave * kBlockKeys; k0 < k_hi; k0 += kWaves * kBlockKeys) {
    // lane k (and k + 32): the row of key k0 + k in the cache (WHOLE: the first's)
    const int32_t slot = slot_of_key<kBlockKeys, WHOLE>(p, u, k_hi, lane, k0, window);
    const uint32_t valid = (uint32_t)keys_of<kBlockKeys, WHOLE>(slot, k0, k_hi);
    const int32_t at = max(slot, 0);  // (a row of the cache for those without one)
    constexpr int BYTES = Q8 ? D : 2 * D;
    const uint8_t *const kp = (const uint8_t *)p.c.k + (WHOLE ? (int64_t)at * BYTES : 0);
    const uint8_t *const vp = (const uint8_t *)p.c.v + (WHOLE ? (int64_t)at * BYTES : 0);
    float ks_r = 0.0f, vs_r = 0.0f;
    if (Q8 && lane < 32) {
      ks_r = p.c.ks[WHOLE ? at + lane : at];
      vs_r = p.c.vs[WHOLE ? at + lane : at];
    }
    // V on its way
    v4u vr[VL];
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      constexpr int PER = Q8 ? D / 16 : D / 8;  // lanes a row
      if constexpr (WHOLE) {
        vr[i] = *(const v4u *)(vp + i * 1024 + lane * 16);
      } else {
        const int32_t row = __shfl(at, i * (64 / PER) + lane / PER);
        vr[i] = *(const v4u *)(vp + (int64_t)row * BYTES + lane % PER * 16);
      }
    }
    // scores
    v4f s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t *const kr = WHOLE ? kp + (16 * t + col) * BYTES + g * 16
                                      : kp + (int64_t)__shfl(at, 16 * t + col) * BYTES + g * 16;
      s[t] = v4f{0, 0, 0, 0};
      if constexpr (Q8) {
        v4u w[D / 64];
#pragma unroll
        for (int k = 0; k < D / 64; ++k)
          w[k] = *(const v4u *)(kr + k * 64);
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
          w[k] = *(const v4u *)(kr + k * 64);
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
    if (Q8 && lane < 32) {
      scale_lds[wave][0][lane] = ks_r;
      scale_lds[wave][1][lane] = vs_r;
    }
    __builtin_amdgcn_wave_barrier();
    // this lane's keys are 16 t + i from here
    const uint32_t has = valid >> (4 * g);
    const int32_t ends = sees - k0 - 4 * g;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      v4f vv = v4f{1, 1, 1, 1};
      if (Q8) {
        s[t] = s[t] * *(const v4f *)&scale_lds[wave][0][16 * t + 4 * g];
        vv = *(const v4f *)&scale_lds[wave][1][16 * t + 4 * g];
      }
      s[t] = s[t] * p.scale2;
#pragma unroll
      for (int i = 0; i < 4; ++i) vs[t][i] = vv[i];
    }
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = (has >> (16 * t + i) & 1) && 16 * t + i < ends;
          s[t][i] = in ? s[t][i] : -__builtin_inff();
          vs[t][i] = in ? vs[t][i] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j / 4][j % 4]);
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
      if (edge && !(valid >> r & 1)) vr[i] = v4u{0, 0, 0, 0};
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
        const int64_t row = WHOLE ? at + k : __builtin_amdgcn_readlane(at, k);
        const float pk = odd_lds[wave][k * kTileRows + col];
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const v2u w = *(const v2u *)((const uint16_t *)p.c.v + row * D + 16 * t + 4 * g);
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

  if constexpr (!Q8 && PARTS > 1) {
    // An infinity among the keys or values times a part of q or p that is 0 is NaN,
    // and stays in the sums: f32 rows whose sums are not finite take the wave's steps
    // again, key by key in f32. (The same steps once more, with a look at every
    // value, cost all calls registers: 12 to 24 % at dim 256.)
    float worst = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) worst = __builtin_fmaf(acc[t][i], 0.0f, worst);
    }
    worst += __shfl_xor(worst, 16);
    worst += __shfl_xor(worst, 32);
    if (__builtin_amdgcn_ballot_w64(!(worst == 0.0f))) {
      // (the tile's other rows keep theirs)
      const float m_had = m, l_had = l;
      m = -__builtin_inff(), l = 0.0f;
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        *(v4f *)(lds + (t * 64 + lane) * 16) = acc[t];
        acc[t] = v4f{0, 0, 0, 0};
      }
      window = PageWindow();
      // a quarter of the row's dims, g's
      const float *const mine = (const float *)p.q.data + (int64_t)(u.lo + i_row) * p.q.row_ld +
                                (int64_t)head * p.q.head_ld + g * (D / 4);
#pragma unroll 1
      for (int32_t k0 = k_lo + wave * kBlockKeys; k0 < k_hi; k0 += kWaves * kBlockKeys) {
        const int32_t slot = slot_of_key<kBlockKeys, WHOLE>(p, u, k_hi, lane, k0, window);
        const uint32_t valid = (uint32_t)keys_of<kBlockKeys, WHOLE>(slot, k0, k_hi);
        const int32_t at = max(slot, 0);
#pragma unroll 1
        for (int k = 0; k < kBlockKeys; ++k) {
          if (!(valid >> k & 1)) continue;
          const int64_t row = (WHOLE ? at + k : __builtin_amdgcn_readlane(at, k)) * (int64_t)D;
          const bool in = k0 + k < sees;
          float score = 0.0f;
#pragma unroll 4
          for (int d = 0; d < D / 4; d += 4) {
            const v4f x = *(const v4f *)(mine + d);
            const v2u w = *(const v2u *)((const uint16_t *)p.c.k + row + g * (D / 4) + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              score = __builtin_fmaf(x[i], bf16_to_float(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu), score);
          }
          score += __shfl_xor(score, 16);
          score += __shfl_xor(score, 32);
          score = in ? score * p.scale2 : -__builtin_inff();
          const float m_new = fmaxf(m, score), mf = finite_max(m_new);
          const float alpha = exp2_f32(m - mf), e = exp2_f32(score - mf);
          m = m_new;
          l = l * alpha + e;
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            const v2u w = *(const v2u *)((const uint16_t *)p.c.v + row + 16 * t + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = bf16_to_float(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
              acc[t][i] = __builtin_fmaf(e, in ? v : 0.0f, acc[t][i] * alpha);
            }
          }
        }
      }
      l = g == 0 ? l : 0.0f;  // (each lane has the row's whole sum)
      if (worst == 0.0f) {
        m = m_had, l = l_had;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] = *(const v4f *)(lds + (t * 64 + lane) * 16);
      }
    }
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

// ------------------------------------------------------- many rows (bf16) --

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kManyRows = 128;  // rows of a tile, 32 for each of four waves
constexpr int kManyThreads = 256;
// Workgroups of a CU: at dim 256 a wave's accumulator and queries alone take 192
// registers, and one workgroup of up to 512 each (no spills) is faster than
// two of 256.
constexpr int many_resident(int dim) { return dim == 256 ? 1 : 2; }

// Unit and part of a workgroup: the longest tiles (a sequence's last) first, a
// kv head's tiles on few XCDs; where all workgroups are resident at once, two per
// CU, the second half in ascending order, so that a CU's two add up to the same.
__device__ __forceinline__ int32_t many_unit(const AttnArgs &p, int32_t block, int32_t &split) {
  const int32_t head = block % p.c.heads, rest = block / p.c.heads;
  split = rest % p.splits;
  int32_t tile = rest / p.splits;
  if (p.snake && 2 * tile >= p.tiles) tile = p.tiles + (p.tiles + 1) / 2 - 1 - tile;
  return head * p.tiles + (p.tiles - 1 - tile);
}

// Two f32 as bf16 to nearest even, in one word.
__device__ __forceinline__ uint32_t round2(float lo, float hi) {
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  typedef float v2f __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{lo, hi}), v2bf));
}

// Tiles of 128 rows, 32 per wave, over keys that the workgroup brings to LDS in
// steps of 32 KT, a step ahead: bf16 pages directly, Q8 ones through registers,
// widened. S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 products. The
// maximum that exponents refer to moves only when one would pass 2^8 (f32 sums and
// bf16's 8 bits are the same at any such scale), so that the accumulator is
// seldom rescaled. WHOLE: a page is a multiple of a step, so a step's rows follow
// each other.
template <int D, bool Q8, int KT, bool WHOLE>
__global__ __launch_bounds__(kManyThreads, many_resident(D)) void attention_many_kernel(const AttnArgs p) {
  constexpr int STEPS = D / 16, DT = D / 32, KEYS = 32 * KT;
  constexpr int CHUNKS = D / 8, ROW = 2 * D;
  constexpr int LOADS = KEYS * CHUNKS / kManyThreads / (Q8 ? 2 : 1);  // 16 B of a page per thread, of K and of V
  constexpr int PER = Q8 ? D / 16 : D / 8;                            // lanes a row
  constexpr int TILE = KEYS * ROW;
  __shared__ __align__(16) uint8_t lds[2][2][TILE];
  __shared__ __align__(16) float scale_lds[2][2][KEYS];
  __shared__ int odd_lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  int32_t split;
  const int32_t unit = many_unit(p, blockIdx.x, split);
  const Unit u = find_unit(p, unit, kManyRows, lane);
  if (u.seq < 0) return;
  const int32_t step_keys = part_keys(u.seen, p.splits);
  const int32_t k_lo = split * step_keys, k_hi = min(u.seen, k_lo + step_keys);
  const int32_t parts = max(1, step_keys ? (u.seen + step_keys - 1) / step_keys : 0);
  if (split >= parts) return;

  auto seen_by = [&](int32_t pk) {
    return (int32_t)min(max(u.first + pk / p.group + 1, (int64_t)0), (int64_t)u.keys);
  };
  const int32_t last = u.n * p.group - 1, row0 = u.row + 32 * wave, packed = row0 + col;
  const bool live = packed <= last;
  const int32_t sees = live ? seen_by(packed) : 0;
  const int32_t all_see = seen_by(u.row);  // what every row of the tile sees
  const int32_t wave_all = seen_by(min(row0, last));
  const int32_t wave_seen = row0 > last ? 0 : seen_by(min(row0 + 31, last));
  // (the scale's sign goes into q; it is not 0, so that a masked score stays -inf)
  const float scale2 = fabsf(p.scale2);
  v8bf q[STEPS];
  {
    const int32_t i_row = live ? packed / p.group : 0;
    const int32_t head = u.head * p.group + (live ? packed - i_row * p.group : 0);
    const uint16_t *const at = (const uint16_t *)p.q.data + (int64_t)(u.lo + i_row) * p.q.row_ld + (int64_t)head * p.q.head_ld;
    const uint32_t sign = p.scale2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const v4u w = *(const v4u *)(at + 16 * s + 8 * h);
      q[s] = __builtin_bit_cast(v8bf, live ? w ^ sign : v4u{0, 0, 0, 0});
    }
  }
  float m = -__builtin_inff(), l = 0.0f;
  bool far = false;  // whether |m| is 2^20 or more
  v16f acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
  }

  // 16 B of a row in LDS: K's swizzle spreads the rows of one chunk, V's the
  // pairs of chunks of four rows
  auto k_swap = [](int r) { return r & (CHUNKS - 1) & 15; };
  auto v_swap = [](int r) { return 2 * (r & (CHUNKS / 2 - 1) & 7); };
  // Where this lane's operands are in a step's rows: chunk 2 k + h of K's row 32 t
  // + col at ka[k % 8] (a swizzle by exclusive or: 32 k at once), and of V's row 32
  // t + 16 c + 8 n + .. the columns 32 d + .. at va[d % 4]; what is left is a
  // constant offset.
  constexpr int KV_A = STEPS < 8 ? STEPS : 8, VV_A = DT < 4 ? DT : 4;
  uint32_t ka[KV_A], va[VV_A];
  {
    const int r = 4 * h + (lane >> 2 & 3), b = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
    const uint32_t kb = col * ROW + (h ^ k_swap(col)) * 16, vb = r * ROW + (b ^ v_swap(r)) * 16 + (lane & 1) * 8;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)&lds[0][0][0];
#pragma unroll
    for (int k = 0; k < KV_A; ++k) ka[k] = base + (kb ^ (32u * k));
#pragma unroll
    for (int d = 0; d < VV_A; ++d) va[d] = base + TILE + (vb ^ (64u * d));
  }

  PageWindow window;
  auto slot_at = [&](int32_t k0) { return slot_of_key<KEYS, WHOLE>(p, u, k_hi, lane, k0, window); };
  auto mask_of = [&](int32_t slot, int32_t k0) { return keys_of<KEYS, WHOLE>(slot, k0, k_hi); };
  constexpr uint64_t kAll = KEYS == 64 ? ~0ull : (1ull << 32) - 1;

  v4u kr[Q8 ? LOADS : 1], vr[Q8 ? LOADS : 1];
  float ks_r = 0.0f, vs_r = 0.0f;
  // A step's rows on their way (a row of the cache stands for those without one).
  // The chunk that a lane brings is the one whose place in LDS is the lane's.
  const int lr = lane / PER, lc = lane % PER;
  const uint32_t k_lane = lr * ROW + (lc ^ k_swap(lr)) * 16, v_lane = lr * ROW + (lc ^ v_swap(lr)) * 16;
  auto ask = [&](int32_t slot, int buf) {
    const int32_t at = max(slot, 0);
    if constexpr (WHOLE) {
      const uint8_t *const kp = (const uint8_t *)p.c.k + (int64_t)at * (Q8 ? D : ROW);
      const uint8_t *const vp = (const uint8_t *)p.c.v + (int64_t)at * (Q8 ? D : ROW);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int x = (wave * LOADS + i) * 64, r0 = x / PER;  // the load's first 16 B and row
        if constexpr (Q8) {
          kr[i] = *(const v4u *)(kp + r0 * D + lane * 16);
          vr[i] = *(const v4u *)(vp + r0 * D + lane * 16);
        } else {
          __builtin_amdgcn_global_load_lds(
              (__attribute__((address_space(1))) void *)(kp + r0 * ROW + (k_lane ^ (uint32_t)(k_swap(r0) * 16))),
              (lds_void *)(lds[buf][0] + x * 16), 16, 0, 0);
          __builtin_amdgcn_global_load_lds(
              (__attribute__((address_space(1))) void *)(vp + r0 * ROW + (v_lane ^ (uint32_t)(v_swap(r0) * 16))),
              (lds_void *)(lds[buf][1] + x * 16), 16, 0, 0);
        }
      }
      if (Q8 && wave == 0 && lane < KEYS) {
        ks_r = p.c.ks[at + lane];
        vs_r = p.c.vs[at + lane];
      }
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int x = (wave * LOADS + i) * 64, r = x / PER + lr;
        const int64_t row = __shfl(at, r);
        if constexpr (Q8) {
          kr[i] = *(const v4u *)((const int8_t *)p.c.k + row * D + lc * 16);
          vr[i] = *(const v4u *)((const int8_t *)p.c.v + row * D + lc * 16);
        } else {
          __builtin_amdgcn_global_load_lds(
              (__attribute__((address_space(1))) void *)((const uint16_t *)p.c.k + row * D + (lc ^ k_swap(r)) * 8),
              (lds_void *)(lds[buf][0] + x * 16), 16, 0, 0);
          __builtin_amdgcn_global_load_lds(
              (__attribute__((address_space(1))) void *)((const uint16_t *)p.c.v + row * D + (lc ^ v_swap(r)) * 8),
              (lds_void *)(lds[buf][1] + x * 16), 16, 0, 0);
        }
      }
      if (Q8 && wave == 0 && lane < KEYS) {
        ks_r = p.c.ks[at];
        vs_r = p.c.vs[at];
      }
    }
  };
  // A step's rows in LDS, as far as they were not brought there.
  auto keep = [&](uint64_t valid, int buf) {
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int x = (wave * LOADS + i) * 64;
        const int r = x / PER + lr;
        const bool has = valid >> r & 1;
        if (!has) vr[i] = v4u{0, 0, 0, 0};
        uint8_t *const kl = lds[buf][0] + r * ROW, *const vl = lds[buf][1] + r * ROW;
        *(v8bf *)(kl + (2 * lc ^ k_swap(r)) * 16) = widen8(kr[i][0], kr[i][1]);
        *(v8bf *)(kl + ((2 * lc + 1) ^ k_swap(r)) * 16) = widen8(kr[i][2], kr[i][3]);
        *(v8bf *)(vl + (2 * lc ^ v_swap(r)) * 16) = widen8(vr[i][0], vr[i][1]);
        *(v8bf *)(vl + ((2 * lc + 1) ^ v_swap(r)) * 16) = widen8(vr[i][2], vr[i][3]);
      }
      if (wave == 0 && lane < KEYS) {
        scale_lds[buf][0][lane] = ks_r;
        scale_lds[buf][1][lane] = vs_r;
      }
    }
  };

  int32_t slot = slot_at(k_lo);
  uint64_t valid = mask_of(slot, k_lo);
  ask(slot, 0);
  keep(valid, 0);
  if (threadIdx.x == 0) odd_lds = 0;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int buf = 0;
  for (int32_t k0 = k_lo; k0 < k_hi; k0 += KEYS, buf ^= 1) {
    slot = slot_at(k0 + KEYS);
    const uint64_t next_valid = mask_of(slot, k0 + KEYS);
    if (k0 + KEYS < k_hi) ask(slot, buf ^ 1);
    uint8_t *const vl = lds[buf][1];
    const uint32_t at_buf = buf * (2 * TILE);
    const bool edge_all = k0 + KEYS > all_see || valid != kAll;  // the same in the workgroup
    bool odd = false;
    if (!Q8 && edge_all) {
      // rows without a key to zeros; infinities and NaN, which some rows may
      // not see, out of the product
      constexpr int EACH = KEYS * CHUNKS / kManyThreads;
#pragma unroll 1
      for (int i = 0; i < EACH; ++i) {
        const int x = i * kManyThreads + threadIdx.x, r = x / CHUNKS;
        v4u w = *(const v4u *)(vl + x * 16);
        const bool has = valid >> r & 1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool lo = (w[k] & 0x7f80u) == 0x7f80u, hi = (w[k] & 0x7f800000u) == 0x7f800000u;
          odd |= has && (lo || hi);
          w[k] = has ? w[k] & (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu) : 0u;
        }
        *(v4u *)(vl + x * 16) = w;
      }
      if (odd) odd_lds = 1;
      __syncthreads();
    }
    const bool edge = k0 + KEYS > wave_all || valid != kAll;
    const bool idle = k0 >= wave_seen;  // (the causal end of the wave's rows)
    v16f s[KT];
    if (!idle) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
          const v8bf a = *(__attribute__((address_space(3))) const v8bf *)(uintptr_t)(
              ka[k % KV_A] + at_buf + 32 * t * ROW + k / KV_A * 256);
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[k], s[t], 0, 0, 0);
        }
      }
      if constexpr (Q8) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v4f ks = *(const v4f *)&scale_lds[buf][0][32 * t + 8 * j + 4 * h];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][4 * j + i] *= ks[i];
          }
        }
      }
      if (edge) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          // this lane's keys are 8 (i / 4) + i % 4 from here
          const uint32_t has = (uint32_t)(valid >> (32 * t)) >> (4 * h);
          const int32_t ends = sees - k0 - 32 * t - 4 * h;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = 8 * (i / 4) + i % 4;
            s[t][i] = (has >> k & 1) && k < ends ? s[t][i] : -__builtin_inff();
          }
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
      }
      top = fmaxf(top, __shfl_xor(top, 32)) * scale2;
      // Exponents are s * scale2 - m in one rounding. What m's own rounding leaves is the
      // same for all keys and small, but of scores from 2^20 on may grow past exp2:
      // those, and infinite ones, are rounded before m is taken off.
      float by = scale2, from = far ? 0.0f : finite_max(m);
      if (__builtin_amdgcn_ballot_w64(top > m + 8.0f || far)) {
        const float m_new = top > m + 8.0f ? top : m;
        const float alpha = m_new == m ? 1.0f : exp2_f32(m - finite_max(m_new));
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
        }
        from = finite_max(m);
        far = !(fabsf(from) < 0x1p20f);
        if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
          for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = far ? s[t][i] * scale2 - from : s[t][i];
          }
          by = far ? 1.0f : by;
          from = far ? 0.0f : from;
        }
      }
      v8bf pb[2 * KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v4f vs = *(const v4f *)&scale_lds[buf][1][32 * t + 8 * j + 4 * h];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = exp2_f32(__builtin_fmaf(s[t][4 * j + i], by, -from));
              l += e;
              // (a masked key's scale may be anything)
              s[t][4 * j + i] = edge && s[t][4 * j + i] == -__builtin_inff() ? 0.0f : e * vs[i];
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            s[t][i] = exp2_f32(__builtin_fmaf(s[t][i], by, -from));
            l += s[t][i];
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          v4u w;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = round2(s[t][8 * c + 2 * k], s[t][8 * c + 2 * k + 1]);
          pb[2 * t + c] = __builtin_bit_cast(v8bf, w);
        }
      }
#pragma unroll
      for (int tc = 0; tc < 2 * KT; ++tc) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          v4s half[2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
            half[n] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)(uintptr_t)(
                va[d % VV_A] + at_buf + (16 * tc + 8 * n) * ROW + d / VV_A * 256));
          const v8s both = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, both), pb[tc], acc[d], 0, 0, 0);
        }
      }
    }
    if (!Q8 && edge_all && odd_lds) {
      // Infinities and NaN among the values: added key by key, to the rows
      // that see them. (K's and V's rows make room for the probabilities.)
      __syncthreads();
      float *const pl = (float *)lds[buf][0] + wave * 1024;
#pragma unroll 1
      for (int t = 0; t < KT; ++t) {
        if (!idle) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            pl[(8 * (j / 4) + 4 * h + j % 4) * 32 + col] = KT > 1 && t ? s[KT - 1][j] : s[0][j];
        }
        __builtin_amdgcn_wave_barrier();
        window.from = -64;  // (the pages are asked for again)
        const int32_t mine = slot_at(k0);
        window.from = -64;
#pragma unroll 1
        for (int k = 0; k < 32 && !idle; ++k) {
          if (!(valid >> (32 * t + k) & 1)) continue;
          const int64_t row = WHOLE ? mine + 32 * t + k : __builtin_amdgcn_readlane(mine, 32 * t + k);
          const float pk = pl[k * 32 + col];
          const bool sees_it = k0 + 32 * t + k < sees;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const v2u w = *(const v2u *)((const uint16_t *)p.c.v + row * D + 32 * d + 8 * j + 4 * h);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = bf16_to_float(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
                if (!(fabsf(v) < __builtin_inff()) && sees_it) acc[d][4 * j + i] += pk * v;
              }
            }
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
      __syncthreads();
      if (threadIdx.x == 0) odd_lds = 0;
    }
    if (k0 + KEYS < k_hi) keep(next_valid, buf ^ 1);
    valid = next_valid;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

  l += __shfl_xor(l, 32);
  if (parts > 1) {
    if (!live) return;
    float *const to = p.part + ((int64_t)(unit * p.splits + split) * kManyRows + 32 * wave + col) * (D + 4);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(v4f *)(to + 32 * d + 8 * j + 4 * h) = v4f{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
    }
    if (h == 0) {
      to[D] = m;
      to[D + 1] = l;
    }
    return;
  }
  // through LDS (each wave its share), for whole rows
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint8_t *const mine = &lds[0][0][0] + wave * TILE;
  static_assert(TILE >= 32 * ROW, "the outputs fit");
#pragma unroll
  for (int d = 0; d < DT; ++d) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v2u w = v2u{round2(acc[d][4 * j] * inv, acc[d][4 * j + 1] * inv),
                        round2(acc[d][4 * j + 2] * inv, acc[d][4 * j + 3] * inv)};
      *(v2u *)(mine + col * ROW + ((4 * d + j) ^ k_swap(col)) * 16 + 8 * h) = w;
    }
  }
  __builtin_amdgcn_wave_barrier();
  constexpr int LANES = D / 8, AT_ONCE = 64 / LANES;
#pragma unroll 4
  for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
    const int r = r0 + lane / LANES, c = lane % LANES;
    const int32_t pk = row0 + r;
    if (pk > last) continue;
    const int32_t row = pk / p.group, hd = u.head * p.group + pk - row * p.group;
    *(v4u *)((uint16_t *)p.o.data + (int64_t)(u.lo + row) * p.o.row_ld + (int64_t)hd * p.o.head_ld + 8 * c) =
        *(const v4u *)(mine + r * ROW + (c ^ k_swap(r)) * 16);
  }
}

// The parts of the units whose keys were split, joined in order.
template <int D, int TILE>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs p) {
  const int32_t unit = blockIdx.x / (TILE / 16), sub = blockIdx.x % (TILE / 16);
  const Unit u = find_unit(p, unit, TILE, threadIdx.x & 63);
  if (u.seq < 0) return;
  const int32_t step_keys = part_keys(u.seen, p.splits);
  const int32_t parts = step_keys ? (u.seen + step_keys - 1) / step_keys : 0;
  if (parts <= 1) return;
  const float *const from = p.part + ((int64_t)unit * p.splits * TILE + 16 * sub) * (D + 4);
  const int32_t live = min(16, u.n * p.group - u.row - 16 * sub);
  // a part's weight in its row: a lane per part
  __shared__ float weight[16][64], whole[16];
  const int lane = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < live; r += 4) {
    v2u st = v2u{0xff800000u, 0u};  // (-inf, 0)
    if (lane < parts) st = *(const v2u *)(from + (int64_t)(lane * TILE + r) * (D + 4) + D);
    const float m = __uint_as_float(st[0]);
    float top = m;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const float f = exp2_f32(m - finite_max(top));
    float total = f * __uint_as_float(st[1]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
    weight[r][lane] = f;
    if (lane == 0) whole[r] = total == 0.0f ? 0.0f : 1.0f / total;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < live * (D / 4); i += 256) {
    const int r = i / (D / 4), c = i % (D / 4);
    const int32_t pk = u.row + 16 * sub + r;
    v4f sum = v4f{0, 0, 0, 0};
#pragma unroll 8
    for (int32_t s = 0; s < parts; ++s)
      sum = sum + *(const v4f *)(from + (int64_t)(s * TILE + r) * (D + 4) + 4 * c) * weight[r][s];
    sum = sum * whole[r];
    const int32_t row = pk / p.group, h = u.head * p.group + pk - row * p.group;
    const int64_t to = (int64_t)(u.lo + row) * p.o.row_ld + (int64_t)h * p.o.head_ld + 4 * c;
    if (p.o.bf16) *(v2u *)((uint16_t *)p.o.data + to) = v2u{pack2(sum[0], sum[1]), pack2(sum[2], sum[3])};
    else *(v4f *)((float *)p.o.data + to) = sum;
  }
}

template <int D, bool Q8>
hipError_t launch_attention_d(const AttnArgs &a, bool bf16, bool many, int32_t units, hipStream_t s) {
  const dim3 grid((unsigned)(units * a.splits)), wg(64 * kWaves);
  constexpr int KT = D == 256 ? 1 : 2;
  if (many && a.c.page_size % (32 * KT) == 0)
    hipLaunchKernelGGL((attention_many_kernel<D, Q8, KT, true>), grid, dim3(kManyThreads), 0, s, a);
  else if (many)
    hipLaunchKernelGGL((attention_many_kernel<D, Q8, KT, false>), grid, dim3(kManyThreads), 0, s, a);
  else if (bf16 && a.c.page_size % kBlockKeys == 0)
    hipLaunchKernelGGL((attention_few_kernel<D, Q8, 1, true>), grid, wg, 0, s, a);
  else if (bf16) hipLaunchKernelGGL((attention_few_kernel<D, Q8, 1, false>), grid, wg, 0, s, a);
  else if (a.c.page_size % kBlockKeys == 0)
    hipLaunchKernelGGL((attention_few_kernel<D, Q8, 3, true>), grid, wg, 0, s, a);
  else hipLaunchKernelGGL((attention_few_kernel<D, Q8, 3, false>), grid, wg, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  if (many) hipLaunchKernelGGL((attention_join_kernel<D, kManyRows>), dim3((unsigned)units * (kManyRows / 16)), wg, 0, s, a);
  else hipLaunchKernelGGL((attention_join_kernel<D, kTileRows>), dim3((unsigned)units), wg, 0, s, a);
  return hipGetLastError();
}

}  // namespace

AttentionPlan attention_plan(int64_t rows, int32_t heads, bool bf16, const KvBatch &b, const KvPages &c,
                             float scale, int32_t test_kernel, int32_t test_splits) {
  AttentionPlan plan;
  const int64_t group = heads / c.heads;
  const int64_t steps = ((int64_t)b.max_pages * c.page_size + kWaves * kBlockKeys - 1) / (kWaves * kBlockKeys);
  // Tiles of 128 rows where a sequence's rows (times the group) fill one on
  // average. Measured, us with tiles of 16 against 128: 16 heads over 4 of 256, 2048
  // keys, one sequence of 16 / 32 / 64 rows 28 / 30 / 44 against 30 / 32 / 37, eight
  // of them 59 / 110 / 135 against 40 / 45 / 92; 8192 Q8 keys, eight sequences of 16 /
  // 32 rows 107 / 195 against 154 / 101; 8 heads of 64, 1024 keys, one sequence of
  // 128 / 512 rows 15 / 25 against 17 / 22. (f32 rows, of three times the operands,
  // always take tiles of 16.)
  plan.many = bf16 && rows * group >= kManyRows * (int64_t)b.sequences;
  if (test_kernel && bf16) plan.many = test_kernel == 2;
  // Tiles of 128 rows mask before they scale: a scale of 0 would make a masked score
  // NaN, one next to it is not a normal number once it meets log2 e.
  if (!(fabsf(scale) >= 0x1p-100f)) plan.many = false;
  const int64_t tile = plan.many ? kManyRows : kTileRows;
  plan.tiles = (int32_t)(rows * group / tile + std::min<int64_t>(b.sequences, rows));
  const int64_t units = (int64_t)plan.tiles * c.heads;
  // Parts of the keys until there are 2 workgroups per CU (tiles of 128 rows) or 8
  // (of 16, two resident at a time: the rest evens out sequences of unlike lengths),
  // up to a lane each in the kernel that joins them.
  plan.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({steps, (plan.many ? 2 : 8) * cu_count() / units, 64}));
  if (test_splits > 0) plan.splits = (int32_t)std::min<int64_t>(steps, test_splits);
  if (plan.splits > 1) plan.part_floats = units * plan.splits * tile * (c.dim + 4);
  return plan;
}

hipError_t launch_attention(const HeadRows &q, const HeadRows &o, int64_t rows, int32_t heads,
                            const KvBatch &b, const KvPages &c, float scale, const AttentionPlan &plan,
                            float *part, int32_t *err_flag, hipStream_t s) {
  const int64_t units = (int64_t)plan.tiles * c.heads;
  if (rows < 1 || units < 1 || units * plan.splits > kMaxMixerBlocks || (plan.splits > 1 && !part))
    return hipErrorInvalidConfiguration;
  AttnArgs a = {q, o, b, c, (float)((double)scale * 1.4426950408889634), (int32_t)rows,
                heads / c.heads, plan.tiles, plan.splits,
                many_resident(c.dim) == 2 && units * plan.splits <= 2 * cu_count() ? 1 : 0, part, err_flag};
  const auto launch = c.dim == 64    ? (c.q8 ? launch_attention_d<64, true> : launch_attention_d<64, false>)
                      : c.dim == 128 ? (c.q8 ? launch_attention_d<128, true> : launch_attention_d<128, false>)
                      : c.dim == 256 ? (c.q8 ? launch_attention_d<256, true> : launch_attention_d<256, false>)
                                     : nullptr;
  return launch ? launch(a, q.bf16, plan.many, (int32_t)units, s) : hipErrorInvalidConfiguration;
}

}  // namespace llmcp_q8
