// q8_experts.hip -- products of Q8_1 rows with the Q8_0 weight of the expert
// that each row's slot names, grouped by expert.
//
// The function per row is the other GEMMs': exact int32 block dots, acc =
// fma(f32(I), sa * dw, acc) or acc + f32(I) * (sa * dw) in block order, so a
// slot's result is bit for bit what the linear of its expert gives.  A
// workgroup takes up to 16 RT slots of one expert and a range of the
// weight's columns; its four waves hold NB tiles of 16 columns each.
#include "q8_kernels.h"

#include <algorithm>

#include "q8_device.h"
#include "q8_gemv.h"

namespace llmcp_q8 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kStageBlocks = 16;               // blocks of K per stage
constexpr int kStageSteps = 4;                 // of four blocks each
constexpr int kTileQs = kStageBlocks * 512;    // values of 16 rows and a stage
constexpr int kTileScales = kStageBlocks * 64; // f32 scales of the same

// ------------------------------------------------------------ repack ---- //

// One thread per (tile, step, lane): the lane's MFMA operands of the step's
// four blocks and their scale (the layout: ExpertLayout in q8_common.h).
__global__ void repack_experts_kernel(const uint8_t *__restrict__ p4, uint8_t *__restrict__ out,
                                      int64_t experts, int64_t rows, int64_t blocks,
                                      ExpertLayout lay) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t steps = (int64_t)lay.stages * kStageSteps;  // scales cover whole stages
  const int lane = (int)(t & 63), li = lane & 15, lq = lane >> 4;
  const int64_t unit = t >> 6;
  const int64_t tile = unit / steps;
  const int step = (int)(unit - tile * steps);
  if (tile >= experts * lay.tiles) return;
  const int64_t e = tile / lay.tiles;
  const int64_t row = (tile - e * lay.tiles) * 16 + li;
  uint8_t *base = out + tile * lay.tile_bytes;
  uint32_t w[4][2] = {};
  uint16_t scale = 0;
  if (row < rows) {
    const int64_t g = (e * rows + row) / kLanes;
    const int r = (int)((e * rows + row) % kLanes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t b = 4 * step + i;
      if (b >= blocks) continue;
      const uint8_t *rec = p4 + (g * blocks + b) * kRecord;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        w[i][c] = *(const uint32_t *)(rec + 8 + 16 * (2 * lq + c) + 4 * r);
    }
    const int64_t b = 4 * step + lq;
    if (b < blocks) scale = *(const uint16_t *)(p4 + (g * blocks + b) * kRecord + 2 * r);
  }
  if (step < lay.steps) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
      *(uint4 *)(base + step * 2048 + p * 1024 + lane * 16) =
          make_uint4(w[2 * p][0], w[2 * p][1], w[2 * p + 1][0], w[2 * p + 1][1]);
  }
  *(uint16_t *)(base + lay.steps * 2048 + (step >> 2) * 512 + lane * 8 + 2 * (step & 3)) = scale;
}

// -------------------------------------------------------------- plan ---- //

// Slot s's group: its expert, or `experts` for a slot without one.
__device__ __forceinline__ int group_of(int id, int experts) {
  return (unsigned)id < (unsigned)experts ? id : experts;
}

// Slots sorted by group and the tiles to compute, by one workgroup: plan[0]
// = tiles, then {group, first, count} per tile, then the slots.  An id that
// is neither an expert nor -1 sets the error flag.  The order of a group's
// slots is that of the atomics; no result depends on it.
__global__ __launch_bounds__(1024) void expert_plan_kernel(const int32_t *__restrict__ ids,
                                                           int32_t slots, int32_t experts,
                                                           int32_t rows, int32_t max_tiles,
                                                           int32_t *__restrict__ plan,
                                                           int32_t *__restrict__ err) {
  __shared__ int count[kMaxExperts + 1], start[kMaxExperts + 2], tile0[kMaxExperts + 2];
  __shared__ int part[2][16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int i = t; i <= experts; i += 1024) count[i] = 0;
  __syncthreads();
  bool bad = false;
  for (int s = t; s < slots; s += 1024) {
    const int id = ids[s];
    bad |= id < -1 || id >= experts;
    atomicAdd(&count[group_of(id, experts)], 1);
  }
  if (__ballot(bad) && lane == 0) *err = 1;
  __syncthreads();
  // exclusive prefix sums of the slots and the tiles of the groups
  int base_s = 0, base_t = 0;
  for (int g0 = 0; g0 <= experts; g0 += 1024) {
    const int g = g0 + t;
    const int c = g <= experts ? count[g] : 0;
    const int n = (c + rows - 1) / rows;
    int ps = c, pt = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int us = __shfl_up(ps, d), ut = __shfl_up(pt, d);
      if (lane >= d) ps += us, pt += ut;
    }
    if (lane == 63) part[0][wave] = ps, part[1][wave] = pt;
    __syncthreads();
    int os = base_s, ot = base_t;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) os += part[0][w], ot += part[1][w];
      base_s += part[0][w], base_t += part[1][w];
    }
    if (g <= experts) start[g] = os + ps - c, tile0[g] = ot + pt - n;
    __syncthreads();
  }
  if (t == 0) plan[0] = min(base_t, max_tiles);
  int32_t *const tiles = plan + 4, *const order = tiles + 4 * max_tiles;
  for (int g = t; g <= experts; g += 1024) {
    const int c = count[g], n = (c + rows - 1) / rows;
    // a group's tiles alike, in whole 16-row tiles
    const int per = n ? ((c + 15) / 16 + n - 1) / n * 16 : 0;
    for (int i = 0; i < n; ++i) {
      const int at = tile0[g] + i;
      if (at >= max_tiles) break;
      const int f = min(i * per, c);
      *(v4i *)(tiles + 4 * at) = v4i{g, start[g] + f, min(per, c - f), 0};
    }
  }
  __syncthreads();
  for (int g = t; g <= experts; g += 1024) count[g] = 0;
  __syncthreads();
  for (int s = t; s < slots; s += 1024) {
    const int g = group_of(ids[s], experts);
    order[start[g] + atomicAdd(&count[g], 1)] = s;
  }
}

// -------------------------------------------------------------- GEMM ---- //

struct ExpertArgs {
  const int8_t *qa;    // Q8_1 rows [.., 32 blocks], dense
  const float *sa;     // their scales [.., blocks]
  int32_t per_row;     // slots per input row: slot s reads row s / per_row
  const int32_t *ids;  // [slots]
  int32_t *err;        // without a plan: set by an id that is out of range
  int32_t slots, experts;
  const int32_t *plan; // expert_plan_kernel's, or null: a tile per slot that
  int32_t max_tiles;   //   is the first of its group (or of 16 RT of them)
  const uint8_t *w0, *w1;
  ExpertLayout lay;
  int32_t blocks;      // K / 32
  int32_t rows;        // N of an expert
  int32_t n_groups;    // column ranges
  int32_t act;
  int32_t y_bf16, vec; // vec: y takes stores of four values
  void *y;             // [slots, ldy]
  int64_t ldy;
  int8_t *hq;          // DUAL: Q8_1 of the SwiGLU's rows, [slots, rows]
  float *hs;
};

template <int RT, int NB, bool DUAL>
struct ExpertShape {
  static constexpr int COLS = 64 * NB / (DUAL ? 2 : 1);  // columns of a workgroup
  static constexpr int STAGE = RT * (kTileQs + kTileScales);
  static constexpr int HLD = COLS + 4;                   // h rows in LDS
  static_assert(RT * 16 * HLD * 4 * (NB == 1 ? 2 : 1) <= 2 * STAGE, "h fits the ring");
};

// The slots of the workgroup's tile into `rows` (LDS): returns their number,
// 0 for a workgroup with nothing to do, and their group.
__device__ __forceinline__ int expert_tile(const ExpertArgs &p, int tile_rows, int &ng, int &group,
                                           int *rows, int *shared) {
  if (p.plan) {
    // equal shares of consecutive (tile, column range) pairs per XCD: a
    // tile's rows and an expert's weight are fetched into one L2
    const int total = __builtin_amdgcn_readfirstlane(p.plan[0]) * p.n_groups;
    const int share = (total + 7) / 8, i = blockIdx.x >> 3;
    const int at = (blockIdx.x & 7) * share + i;
    if (i >= share || at >= total) return 0;
    const int tile = at / p.n_groups;
    ng = at - tile * p.n_groups;
    const v4i e = *(const v4i *)(p.plan + 4 + 4 * (int64_t)tile);
    group = __builtin_amdgcn_readfirstlane(e[0]);
    const int count = __builtin_amdgcn_readfirstlane(e[2]);
    if ((int)threadIdx.x < count)
      rows[threadIdx.x] = p.plan[4 + 4 * (int64_t)p.max_tiles + e[1] + threadIdx.x];
    __syncthreads();
    return count;
  }
  const int s = blockIdx.x / p.n_groups;
  ng = blockIdx.x - s * p.n_groups;
  const int id = __builtin_amdgcn_readfirstlane(p.ids[s]);
  group = group_of(id, p.experts);
  if (ng == 0 && threadIdx.x == 0 && (id < -1 || id >= p.experts)) *p.err = 1;
  if (threadIdx.x < 64) {
    // the slots of this group before s, and from s on
    int before = 0, after = 0;
    const int lane = threadIdx.x;
    for (int c = 0; c < p.slots; c += 64) {
      const int i = c + lane;
      const bool hit = i < p.slots && group_of(p.ids[i], p.experts) == group;
      before += __popcll(__ballot(hit && i < s));
    }
    if (before % tile_rows == 0)
      for (int c = s & ~63; c < p.slots; c += 64) {
        const int i = c + lane;
        const bool hit = i >= s && i < p.slots && group_of(p.ids[i], p.experts) == group;
        const uint64_t m = __ballot(hit);
        const int at = after + __popcll(m & ((1ull << lane) - 1));
        if (hit && at < tile_rows) rows[at] = i;
        after += __popcll(m);
      }
    if (lane == 0) *shared = min(after, tile_rows);
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*shared);
}

// The workgroup's sums over NRT 16-row tiles of slots (NRT <= RT).
template <int NRT, int RT, int NB, bool FMA, bool DUAL>
__device__ __forceinline__ void expert_sums(const ExpertArgs &p, int count, const int *rows,
                                            const uint8_t *const (&wt)[NB], uint8_t *smem,
                                            float (&acc)[NB][RT][4]) {
  constexpr int STAGE = ExpertShape<RT, NB, DUAL>::STAGE;
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4;
  const int steps = p.lay.steps, stages = p.lay.stages;
  // ---- rows into LDS: thread (row li, 16 B piece g and g + 16 of 32)
  const int g = tid >> 4;
  const int8_t *src[NRT];
  const float *ssrc[NRT];
  bool live[NRT];
#pragma unroll
  for (int r = 0; r < NRT; ++r) {
    const int i = 16 * r + li;
    live[r] = i < count;
    const int64_t row = rows[live[r] ? i : 0] / p.per_row;
    src[r] = p.qa + row * p.blocks * kBlock;
    ssrc[r] = p.sa + row * p.blocks;
  }
  v4i av[NRT][2];
  float as[NRT];
  auto load_rows = [&](int stage) __attribute__((always_inline)) {
    const int b0 = stage * kStageBlocks;
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int b = min(b0 + 8 * h + (g >> 1), p.blocks - 1);
        av[r][h] = *(const v4i *)(src[r] + b * kBlock + 16 * (g & 1));
      }
      as[r] = ssrc[r][min(b0 + g, p.blocks - 1)];
    }
  };
  auto store_rows = [&](int stage) __attribute__((always_inline)) {
    uint8_t *const at = smem + (stage & 1) * STAGE;
    const int b0 = stage * kStageBlocks;
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int b = 8 * h + (g >> 1);
        v4i v = av[r][h];
        if (!live[r] || b0 + b >= p.blocks) v = v4i{0, 0, 0, 0};
        uint8_t *const to = at + r * kTileQs + (b >> 1) * 1024 + 2 * (g & 1) * 256 + li * 16 + (b & 1) * 8;
        *(v2i *)to = v2i{v[0], v[1]};
        *(v2i *)(to + 256) = v2i{v[2], v[3]};
      }
      const bool ok = live[r] && b0 + g < p.blocks;
      *(float *)(at + RT * kTileQs + r * kTileScales + g * 64 + li * 4) = ok ? as[r] : 0.0f;
    }
  };
  // ---- weights: a stage of each tile in registers, each step's replaced by
  // the next stage's as soon as its MFMAs have taken it
  v4i wq[NB][kStageSteps][2];
  uint2 wd[NB], wdn[NB];
  auto load_step = [&](int stage, int q) __attribute__((always_inline)) {
    const int st = min(stage * kStageSteps + q, steps - 1);
#pragma unroll
    for (int t = 0; t < NB; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        wq[t][q][j] = __builtin_nontemporal_load(
            (const v4i *)(wt[t] + (uint32_t)st * 2048u + j * 1024 + lane * 16));
  };
  auto load_scales = [&](int stage, uint2 (&d)[NB]) __attribute__((always_inline)) {
    const int sg = min(stage, stages - 1);
#pragma unroll
    for (int t = 0; t < NB; ++t)
      d[t] = *(const uint2 *)(wt[t] + (uint32_t)steps * 2048u + sg * 512 + lane * 8);
  };
  load_rows(0);
  load_scales(0, wd);
#pragma unroll
  for (int q = 0; q < kStageSteps; ++q) load_step(0, q);
  store_rows(0);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NB; ++t)
#pragma unroll
    for (int r = 0; r < NRT; ++r)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[t][r][v] = 0.0f;

  for (int s = 0; s < stages; ++s) {
    const uint8_t *const at = smem + (s & 1) * STAGE;
    load_rows(s + 1 < stages ? s + 1 : s);
    load_scales(s + 1, wdn);
#pragma unroll
    for (int q = 0; q < kStageSteps; ++q) {
      if (s * kStageSteps + q >= steps) break;
#pragma unroll
      for (int r = 0; r < NRT; ++r) {
        const v4i a0 = *(const v4i *)(at + r * kTileQs + (2 * q) * 1024 + lane * 16);
        const v4i a1 = *(const v4i *)(at + r * kTileQs + (2 * q + 1) * 1024 + lane * 16);
        const float sa = *(const float *)(at + RT * kTileQs + r * kTileScales + (4 * q + lq) * 64 + li * 4);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
          const uint32_t dw = q < 2 ? wd[t].x : wd[t].y;
          const v16f z = {};
          const v16f f = __builtin_amdgcn_mfma_f32_16x16x1f32(
              half_bits_to_float((q & 1) ? dw >> 16 : dw & 0xffffu), sa, z, 0, 0, 0);
          v4i c[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v4i w = wq[t][q][j >> 1], a = j < 2 ? a0 : a1;
            const v2i wv = (j & 1) ? v2i{w[2], w[3]} : v2i{w[0], w[1]};
            const v2i xv = (j & 1) ? v2i{a[2], a[3]} : v2i{a[0], a[1]};
            c[j] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, wv),
                                                         __builtin_bit_cast(long, xv),
                                                         v4i{0, 0, 0, 0}, 0, 0, 0);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const float dot = (float)c[j][v];
              if (FMA) {
                acc[t][r][v] = __builtin_fmaf(dot, f[4 * j + v], acc[t][r][v]);
              } else {
                const float contrib = dot * f[4 * j + v];
                acc[t][r][v] = acc[t][r][v] + contrib;
              }
            }
        }
      }
      load_step(s + 1, q);
    }
#pragma unroll
    for (int t = 0; t < NB; ++t) wd[t] = wdn[t];
    if (s + 1 < stages) store_rows(s + 1);
    __syncthreads();
  }
}

template <int NRT, int RT, int NB, bool FMA, bool DUAL>
__device__ __forceinline__ void expert_tile_run(const ExpertArgs &p, int ng, int group, int count,
                                                const int *rows, uint8_t *smem) {
  typedef ExpertShape<RT, NB, DUAL> Sh;
  const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = ng * Sh::COLS;
  // the wave's tiles of 16 columns (a wave past the last repeats it)
  const uint8_t *wt[NB];
  int tile[NB];
#pragma unroll
  for (int t = 0; t < NB; ++t) {
    const bool up = DUAL && (NB == 2 ? t == 1 : (wave & 1) != 0);
    const int i = DUAL ? (NB == 2 ? wave : wave >> 1) : wave * NB + t;
    tile[t] = col0 / 16 + i;
    const int c = min(tile[t], p.lay.tiles - 1);
    wt[t] = (up ? p.w1 : p.w0) + (int64_t)group * p.lay.expert_bytes() + (uint32_t)c * (uint32_t)p.lay.tile_bytes;
  }
  float acc[NB][RT][4];
  expert_sums<NRT, RT, NB, FMA, DUAL>(p, count, rows, wt, smem, acc);

  if constexpr (!DUAL) {
#pragma unroll
    for (int t = 0; t < NB; ++t) {
      const int n = tile[t] * 16 + 4 * lq;
#pragma unroll
      for (int r = 0; r < NRT; ++r) {
        float o[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = acc[t][r][v];
        activate_array(o, p.act);
        const int i = 16 * r + li;
        if (i >= count || n >= p.rows) continue;
        const int64_t at = (int64_t)rows[i] * p.ldy + n;
        if (p.y_bf16) {
          uint16_t h[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) h[v] = float_to_bf16(o[v]);
          uint16_t *const y = (uint16_t *)p.y + at;
          if (p.vec) {
            *(uint2 *)y = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = h[v];
          }
        } else {
          float *const y = (float *)p.y + at;
          if (p.vec) {
            *(float4 *)y = make_float4(o[0], o[1], o[2], o[3]);
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = o[v];
          }
        }
      }
    }
  } else {
    // h = silu(gate) * up through LDS (the ring's place: the last barrier of
    // the sums lies behind every read of it), then its Q8_1 by rows
    float *const hb = (float *)smem, *const ub = hb + RT * 16 * Sh::HLD;
    const int c = 16 * (NB == 2 ? wave : wave >> 1) + 4 * lq;
    const bool bf16 = p.y_bf16 != 0;
#pragma unroll
    for (int r = 0; r < NRT; ++r) {
      float o[4];
      if constexpr (NB == 2) {
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = acc[0][r][v];
        activate_array(o, ACT_SILU);
#pragma unroll
        for (int v = 0; v < 4; ++v)
          o[v] = bf16 ? bf16_to_float(float_to_bf16(o[v])) * bf16_to_float(float_to_bf16(acc[NB - 1][r][v]))
                      : o[v] * acc[NB - 1][r][v];
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = acc[0][r][v];
        if (!(wave & 1)) activate_array(o, ACT_SILU);
        if (bf16) {
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = bf16_to_float(float_to_bf16(o[v]));
        }
      }
      float *const to = (NB == 1 && (wave & 1)) ? ub : hb;
      *(float4 *)(to + (16 * r + li) * Sh::HLD + c) = make_float4(o[0], o[1], o[2], o[3]);
    }
    __syncthreads();
    constexpr int NBLK = Sh::COLS / 32;
    const int l8 = threadIdx.x & 7;
    for (int u = threadIdx.x >> 3; u < NRT * 16 * NBLK; u += 32) {
      const int r = u / NBLK, b = u - r * NBLK;
      float4 v = *(const float4 *)(hb + r * Sh::HLD + 32 * b + 4 * l8);
      if constexpr (NB == 1) {
        const float4 w = *(const float4 *)(ub + r * Sh::HLD + 32 * b + 4 * l8);
        v = make_float4(v.x * w.x, v.y * w.y, v.z * w.z, v.w * w.w);
      }
      if (bf16)
        v = make_float4(bf16_to_float(float_to_bf16(v.x)), bf16_to_float(float_to_bf16(v.y)),
                        bf16_to_float(float_to_bf16(v.z)), bf16_to_float(float_to_bf16(v.w)));
      int32_t q;
      float s;
      quantize_block8(v, true, &q, &s);
      const int n = col0 + 32 * b;
      if (r < count && n < p.rows) {
        const int64_t slot = rows[r];
        *(int32_t *)(p.hq + slot * p.rows + n + 4 * l8) = q;
        if (l8 == 0) p.hs[slot * (p.rows / kBlock) + n / kBlock] = s;
      }
    }
  }
}

// Rows of slots without an expert: zeros.
template <int COLS>
__device__ __forceinline__ void expert_zero_rows(const ExpertArgs &p, int ng, int count, const int *rows) {
  for (int i = threadIdx.x; i < count * COLS; i += 256) {
    const int r = i / COLS, n = ng * COLS + i % COLS;
    if (n >= p.rows) continue;
    const int64_t at = (int64_t)rows[r] * p.ldy + n;
    if (p.y_bf16) ((uint16_t *)p.y)[at] = 0;
    else ((float *)p.y)[at] = 0.0f;
  }
}

template <int RT, int NB, bool FMA, bool DUAL>
__global__ __launch_bounds__(256, 2) void expert_kernel(const ExpertArgs p) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef ExpertShape<RT, NB, DUAL> Sh;
  __shared__ __align__(1024) uint8_t smem[2 * Sh::STAGE];
  __shared__ int rows[16 * RT], shared;
  int ng = 0, group = 0;
  const int count = expert_tile(p, 16 * RT, ng, group, rows, &shared);
  if (count == 0) return;
  if (group >= p.experts) {
    if constexpr (!DUAL) expert_zero_rows<Sh::COLS>(p, ng, count, rows);
    return;
  }
  const int nrt = (count + 15) >> 4;
  if (RT == 1 || nrt == 1) return expert_tile_run<1, RT, NB, FMA, DUAL>(p, ng, group, count, rows, smem);
  if constexpr (RT >= 2)
    if (RT == 2 || nrt == 2) return expert_tile_run<2, RT, NB, FMA, DUAL>(p, ng, group, count, rows, smem);
  if constexpr (RT >= 4) {
    if (nrt == 3) return expert_tile_run<3, RT, NB, FMA, DUAL>(p, ng, group, count, rows, smem);
    return expert_tile_run<4, RT, NB, FMA, DUAL>(p, ng, group, count, rows, smem);
  }
#endif
}

// ----------------------------------------------------------- combine ---- //

// y[t] = residual[t] + sum over its slots j, in order, of w[t, j] * o[t, j]:
// an f32 FMA chain from the residual (or zero), rounded once; slots without
// an expert add nothing.  Four columns per thread.
template <bool BF16>
__global__ __launch_bounds__(256) void expert_combine_kernel(
    const void *__restrict__ o, const int32_t *__restrict__ ids, const float *__restrict__ w,
    int32_t top_k, int32_t experts, int64_t m, int32_t cols, const void *residual, int64_t ldr,
    int raligned, void *y, int64_t ldy, int yaligned) {
  const uint32_t quads = cols / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / quads;
  if (t >= m) return;
  const int c = 4 * (int)(i - t * quads);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (residual) v = load_act4(residual, t * ldr + c, BF16, raligned != 0);
  for (int j = 0; j < top_k; ++j) {
    const int64_t s = t * top_k + j;
    const int id = ids[s];
    if ((unsigned)id >= (unsigned)experts) continue;
    const float f = w ? w[s] : 1.0f;
    const float4 x = load_act4(o, s * cols + c, BF16, true);
    v.x = __builtin_fmaf(f, x.x, v.x);
    v.y = __builtin_fmaf(f, x.y, v.y);
    v.z = __builtin_fmaf(f, x.z, v.z);
    v.w = __builtin_fmaf(f, x.w, v.w);
  }
  if (BF16) {
    uint16_t *const to = (uint16_t *)y + t * ldy + c;
    const uint16_t a = float_to_bf16(v.x), b = float_to_bf16(v.y), d = float_to_bf16(v.z),
                   e = float_to_bf16(v.w);
    if (yaligned) {
      *(uint2 *)to = make_uint2(a | (uint32_t)b << 16, d | (uint32_t)e << 16);
    } else {
      to[0] = a, to[1] = b, to[2] = d, to[3] = e;
    }
  } else {
    float *const to = (float *)y + t * ldy + c;
    if (yaligned) {
      *(float4 *)to = v;
    } else {
      to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    }
  }
}

// ------------------------------------------------------------- route ---- //

// Order of f32 logits as unsigned: NaN and -inf (never chosen) 0, then
// ascending with the value.
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
  return !(v > -__builtin_inff()) ? 0u : (v == 0.0f ? 0x80000000u : k);
}

// One wave per row, PER logits per lane (logit i in lane i % 64): top_k
// rounds, each the largest (key, lowest index) of the wave.
template <bool BF16, int PER>
__global__ __launch_bounds__(256) void route_kernel(const void *__restrict__ logits, int64_t ld,
                                                    int64_t m, int32_t experts, int32_t top_k,
                                                    int normalize, float scale,
                                                    int32_t *__restrict__ ids,
                                                    float *__restrict__ weights) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= m) return;  // uniform per wave
  float l[PER];
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = 64 * i + lane;
    l[i] = -__builtin_inff();
    if (e < experts)
      l[i] = BF16 ? bf16_to_float(((const uint16_t *)logits)[row * ld + e])
                  : ((const float *)logits)[row * ld + e];
    key[i] = logit_key(l[i]);
  }
  // round 0's winner is the row's maximum: exp(l - max) needs it first
  float top = 0.0f, total = 0.0f, mine = 0.0f;
  int id = -1;
  for (int j = 0; j < top_k; ++j) {
    // the largest key first, then the lowest index
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint64_t k = (uint64_t)key[i] << 32 | (uint32_t)~(64 * i + lane);
      best = key[i] && k > best ? k : best;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, d);
      best = o > best ? o : best;
    }
    if (best == 0) break;  // only masked logits are left
    const int e = (int)~(uint32_t)best;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (64 * i + lane == e) v = l[i], key[i] = 0;
    v = __shfl(v, e & 63);
    if (j == 0) top = v;
    // (the maximum itself gives 1, also where it is infinite)
    const float p = v == top ? 1.0f : exp_f32(v - top);
    total += p;
    if (lane == j) id = e, mine = p;
  }
  if (!normalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (l[i] > -__builtin_inff()) total += l[i] == top ? 1.0f : exp_f32(l[i] - top);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor(total, d);
  }
  if (lane < top_k) {
    ids[row * top_k + lane] = id;
    weights[row * top_k + lane] = id >= 0 ? mine / total * scale : 0.0f;
  }
}

}  // namespace

hipError_t launch_repack_experts(const uint8_t *p4, uint8_t *out, int64_t experts, int64_t rows,
                                 int64_t cols, hipStream_t s) {
  const ExpertLayout lay = expert_layout(rows, cols);
  // a launch holds fewer than 2^32 threads: experts in as many as it takes
  const int64_t per = (int64_t)lay.tiles * lay.stages * kStageSteps * 64;
  const int64_t most = std::max<int64_t>(1, ((1ll << 31) / per));
  for (int64_t e = 0; e < experts; e += most) {
    const int64_t n = std::min(most, experts - e);
    hipLaunchKernelGGL(repack_experts_kernel, dim3((unsigned)((n * per + 255) / 256)), dim3(256), 0, s,
                       p4 + e * rows * (cols / kBlock) * 34, out + e * lay.expert_bytes(), n, rows,
                       cols / kBlock, lay);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

int32_t expert_tile_rows(int64_t slots, int64_t experts) {
  const int64_t mean = slots / std::max<int64_t>(1, std::min(slots, experts));
  return mean <= 10 ? 16 : mean <= 20 ? 32 : 64;
}

int64_t expert_max_tiles(int64_t slots, int64_t experts) {
  return slots / expert_tile_rows(slots, experts) + std::min(slots, experts + 1);
}

int64_t expert_plan_ints(int64_t slots, int64_t experts) {
  return slots <= kDirectSlots ? 0 : 4 + 4 * expert_max_tiles(slots, experts) + slots;
}

hipError_t launch_expert_plan(const int32_t *ids, int64_t slots, int32_t experts, int32_t *plan,
                              int32_t *err_flag, hipStream_t s) {
  hipLaunchKernelGGL(expert_plan_kernel, dim3(1), dim3(1024), 0, s, ids, (int32_t)slots, experts,
                     expert_tile_rows(slots, experts), (int32_t)expert_max_tiles(slots, experts), plan,
                     err_flag);
  return hipGetLastError();
}

template <int RT, int NB, bool DUAL>
static hipError_t launch_shape(ExpertArgs &a, bool fma, hipStream_t s) {
  constexpr int COLS = ExpertShape<RT, NB, DUAL>::COLS;
  a.n_groups = (a.rows + COLS - 1) / COLS;
  const int64_t wgs = a.plan ? ((int64_t)a.max_tiles * a.n_groups + 7) / 8 * 8
                             : (int64_t)a.slots * a.n_groups;
  // HIP bounds a grid's work-items by 2^32 - 1
  if (wgs * 256 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  if (fma)
    hipLaunchKernelGGL((expert_kernel<RT, NB, true, DUAL>), dim3((unsigned)wgs), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((expert_kernel<RT, NB, false, DUAL>), dim3((unsigned)wgs), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_experts(const ExpertLaunch &l, hipStream_t s) {
  ExpertArgs a = {};
  a.qa = l.qa;
  a.sa = l.sa;
  a.per_row = l.per_row;
  a.ids = l.ids;
  a.err = l.err_flag;
  a.slots = (int32_t)l.slots;
  a.experts = l.experts;
  a.plan = l.plan;
  a.max_tiles = (int32_t)expert_max_tiles(l.slots, l.experts);
  a.w0 = l.w;
  a.w1 = l.up;
  a.lay = expert_layout(l.rows, l.cols);
  a.blocks = (int32_t)(l.cols / kBlock);
  a.rows = (int32_t)l.rows;
  a.act = l.activation;
  a.y_bf16 = l.bf16 ? 1 : 0;
  a.y = l.y;
  a.ldy = l.ldy;
  a.vec = (uintptr_t)l.y % (l.bf16 ? 8 : 16) == 0 && l.ldy % 4 == 0 ? 1 : 0;
  a.hq = l.hq;
  a.hs = l.hs;
  const bool dual = l.up != nullptr;
  switch (expert_tile_rows(l.slots, l.experts)) {
    case 16:
      return dual ? launch_shape<1, 1, true>(a, l.fma, s) : launch_shape<1, 1, false>(a, l.fma, s);
    case 32:
      return dual ? launch_shape<2, 2, true>(a, l.fma, s) : launch_shape<2, 2, false>(a, l.fma, s);
    default:
      return dual ? launch_shape<4, 2, true>(a, l.fma, s) : launch_shape<4, 2, false>(a, l.fma, s);
  }
}

hipError_t launch_expert_combine(const void *o, const int32_t *ids, const float *w, int32_t top_k,
                                 int32_t experts, int64_t m, int64_t cols, const void *residual,
                                 int64_t ldr, void *y, int64_t ldy, bool bf16, hipStream_t s) {
  const int64_t wgs = (m * (cols / 4) + 255) / 256;
  if (wgs * 256 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  const int64_t a = bf16 ? 8 : 16;
  const int ra = (uintptr_t)residual % a == 0 && ldr % 4 == 0;
  const int ya = (uintptr_t)y % a == 0 && ldy % 4 == 0;
  if (bf16)
    hipLaunchKernelGGL((expert_combine_kernel<true>), dim3((unsigned)wgs), dim3(256), 0, s, o, ids, w,
                       top_k, experts, m, (int32_t)cols, residual, ldr, ra, y, ldy, ya);
  else
    hipLaunchKernelGGL((expert_combine_kernel<false>), dim3((unsigned)wgs), dim3(256), 0, s, o, ids, w,
                       top_k, experts, m, (int32_t)cols, residual, ldr, ra, y, ldy, ya);
  return hipGetLastError();
}

template <bool BF16>
static hipError_t launch_route_t(const void *logits, int64_t ld, int64_t m, int32_t experts,
                                 int32_t top_k, bool normalize, float scale, int32_t *ids,
                                 float *weights, hipStream_t s) {
  const dim3 grid((unsigned)((m + 3) / 4)), wg(256);
  const int n = normalize ? 1 : 0;
  if (experts <= 64)
    hipLaunchKernelGGL((route_kernel<BF16, 1>), grid, wg, 0, s, logits, ld, m, experts, top_k, n, scale, ids, weights);
  else if (experts <= 128)
    hipLaunchKernelGGL((route_kernel<BF16, 2>), grid, wg, 0, s, logits, ld, m, experts, top_k, n, scale, ids, weights);
  else if (experts <= 256)
    hipLaunchKernelGGL((route_kernel<BF16, 4>), grid, wg, 0, s, logits, ld, m, experts, top_k, n, scale, ids, weights);
  else
    hipLaunchKernelGGL((route_kernel<BF16, 16>), grid, wg, 0, s, logits, ld, m, experts, top_k, n, scale, ids, weights);
  return hipGetLastError();
}

hipError_t launch_route(const void *logits, bool bf16, int64_t ld, int64_t m, int32_t experts,
                        int32_t top_k, bool normalize, float scale, int32_t *ids, float *weights,
                        hipStream_t s) {
  if ((m + 3) / 4 * 256 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  return bf16 ? launch_route_t<true>(logits, ld, m, experts, top_k, normalize, scale, ids, weights, s)
              : launch_route_t<false>(logits, ld, m, experts, top_k, normalize, scale, ids, weights, s);
}

}  // namespace llmcp_q8
