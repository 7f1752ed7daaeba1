// q8_experts.hip -- products of Q8_1 rows with the Q8_0 weight of the expert
// that each row's slot names, grouped by expert.
//
// The function per row is the other GEMMs': exact int32 block dots, acc =
// fma(f32(I), sa * dw, acc) or acc + f32(I) * (sa * dw) in block order, so a
// slot's result is bit for bit what the linear of its expert gives.  A
// workgroup takes up to 4, 8, 16, 32 or 64 slots of one expert (a token's
// alone: one) and a range of the weight's columns.
#include "q8_kernels.h"

#include <algorithm>

#include "q8_device.h"
#include "q8_gemv.h"

namespace llmcp_q8 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v32f __attribute__((ext_vector_type(32)));

// ------------------------------------------------------------ repack ---- //

// One thread per (tile, step, lane): 16 B of two of the step's four blocks and
// one scale (the layout: ExpertLayout in q8_common.h).
__global__ void repack_experts_kernel(const uint8_t *__restrict__ p4, uint8_t *__restrict__ out,
                                      int64_t experts, int64_t rows, int64_t blocks,
                                      ExpertLayout lay) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int lane = (int)(t & 63), li = lane & 15, lq = lane >> 4;
  const int64_t unit = t >> 6;
  const int64_t tile = unit / lay.steps;
  const int step = (int)(unit - tile * lay.steps);
  if (tile >= experts * lay.tiles) return;
  const int64_t e = tile / lay.tiles;
  const int64_t row = (tile - e * lay.tiles) * 16 + li;
  uint8_t *base = out + tile * lay.tile_bytes();
  const int64_t g = (e * rows + row) / kLanes;
  const int r = (int)((e * rows + row) % kLanes);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    uint32_t w[4] = {0, 0, 0, 0};
    const int64_t b = 4 * step + 2 * p + (lq >> 1);
    if (row < rows && b < blocks) {
      const uint8_t *rec = p4 + (g * blocks + b) * kRecord;
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = *(const uint32_t *)(rec + 8 + 16 * (4 * (lq & 1) + c) + 4 * r);
    }
    *(uint4 *)(base + step * 2048 + p * 1024 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int64_t b = 4 * step + lq;
  uint16_t scale = 0;
  if (row < rows && b < blocks) scale = *(const uint16_t *)(p4 + (g * blocks + b) * kRecord + 2 * r);
  *(uint16_t *)(base + lay.steps * 2048 + step * 128 + li * 8 + lq * 2) = scale;
}

// -------------------------------------------------------------- plan ---- //

// Slot s's group: its expert, or `experts` for a slot without one.
__device__ __forceinline__ int group_of(int id, int experts) {
  return (unsigned)id < (unsigned)experts ? id : experts;
}

// The sum of v over this lane and those before it (lane moves: a permute
// through LDS takes over 100 clocks).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_plus(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_plus<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v = dpp_plus<0x112, 0xf>(v);
  v = dpp_plus<0x114, 0xf>(v);
  v = dpp_plus<0x118, 0xf>(v);
  v = dpp_plus<0x142, 0xa>(v);  // row_bcast:15 into the odd rows, 31 into the upper half
  return dpp_plus<0x143, 0xc>(v);
}

// The tiles to compute, by one workgroup: {group, first, slots} of max_tiles
// tiles (0 slots: none), then the slots sorted by group, a tile's from `first`
// on.  A group's tiles are consecutive, full but the last; tile i of T takes
// place (i % C) * 8 + i / C with C = ceil(T / 8), so that with places dealt to
// the XCDs in turn each XCD gets whole runs of them, an expert's on one or two.
// An id that is neither an expert nor -1 sets the error flag.  The order of a
// group's slots is that of the atomics; no result depends on it.
// Bound by latency, one workgroup's passes over the ids: with the rows' Q8_1
// beside it 4.0 us for 640 slots (and as many rows of 768), 4.9 for 2664 (333
// rows of 2560), 14 for 32768 (4096 rows).
__device__ void expert_plan(const int32_t *__restrict__ ids, int32_t slots, int32_t experts,
                            int32_t tile_rows, int32_t max_tiles, int32_t *__restrict__ plan,
                            int32_t *__restrict__ err) {
  // groups 0 .. experts, the last the slots without one
  __shared__ int count[kMaxExperts + 1], before[kMaxExperts + 1], tile0[kMaxExperts + 1];
  __shared__ int part[2][16];
  constexpr int kKeep = 32;
  __shared__ __align__(16) uint16_t order[1024 * kKeep];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  for (int i = t; i <= experts; i += 1024) count[i] = 0;
  for (int i = t; i < max_tiles; i += 1024) plan[4 * i + 2] = 0;
  __syncthreads();
  // A thread's ids, all in flight together (one by one 32768 slots took 40
  // us), and their places in their groups, kept in registers up to kKeep
  // ids; beyond, in batches that are gone through twice.
  uint32_t held[kKeep];  // group << 20 | place in it (at most 2^20 slots)
  bool bad = false;
  const __amdgpu_buffer_rsrc_t ri =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<int32_t *>(ids), 0, slots * 4, 0x00020000);
  auto count_in = [&](int s0) __attribute__((always_inline)) {
    // (few slots: the rounds without one are not gone through)
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      if (s0 + 1024 * k >= slots) break;
      held[k] = __builtin_amdgcn_raw_buffer_load_b32(ri, (s0 + 1024 * k + t) * 4, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      if (s0 + 1024 * k >= slots) break;
      if (s0 + 1024 * k + t >= slots) continue;
      const int id = (int)held[k], g = group_of(id, experts);
      bad |= id < -1 || id >= experts;
      held[k] = (uint32_t)g << 20 | (uint32_t)atomicAdd(&count[g], 1);
    }
  };
  for (int s0 = 0; s0 < slots; s0 += 1024 * kKeep) count_in(s0);
  if (__ballot(bad) && lane == 0) *err = 1;
  __syncthreads();
  // the groups' first slots and tiles (exclusive prefix sums); then a tile's
  // header by the thread of its group
  int total = 0, sorted = 0;
  for (int g0 = 0; g0 <= experts; g0 += 1024) {
    const int g = g0 + t;
    const int c = g <= experts ? count[g] : 0;
    const int n = (c + tile_rows - 1) / tile_rows;
    const int pt = wave_scan(n), ps = wave_scan(c);
    if (lane == 63) part[0][wave] = pt, part[1][wave] = ps;
    __syncthreads();
    // over the sixteen waves: each scans their sums itself
    const int wt = wave_scan(part[0][lane & 15]), ws = wave_scan(part[1][lane & 15]);
    const int tiles = total + (wave ? __builtin_amdgcn_readlane(wt, wave - 1) : 0);
    const int above = sorted + (wave ? __builtin_amdgcn_readlane(ws, wave - 1) : 0);
    total += __builtin_amdgcn_readlane(wt, 15), sorted += __builtin_amdgcn_readlane(ws, 15);
    if (g <= experts) before[g] = above + ps - c, tile0[g] = tiles + pt - n;
    __syncthreads();
  }
  const int run = max((total + 7) / 8, 1);
  for (int g = t; g <= experts; g += 1024) {
    const int c = count[g];
    int r = tile0[g] % run, x = tile0[g] / run;
    for (int f = 0; f < c; f += tile_rows) {
      *(v4i *)(plan + 4 * (8 * r + x)) = v4i{g, before[g] + f, min(tile_rows, c - f), 0};
      if (++r == run) r = 0, ++x;
    }
  }
  int32_t *const sorted_slots = plan + 4 * max_tiles;
  if (slots <= 1024 * kKeep) {
    // through LDS, to be written side by side (scattered from this one
    // workgroup, a line per slot, 32768 of them took 15 us)
#pragma unroll
    for (int k = 0; k < kKeep && 1024 * k < slots; ++k)
      if (1024 * k + t < slots) order[before[held[k] >> 20] + (held[k] & 0xFFFFFu)] = (uint16_t)(1024 * k + t);
    __syncthreads();
#pragma unroll 8
    for (int i = 4 * t; i < slots; i += 4096) {
      const uint2 four = *(const uint2 *)(order + i);
      *(v4i *)(sorted_slots + i) = v4i{(int)(four.x & 0xffffu), (int)(four.x >> 16),  // (up to
                                       (int)(four.y & 0xffffu), (int)(four.y >> 16)};  // three past the end)
    }
    return;
  }
  __syncthreads();
  for (int g = t; g <= experts; g += 1024) count[g] = 0;
  __syncthreads();
  for (int s0 = 0; s0 < slots; s0 += 1024 * kKeep) {
    count_in(s0);
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (s0 + 1024 * k + t < slots)
        sorted_slots[before[held[k] >> 20] + (held[k] & 0xFFFFFu)] = s0 + 1024 * k + t;
  }
}

// quantize_block8 of N raw pieces side by side; again one by one for a rare
// extreme scale.
template <bool BF16, int N>
__device__ __forceinline__ void quantize_pieces(const uint4 (&v)[N], int32_t (&q)[N], float (&s)[N]) {
  bool slow = false;
#pragma unroll
  for (int k = 0; k < N; ++k) slow |= quantize_block8_fast(act4_of_raw<BF16>(v[k]), &q[k], &s[k]);
  if (__builtin_amdgcn_ballot_w64(slow)) {
#pragma unroll
    for (int k = 0; k < N; ++k) quantize_block8(act4_of_raw<BF16>(v[k]), true, &q[k], &s[k]);
  }
}

// What comes before the products of many slots: workgroup 0 plans, the
// others quantize the rows (x null: nothing to quantize).
constexpr int kQuantUnits = 4;
__global__ __launch_bounds__(1024) void expert_prepare_kernel(
    const int32_t *__restrict__ ids, int32_t slots, int32_t experts, int32_t tile_rows,
    int32_t max_tiles, int32_t *__restrict__ plan, int32_t *__restrict__ err,
    const void *__restrict__ x, int bf16, int aligned, int64_t ldx, int64_t m, int32_t blocks,
    int32_t per, int8_t *__restrict__ qa, float *__restrict__ sa) {
  if (blockIdx.x == 0) return expert_plan(ids, slots, experts, tile_rows, max_tiles, plan, err);
  // (row, block) units, eight threads each, `per` of them in flight per thread
  // (the plan's registers leave room for one workgroup per CU)
  const int p = threadIdx.x & 7;
  const int64_t u0 = ((int64_t)blockIdx.x - 1) * 128 * per + (threadIdx.x >> 3);
  const int64_t units = m * blocks;
  auto quantize = [&](auto BF16, auto ALIGNED) __attribute__((always_inline)) {
    uint4 v[kQuantUnits];
#pragma unroll
    for (int k = 0; k < kQuantUnits; ++k) {
      v[k] = make_uint4(0, 0, 0, 0);
      if (k >= per) continue;
      const uint32_t u = (uint32_t)min(u0 + 128 * k, units - 1);
      const uint32_t row = u / (uint32_t)blocks;
      const uint32_t col = (u - row * (uint32_t)blocks) * kBlock + 4 * p;
      v[k] = load_raw4<BF16(), ALIGNED()>(x, (int64_t)row * ldx + col);
    }
    int32_t q[kQuantUnits];
    float s[kQuantUnits];
    quantize_pieces<BF16()>(v, q, s);
#pragma unroll
    for (int k = 0; k < kQuantUnits; ++k) {
      const int64_t u = u0 + 128 * k;
      if (k >= per || u >= units) break;
      *(int32_t *)(qa + u * kBlock + 4 * p) = q[k];
      if (p == 0) sa[u] = s[k];
    }
  };
  const std::true_type yes;
  const std::false_type no;
  if (bf16) aligned ? quantize(yes, yes) : quantize(yes, no);
  else aligned ? quantize(no, yes) : quantize(no, no);
}

// ---------------------------------------------------------- products ---- //

struct ExpertArgs {
  const int8_t *qa;    // Q8_1 rows [.., 32 blocks], dense
  const float *sa;     // their scales [.., blocks]
  const void *x;       // up to 4 slots: the rows themselves, quantized by each
  int64_t ldx;         //   workgroup (x_type 1: f32, 2: bf16)
  int32_t x_type;      // 0: qa / sa
  int32_t x_aligned;
  int32_t per_row;     // slots per input row: slot s reads row s / per_row
  const int32_t *ids;  // [slots]
  int32_t *err;        // without a plan: set by an id that is out of range
  int32_t slots, experts;
  const int32_t *plan; // expert_plan's, or null: a tile per slot that is the
  int32_t max_tiles;   //   first of its group (or of 16 of them)
  const uint8_t *w0, *w1;
  ExpertLayout lay;
  int32_t blocks;      // K / 32
  int32_t rows;        // N of an expert
  int32_t n_groups;    // column ranges
  int32_t repeat;      // column ranges that a workgroup takes one after another
  int64_t in_rows;     // rows of qa / sa
  int32_t act;
  int32_t y_bf16, vec; // vec: y takes stores of four values
  void *y;             // [slots, ldy]
  int64_t ldy;
  int8_t *hq;          // DUAL: Q8_1 of the SwiGLU's rows, [slots, rows]
  float *hs;
};

// The plan's tile and the column range of this workgroup; its slots into
// `rows` (LDS, no barrier).  Returns the number of slots.
__device__ __forceinline__ int planned_tile(const ExpertArgs &p, int &ng, int &group, int *rows) {
  const int i = blockIdx.x >> 3;
  const int tile = i / p.n_groups * 8 + (blockIdx.x & 7);
  ng = i - i / p.n_groups * p.n_groups;
  const v4i e = *(const v4i *)(p.plan + 4 * (int64_t)tile);
  group = __builtin_amdgcn_readfirstlane(e[0]);
  const int count = __builtin_amdgcn_readfirstlane(e[2]);
  if ((int)threadIdx.x < count) rows[threadIdx.x] = p.plan[4 * (int64_t)p.max_tiles + e[1] + threadIdx.x];
  return count;
}

// Rows of slots without an expert: zeros in columns [col0, col0 + cols).
__device__ __forceinline__ void expert_zero_rows(const ExpertArgs &p, int col0, int cols, int count,
                                                 const int *rows) {
  for (int i = threadIdx.x; i < count * cols; i += 256) {
    const int r = i / cols, n = col0 + i % cols;
    if (n >= p.rows) continue;
    const int64_t at = (int64_t)rows[r] * p.ldy + n;
    if (p.y_bf16) ((uint16_t *)p.y)[at] = 0;
    else ((float *)p.y)[at] = 0.0f;
  }
}

__device__ __forceinline__ float as_bf16(float v) { return bf16_to_float(float_to_bf16(v)); }

// One step of the platform's chain: acc + dot * f.
template <bool FMA>
__device__ __forceinline__ float chain(int dot, float f, float acc) {
  if (FMA) return __builtin_fmaf((float)dot, f, acc);
  const float contrib = (float)dot * f;
  return acc + contrib;
}

// A barrier that waits for this wave's LDS operations and nothing else: the
// global loads in flight stay there (__syncthreads waits for them too).
__device__ __forceinline__ void lds_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

typedef unsigned v4u __attribute__((ext_vector_type(4)));

// silu for a result that is rounded to bf16 next: the rounded values of
// silu_f32 (activate_array), most of them without its f64 exponential.  In
// f32, exp(-v) = 2^h (1 + l ln 2) with h + l = -v log2(e), h its rounding; the
// hardware's 2^x and 1/x are good to one step (2^-23), so the result is
// within 3 * 2^-23 of silu and silu_f32's four roundings 4 * 2^-24: the two
// differ by less than 2^-20, at most 16 steps of f32.  Where no midpoint
// of bf16 lies within 17 steps both round to the same value; where one does
// (one value in 2000), or where |v| leaves the range of that reckoning, the
// array is done again exactly.  (llmcp_q8_selftest_silu compares all 2^32
// floats on the running card: no difference.)
//
// One value by the f32 form; sets `slow` where it is not to be taken.
__device__ __forceinline__ float silu_bf16_fast(float x, bool &slow) {
  const float h = x * -1.44269502f;
  const float l = __builtin_fmaf(x, -1.92596303e-8f, __builtin_fmaf(x, -1.44269502f, -h));
  const float e0 = __builtin_amdgcn_exp2f(h);
  const float e = __builtin_fmaf(e0, l * 0.693147182f, e0);
  const float r = x * __builtin_amdgcn_rcpf(1.0f + e);
  const uint32_t low = __builtin_bit_cast(uint32_t, r) & 0xffffu;
  const float a = fabsf(x);
  slow |= low - (0x8000u - 17u) <= 34u || !(a < 80.0f) || (a < 0x1p-100f && x != 0.0f);
  return r;
}
template <int N>
__device__ __forceinline__ void silu_for_bf16(float (&v)[N]) {
  float r[N];
  bool slow = false;
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = silu_bf16_fast(v[i], slow);
  if (__builtin_amdgcn_ballot_w64(slow) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = r[i];
  } else {
    activate_array(v, ACT_SILU);
  }
}

// Over the float bit patterns [lo, lo + 2^31): out[0] counts the f32 form's
// values that would be taken and round to another bf16 than silu_f32 (each by
// itself, whatever its neighbours need), out[1] silu_for_bf16's that do,
// out[2] the values that the f32 form leaves.  NaNs are alike.
__global__ __launch_bounds__(256) void selftest_silu_kernel(uint32_t lo, unsigned long long *out) {
  const float v = __builtin_bit_cast(float, lo + blockIdx.x * 256u + threadIdx.x);
  const uint16_t want = float_to_bf16(silu_f32(v));
  bool slow = false;
  const float r = silu_bf16_fast(v, slow);
  float whole[1] = {v};
  silu_for_bf16(whole);
  auto unlike = [&](float x) {
    const uint16_t got = float_to_bf16(x);
    return got != want && !((got & 0x7fff) > 0x7f80 && (want & 0x7fff) > 0x7f80);
  };
  const uint64_t bad = __ballot(!slow && unlike(r)), off = __ballot(unlike(whole[0])), left = __ballot(slow);
  if ((threadIdx.x & 63) == 0) {
    if (bad) atomicAdd(out, (unsigned long long)__popcll(bad));
    if (off) atomicAdd(out + 1, (unsigned long long)__popcll(off));
    if (left) atomicAdd(out + 2, (unsigned long long)__popcll(left));
  }
}

// A product's activation before its store.
template <int N>
__device__ __forceinline__ void activate_out(float (&v)[N], int act, int bf16) {
  if (act == ACT_SILU && bf16) silu_for_bf16(v);
  else activate_array(v, act);
}

// The Q8_1 of h in LDS ([slot][ld] f32, 32 columns from col0 on per block)
// into hq / hs; threads in groups of eight.
__device__ __forceinline__ void store_h(const ExpertArgs &p, const float *hb, int ld, int nblk,
                                        int col0, int count, const int *rows) {
  const int l8 = threadIdx.x & 7;
  const int units = (count * nblk + 7) & ~7;  // whole waves
  for (int u = threadIdx.x >> 3; u < units; u += 32) {
    const int r = min(u / nblk, count - 1), b = u % nblk;
    const float4 v = *(const float4 *)(hb + r * ld + 32 * b + 4 * l8);
    int32_t q;
    float s;
    quantize_block8(v, true, &q, &s);
    const int n = col0 + 32 * b;
    if (u < count * nblk && n < p.rows) {
      const int64_t slot = rows[r];
      *(int32_t *)(p.hq + slot * p.rows + n + 4 * l8) = q;
      if (l8 == 0) p.hs[slot * (p.rows / kBlock) + n / kBlock] = s;
    }
  }
}

// ---- few slots per expert: up to 4 NV = 4, 8 or 16, on 16 x 16 tiles
//
// Bound by the stream of the weights.  The rows are the A operand and the
// weights B, so a result's slot is its register and lane quarter: slot i is
// put at row 4 (i % 4) + i / 4, and 4 NV slots need NV of the four registers
// of each MFMA result: the epilogue of a step of four blocks is 8 NV
// operations.  Each wave streams its tiles of 16 columns straight into the
// registers that the MFMAs read, a ring of kFewRing steps, without a pause
// from tile to tile; the rows stay in LDS for all of them.  A step issues its
// MFMAs, reads the next step's rows and then runs the epilogue of the step
// before, so that a lone wave waits for none of them.  Measured: 16 tokens
// through 8 of 128 experts of [768, 2560], gate and up 64 us (344 MB, 5.3
// TB/s), down 38 us (172 MB, 4.5 TB/s); what is missing to the 6.4 TB/s of a
// plain read is the launch and the last workgroups.
//
// LDS: [slots][a_ld] values (a block pair's 64 B: quarter, block parity,
// eight values), [slots][s_ld] scales.

struct FewLds {
  int steps2;      // steps rounded up to a pair
  int a_ld, s_ld;  // of a row of values (bytes) and of scales (floats)
  __host__ __device__ static FewLds of(int steps) {
    // rows 16 B apart modulo 256 B, scales an odd number of 16 B: what the
    // lanes of one read take lies in different banks
    const int s2 = (steps + 1) & ~1;
    return {s2, s2 * 128 + 16, 4 * (s2 + 1)};
  }
  __host__ __device__ int bytes(int n) const { return n * (a_ld + 4 * s_ld); }
};
constexpr int kFewHLd = 36;
constexpr int kFewBox = 2 * 4 * 64 * 4 + 16 * kFewHLd * 4;  // DUAL: up sums, h
constexpr int kFewLdsMost = 159 * 1024;
constexpr int kFewRing = 6;  // steps of a wave's tile in flight

// The ring's place q takes step st of the tile at byte `tile` of the expert
// (st >= live: zeros, without touching memory), the lane's scale from byte
// scale_at of the step's.  No load is branched around:
// the compiler counts the loads in flight to know which have come.
struct FewRing {
  v4u w[kFewRing][2];
  uint32_t d[kFewRing];
};
__device__ __forceinline__ void few_load(FewRing &ring, int q, const uint8_t *wexp, uint32_t tile,
                                         int st, int live, int steps, int lane, int scale_at) {
  const DmaStage a = dma_stage(st, live, tile + (uint32_t)st * 2048u);
  const DmaStage b = dma_stage(st, live, tile + (uint32_t)steps * 2048u + (uint32_t)st * 128u);
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(wexp), 0, a.extent, 0x00020000);
  constexpr int kNt = 2;  // non-temporal: read once
  ring.w[q][0] = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16, a.offset, kNt);
  ring.w[q][1] = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16 + 1024, a.offset, kNt);
  ring.d[q] = __builtin_amdgcn_raw_buffer_load_b16(r, scale_at, b.offset, kNt);
}

// A step's dots (four blocks) and scale products.
struct FewDots {
  v4i c[4];
  v16f f;
};
// A step's rows: the MFMA operands of its two block pairs, the lane's scale.
struct FewRows {
  v4i x[2];
  float s;
};

__device__ __forceinline__ void few_dots(FewDots &o, const FewRows &x, const v4u (&w)[2], uint32_t d) {
  const v16f z = {};
  o.f = __builtin_amdgcn_mfma_f32_16x16x1f32(x.s, half_bits_to_float(d), z, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    // lanes 0-31 hold the pair's even block, 32-63 the odd one; the swap
    // leaves each block its own operand, eights 0, 2, 1, 3
    const auto lo = __builtin_amdgcn_permlane32_swap(w[j][0], w[j][2], false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(w[j][1], w[j][3], false, false);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const v2i wv = {(int)lo[k], (int)hi[k]};
      const v2i xv = {x.x[j][2 * k], x.x[j][2 * k + 1]};
      o.c[2 * j + k] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
          __builtin_bit_cast(long, xv), __builtin_bit_cast(long, wv), v4i{0, 0, 0, 0}, 0, 0, 0);
    }
  }
}

// One tile: acc = the chains of 4 NV slots over its steps.  The ring holds
// the tile's first steps and goes on to `after` steps of the tile at `next`;
// x holds step 0's rows, at the end as well (read_rows reads a step's).
template <int NV, bool FMA, class ReadRows>
__device__ __forceinline__ void few_tile(FewRing &ring, const uint8_t *wexp, uint32_t cur,
                                         uint32_t next, int after, int steps, FewRows &x,
                                         ReadRows &&read_rows, float (&acc)[NV]) {
  const int lane = threadIdx.x & 63, scale_at = (lane & 15) * 8 + (lane >> 4) * 2;
  const int steps2 = (steps + 1) & ~1, stages = (steps2 + kFewRing - 1) / kFewRing;
  auto epilogue = [&](const FewDots &o) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int v = 0; v < NV; ++v) acc[v] = chain<FMA>(o.c[j][v], o.f[4 * j + v], acc[v]);
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) acc[v] = 0.0f;
  FewDots even, odd = {};  // (the step before the first: nothing to add)
  for (int s = 0; s < stages; ++s) {
    const bool last = s + 1 == stages;
    const uint32_t from = last ? next : cur;
    const int st0 = last ? 0 : kFewRing * (s + 1), live = last ? after : steps;
    static_for<kFewRing / 2>([&](auto Q) __attribute__((always_inline)) {
      constexpr int q = 2 * decltype(Q)::value;
      const int st = kFewRing * s + q;
      if (st < steps2) {
        few_dots(even, x, ring.w[q], ring.d[q]);
        read_rows(x, st + 1);
        __builtin_amdgcn_sched_barrier(0);
        epilogue(odd);
        few_dots(odd, x, ring.w[q + 1], ring.d[q + 1]);
        read_rows(x, st + 2 == steps2 ? 0 : st + 2);
        __builtin_amdgcn_sched_barrier(0);
        epilogue(even);
      }
      few_load(ring, q, wexp, from, st0 + q, live, steps, lane, scale_at);
      few_load(ring, q + 1, wexp, from, st0 + q + 1, live, steps, lane, scale_at);
    });
  }
  epilogue(odd);
}

template <int NV, bool FMA, bool DUAL>
__device__ __forceinline__ void few_run(const ExpertArgs &p, int ng, int count, const int *rows,
                                        const uint8_t *wexp, FewRing &ring, const uint8_t *smem,
                                        int used, float *box) {
  const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = p.lay.steps;
  const FewLds lds = FewLds::of(steps);
  // the slot at MFMA row li (any other's data for a row past the last)
  const int mine = min((li >> 2) + 4 * (li & 3), count - 1);
  const uint8_t *const a = smem + mine * lds.a_ld + lq * 16;
  const float *const sa = (const float *)(smem + used * lds.a_ld) + mine * lds.s_ld + lq;
  const uint32_t tile_bytes = (uint32_t)p.lay.tile_bytes();
  auto tile_of = [&](int it) {
    return DUAL ? (ng * p.repeat + it) * 2 + (wave >> 1) : (ng * p.repeat + it) * 4 + wave;
  };
  auto read_rows = [&](FewRows &x, int st) __attribute__((always_inline)) {
    x.x[0] = *(const v4i *)(a + st * 128);
    x.x[1] = *(const v4i *)(a + st * 128 + 64);
    x.s = sa[4 * st];
  };
  FewRows x;
  read_rows(x, 0);
  for (int it = 0; it < p.repeat; ++it) {
    float acc[NV];
    few_tile<NV, FMA>(ring, wexp, (uint32_t)min(tile_of(it), p.lay.tiles - 1) * tile_bytes,
                      (uint32_t)min(tile_of(it + 1), p.lay.tiles - 1) * tile_bytes,
                      it + 1 < p.repeat ? steps : 0, steps, x, read_rows, acc);
    const int n = tile_of(it) * 16 + li;
    if constexpr (!DUAL) {
      activate_out(acc, p.act, p.y_bf16);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int i = 4 * v + lq;
        if (i >= count || n >= p.rows) continue;
        const int64_t at = (int64_t)rows[i] * p.ldy + n;
        if (p.y_bf16) ((uint16_t *)p.y)[at] = float_to_bf16(acc[v]);
        else ((float *)p.y)[at] = acc[v];
      }
    } else {
      // the up wave's sums to the gate wave, h to LDS, its Q8_1 by rows
      float *const ub = box + (wave >> 1) * 256, *const hb = box + 512;
      if (wave & 1) {
#pragma unroll
        for (int v = 0; v < NV; ++v) ub[v * 64 + lane] = acc[v];
      }
      lds_barrier();
      if (!(wave & 1)) {
        activate_out(acc, ACT_SILU, p.y_bf16);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float u = ub[v * 64 + lane];
          const float h = p.y_bf16 ? as_bf16(as_bf16(acc[v]) * as_bf16(u)) : acc[v] * u;
          hb[(4 * v + lq) * kFewHLd + 16 * (wave >> 1) + li] = h;
        }
      }
      lds_barrier();
      store_h(p, hb, kFewHLd, 1, (ng * p.repeat + it) * 32, count, rows);
    }
  }
}

template <int NV, bool FMA, bool DUAL>
__global__ __launch_bounds__(256, 3) void expert_few_kernel(const ExpertArgs p) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int TILE = 4 * NV;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int rows[TILE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int steps = p.lay.steps;
  int ng = 0, group = 0, count = 0;
  if (p.plan) {
    count = planned_tile(p, ng, group, rows);
    if (count == 0) return;
  } else if constexpr (NV > 1) {
    // the slots counted by group, tile blockIdx.x / n_groups of the groups'
    // tiles found (counts do not depend on the atomics' order), its slots in
    // their own order
    __shared__ int hist[kDirectSlots], found[2];
    const int tile = blockIdx.x / p.n_groups;
    ng = blockIdx.x - tile * p.n_groups;
    hist[tid] = 0;
    if (tid == 0) found[0] = -1;
    const int id = p.ids[min(tid, p.slots - 1)];
    lds_barrier();
    if (tid < p.slots) atomicAdd(&hist[group_of(id, p.experts)], 1);
    if (blockIdx.x == 0 && (id < -1 || id >= p.experts)) *p.err = 1;
    lds_barrier();
    if (wave == 0) {
      int n[4], sum = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += n[k] = (hist[4 * lane + k] + TILE - 1) / TILE;
      int before = wave_scan(sum) - sum;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (tile >= before && tile < before + n[k]) found[0] = 4 * lane + k, found[1] = tile - before;
        before += n[k];
      }
    }
    lds_barrier();
    group = __builtin_amdgcn_readfirstlane(found[0]);
    if (group < 0) return;
    const int first = __builtin_amdgcn_readfirstlane(found[1]) * TILE;
    count = min(__builtin_amdgcn_readfirstlane(hist[group]) - first, TILE);
    if (wave == 0) {
      int before = 0;
      for (int c = 0; c < p.slots; c += 64) {
        const int i = c + lane;
        const bool hit = i < p.slots && group_of(p.ids[min(i, p.slots - 1)], p.experts) == group;
        const uint64_t m = __ballot(hit);
        const int at = before + __popcll(m & ((1ull << lane) - 1)) - first;
        if (hit && at >= 0 && at < TILE) rows[at] = i;
        before += __popcll(m);
      }
    }
  } else {
    // every wave looks over all slots: those of this group before s, and the
    // tile's from s on
    const int s = blockIdx.x / p.n_groups;
    ng = blockIdx.x - s * p.n_groups;
    int id[kDirectSlots / 64];
#pragma unroll
    for (int c = 0; c < kDirectSlots / 64; ++c) id[c] = p.ids[min(64 * c + lane, p.slots - 1)];
    int own = 0;
#pragma unroll
    for (int c = 0; c < kDirectSlots / 64; ++c)
      if (s >> 6 == c) own = __builtin_amdgcn_readlane(id[c], s & 63);
    group = group_of(own, p.experts);
    if (ng == 0 && tid == 0 && (own < -1 || own >= p.experts)) *p.err = 1;
    int before = 0;
#pragma unroll
    for (int c = 0; c < kDirectSlots / 64; ++c) {
      const int i = 64 * c + lane;
      const bool hit = i < p.slots && group_of(id[c], p.experts) == group;
      before += __popcll(__ballot(hit && i < s));
      const uint64_t m = __ballot(hit && i >= s);
      const int at = count + __popcll(m & ((1ull << lane) - 1));
      if (wave == 0 && hit && i >= s && at < TILE) rows[at] = i;
      count += __popcll(m);
    }
    if (before % TILE != 0) return;
    count = min(count, TILE);
  }
  const int cols = (DUAL ? 32 : 64) * p.repeat;
  if (group >= p.experts) {
    __syncthreads();
    if constexpr (!DUAL) expert_zero_rows(p, ng * cols, cols, count, rows);
    return;
  }
  // the weights' first steps on their way before anything waits for the rows
  const uint8_t *const wexp = (DUAL && (wave & 1) ? p.w1 : p.w0) + (int64_t)group * p.lay.expert_bytes();
  FewRing ring;
  {
    const int tile = DUAL ? ng * p.repeat * 2 + (wave >> 1) : ng * p.repeat * 4 + wave;
    const uint32_t at = (uint32_t)min(tile, p.lay.tiles - 1) * (uint32_t)p.lay.tile_bytes();
#pragma unroll
    for (int q = 0; q < kFewRing; ++q)
      few_load(ring, q, wexp, at, q, steps, steps, lane, (lane & 15) * 8 + (lane >> 4) * 2);
  }
  lds_barrier();
  // ---- the rows' Q8_1 into LDS
  const FewLds lds = FewLds::of(steps);
  const int used = min(TILE, p.slots);  // rows that the LDS holds
  float *const ls = (float *)(smem + used * lds.a_ld);
  auto copy = [&]() __attribute__((always_inline)) {
    // a half block and a scale per thread, four of each in flight
    const int halves = 2 * p.blocks;
    for (int u0 = 0; u0 < count * halves; u0 += 1024) {
      v4i v[4];
      float sc[4];
      int r[4], h[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int u = min(u0 + 256 * k + tid, count * halves - 1);
        r[k] = u / halves, h[k] = u - r[k] * halves;
        const int64_t row = rows[r[k]] / p.per_row;
        v[k] = *(const v4i *)(p.qa + (row * p.blocks) * kBlock + 16 * h[k]);
        sc[k] = p.sa[row * p.blocks + (h[k] >> 1)];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (u0 + 256 * k + tid >= count * halves) continue;
        const int b = h[k] >> 1;
        uint8_t *const to = smem + r[k] * lds.a_ld + (b >> 1) * 64 + (h[k] & 1) * 16 + (b & 1) * 8;
        *(v2i *)to = v2i{v[k][0], v[k][1]};
        *(v2i *)(to + 32) = v2i{v[k][2], v[k][3]};
        if (!(h[k] & 1)) ls[r[k] * lds.s_ld + b] = sc[k];
      }
    }
  };
  // quantized here, eight lanes per block, four blocks of each in flight
  auto quantize = [&](auto BF16, auto ALIGNED) __attribute__((always_inline)) {
    const int l8 = tid & 7;
    for (int u0 = 0; u0 < count * p.blocks; u0 += 128) {
      uint4 v[4];
      int r[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int u = min(u0 + 32 * k + (tid >> 3), count * p.blocks - 1);
        r[k] = u / p.blocks, b[k] = u - r[k] * p.blocks;
        v[k] = load_raw4<BF16(), ALIGNED()>(
            p.x, (int64_t)(rows[r[k]] / p.per_row) * p.ldx + b[k] * kBlock + 4 * l8);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // (side by side 2 % slower here: other workgroups fill the waits)
        int32_t q;
        float sc;
        quantize_block8(act4_of_raw<BF16()>(v[k]), true, &q, &sc);
        if (u0 + 32 * k + (tid >> 3) >= count * p.blocks) continue;
        const int quarter = (l8 >> 1 & 1) * 2 + (l8 >> 2);  // eights 0, 2, 1, 3
        *(int32_t *)(smem + r[k] * lds.a_ld + (b[k] >> 1) * 64 + quarter * 16 + (b[k] & 1) * 8 +
                     (l8 & 1) * 4) = q;
        if (l8 == 0) ls[r[k] * lds.s_ld + b[k]] = sc;
      }
    }
  };
  if (NV > 1 || !p.x_type) {
    copy();
  } else if constexpr (NV == 1) {
    const std::true_type yes;
    const std::false_type no;
    if (p.x_type == 2) p.x_aligned ? quantize(yes, yes) : quantize(yes, no);
    else p.x_aligned ? quantize(no, yes) : quantize(no, no);
  }
  // blocks past the last: weights of zero against any values, scales of zero
  for (int u = tid; u < count * 8; u += 256) {
    const int b = p.blocks + (u & 7);
    if (b < 4 * lds.steps2) ls[(u >> 3) * lds.s_ld + b] = 0.0f;
  }
  lds_barrier();
  float *const box = (float *)(smem + lds.bytes(used));
  few_run<NV, FMA, DUAL>(p, ng, count, rows, wexp, ring, smem, used, box);
#endif
}

// ---- few tokens: a slot's own row, no sharing
//
// A CU takes about 13 B a clock from beyond its L2 however few of the others
// do (a workgroup that reads 174 KB takes 11 us whether there are 24 of them or
// 240), so a token's products are as fast as the bytes are spread evenly, and
// as what comes before the first and after the last load is short.

// What a row is: Q8_1, or f32 or bf16 to be quantized here.
enum { ROW_Q8 = 0, ROW_F32 = 1, ROW_BF16 = 2 };

// A wave's part of a row in LDS, `count` blocks from `first` on: values in
// order, scales (zero past the row's last block).  `start` issues the first
// loads, `store` waits for them.
template <int KIND, int U>
struct TokenRow {
  uint4 v[U];  // eight lanes per block
  v4i q;       // ROW_Q8: half a block per lane, a scale per lane
  float s;
  __device__ __forceinline__ uint4 load(const ExpertArgs &p, int64_t row, int block) const {
    const int64_t at = row * p.ldx + (int64_t)min(block, p.blocks - 1) * kBlock + 4 * (threadIdx.x & 7);
    return load_raw4<KIND == ROW_BF16, true>(p.x, at);
  }
  __device__ __forceinline__ void start(const ExpertArgs &p, int64_t row, int first) {
    const int lane = threadIdx.x & 63;
    if constexpr (KIND != ROW_Q8) {
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = load(p, row, first + 8 * k + (lane >> 3));
    } else {
      q = *(const v4i *)(p.qa + row * p.blocks * kBlock + 16 * min(2 * first + lane, 2 * p.blocks - 1));
      s = p.sa[row * p.blocks + min(first + lane, p.blocks - 1)];
    }
  }
  __device__ __forceinline__ void store(const ExpertArgs &p, int64_t row, int first, int count,
                                        uint8_t *values, float *scales) {
    const int lane = threadIdx.x & 63, l8 = lane & 7;
    if constexpr (KIND != ROW_Q8) {
      auto put = [&](int32_t b, float sc, int u) __attribute__((always_inline)) {
        if (u >= count) return;
        *(int32_t *)(values + u * kBlock + 4 * l8) = b;
        if (l8 == 0) scales[u] = first + u < p.blocks ? sc : 0.0f;
      };
      int32_t b[U];
      float sc[U];
      quantize_pieces<KIND == ROW_BF16>(v, b, sc);
#pragma unroll
      for (int k = 0; k < U; ++k) put(b[k], sc[k], 8 * k + (lane >> 3));
      for (int u = 8 * U; u < count; u += 8) {
        quantize_block8(act4_of_raw<KIND == ROW_BF16>(load(p, row, first + u + (lane >> 3))), true, &b[0], &sc[0]);
        put(b[0], sc[0], u + (lane >> 3));
      }
    } else {
      const int8_t *const qrow = p.qa + row * p.blocks * kBlock;
      const float *const srow = p.sa + row * p.blocks;
      if (lane < 2 * count) *(v4i *)(values + 16 * lane) = q;
      if (lane < count) scales[lane] = first + lane < p.blocks ? s : 0.0f;
      for (int u = lane + 64; u < 2 * count; u += 64)
        *(v4i *)(values + 16 * u) = *(const v4i *)(qrow + 16 * min(2 * first + u, 2 * p.blocks - 1));
      for (int u = lane + 64; u < count; u += 64)
        scales[u] = first + u < p.blocks ? srow[first + u] : 0.0f;
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own stores
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  }
};

// ---- the SwiGLU of a slot
//
// A workgroup takes 8 columns of gate and of up, two waves each, half of the
// steps per wave.  A lane takes half a block of a row, four v_dot4; two steps
// together give every lane a block's dot, which goes to LDS with the scale
// product, and sixteen lanes run the chains over them in block order.  h is
// left in the output's type; the down products quantize it.  Measured: 8
// experts of [768, 2560], 33 MB, 8.0 us (11 to 12 on tiles of 16 columns, 32
// per workgroup and 192 workgroups; a plain read of as much 7.1).

constexpr int kUpPairs = 5;  // pairs of steps of a wave in flight
struct UpRing {
  v4u w[kUpPairs][2];
  uint32_t d[kUpPairs];
};

// Steps of a wave (an even number) and the LDS: the row, then [gate, up][pair of
// blocks][column][block] {dot, factor} of whole batches of the chain.
constexpr int kUpBatch = 16;  // blocks read while as many before are added
__host__ __device__ inline int token_up_steps(int steps) { return ((steps + 1) / 2 + 1) & ~1; }
__host__ __device__ inline int token_up_blocks(int steps) { return (4 * steps + kUpBatch - 1) & -kUpBatch; }
__host__ __device__ inline int token_up_lds(int steps) {
  return 2 * token_up_steps(steps) * (128 + 16) + (2 * token_up_blocks(steps) + kUpBatch) * 8 * 8;
}

// The ring's place q takes steps st and st + 1 of the eight rows whose values
// and scales begin at bytes `values` and `scales` of the expert; from `live` on
// they are zeros, without touching memory.
__device__ __forceinline__ void up_load(UpRing &ring, int q, const uint8_t *wexp, uint32_t values,
                                        uint32_t scales, int st, int live, int lane) {
  constexpr int kNt = 2;  // non-temporal: read once
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const DmaStage a = dma_stage(st + i, live, values + (uint32_t)(st + i) * 2048u);
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(wexp), 0, a.extent, 0x00020000);
    ring.w[q][i] = __builtin_amdgcn_raw_buffer_load_b128(r, (lane >> 3) * 256 + (lane & 7) * 16, a.offset, kNt);
  }
  // the second step's by the lanes of second halves (if there is one)
  const DmaStage d = dma_stage(st, live, scales + (uint32_t)st * 128u);
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(wexp), 0, d.extent, 0x00020000);
  const int second = (st + 1 - live) >> 31 & 128;
  ring.d[q] = __builtin_amdgcn_raw_buffer_load_b16(
      r, (lane & 7) * 8 + (lane >> 4) * 2 + (lane & 8 ? second : 0), d.offset, kNt);
}

template <bool FMA, bool BF16, int KIND>
__global__ __launch_bounds__(256) void expert_token_up_kernel(const ExpertArgs p) {
#ifdef __HIP_DEVICE_COMPILE__
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = p.lay.steps, slot = blockIdx.y;
  const int64_t row = slot / p.per_row;
  const int per = token_up_steps(steps);
  const int first = min((wave >> 1) * per, steps), end = min(first + per, steps);
  float *const scales = (float *)(smem + 2 * per * 128);
  float2 *const box = (float2 *)(smem + 2 * per * (128 + 16));
  // a quarter of the row per wave (an even number of blocks)
  const int quarter = 2 * per;
  TokenRow<KIND, 3> x;
  x.start(p, row, wave * quarter);
  const int id = __builtin_amdgcn_readfirstlane(p.ids[slot]);
  if ((unsigned)id >= (unsigned)p.experts) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && id != -1) *p.err = 1;
    return;
  }
  const uint8_t *const wexp = (wave & 1 ? p.w1 : p.w0) + (int64_t)id * p.lay.expert_bytes();
  const uint32_t tile = (blockIdx.x >> 1) * (uint32_t)p.lay.tile_bytes();
  const uint32_t wat = tile + (blockIdx.x & 1) * 128u;
  const uint32_t dat = tile + (uint32_t)steps * 2048u + (blockIdx.x & 1) * 64u;
  UpRing ring;
  static_for<kUpPairs>([&](auto Q) __attribute__((always_inline)) {
    constexpr int q = decltype(Q)::value;
    up_load(ring, q, wexp, wat, dat, first + 2 * q, end, lane);
    // (the later loads wait for room in the CU's queue as it is)
    if constexpr (q == 1)
      x.store(p, row, wave * quarter, quarter, smem + wave * quarter * kBlock, scales + wave * quarter);
  });
  // blocks of the last batch that no step writes
  const int blocks = token_up_blocks(steps), written = 4 * ((steps + 1) & ~1);
  for (int i = threadIdx.x; i < (blocks - written) * 16; i += 256)
    box[(i & 8 ? blocks * 8 : 0) + written * 8 + (i >> 4) * 8 + (i & 7)] = make_float2(0.0f, 0.0f);
  lds_barrier();
  // lane: column lane % 8, half (lane / 8) % 2 of block lane / 16, of whose two
  // steps it keeps that of its half
  const bool upper = lane & 8;
  auto pass = [&](int s, auto LOADS, auto FULL) __attribute__((always_inline)) {
    const uint8_t *const xv = smem + s * 128 + (lane >> 3) * 16;
    const float *const xs = scales + 4 * s + (upper ? 4 : 0) + (lane >> 4);
    float2 *const to = box + (wave & 1) * blocks * 8 + (s + (upper ? 1 : 0)) * 32 + (lane >> 5) * 16 +
                       (lane & 7) * 2 + (lane >> 4 & 1);
    static_for<kUpPairs>([&](auto Q) __attribute__((always_inline)) {
      constexpr int q = decltype(Q)::value;
      if (FULL || s + 2 * q < end) {
        int c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const v4i v = *(const v4i *)(xv + (2 * q + i) * 128);
          c[i] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) c[i] = __builtin_amdgcn_sdot4((int)ring.w[q][i][k], v[k], c[i], false);
        }
        // the other half's part of this lane's step (row_ror:8)
        const int send = upper ? c[0] : c[1];
        const int dot = (upper ? c[1] : c[0]) + __builtin_amdgcn_update_dpp(0, send, 0x128, 0xf, 0xf, false);
        to[2 * q * 32] = make_float2((float)dot, xs[8 * q] * half_bits_to_float(ring.d[q]));
      }
      if (LOADS) up_load(ring, q, wexp, wat, dat, s + 2 * (q + kUpPairs), end, lane);
    });
  };
  int st = first;
  for (; st + 2 * kUpPairs < end; st += 2 * kUpPairs) pass(st, std::true_type(), std::true_type());
  if (st + 2 * kUpPairs == end) pass(st, std::false_type(), std::true_type());
  else pass(st, std::false_type(), std::false_type());
  lds_barrier();
  if (wave != 0) return;
  // lanes 0-7: the gate's columns, 8-15: the up's (the others repeat)
  const float4 *t = (const float4 *)box + (upper ? blocks * 4 : 0) + (lane & 7);
  float acc[1] = {0.0f};
  constexpr int B = kUpBatch / 2;
  auto read = [&](float4 (&v)[B], int b) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < B; ++k) v[k] = t[(b / 2 + k) * 8];
  };
  auto add = [&](const float4 (&v)[B]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < B; ++k) {
      if (FMA) {
        acc[0] = __builtin_fmaf(v[k].x, v[k].y, acc[0]);
        acc[0] = __builtin_fmaf(v[k].z, v[k].w, acc[0]);
      } else {
        const float c0 = v[k].x * v[k].y, c1 = v[k].z * v[k].w;
        acc[0] = acc[0] + c0;
        acc[0] = acc[0] + c1;
      }
    }
  };
  float4 even[B], odd[B];  // (behind the last batch: memory that is not used)
  read(even, 0);
  for (int b = 0; b < blocks; b += 2 * kUpBatch) {
    read(odd, b + kUpBatch);
    add(even);
    if (b + kUpBatch >= blocks) break;
    read(even, b + 2 * kUpBatch);
    add(odd);
  }
  const float u = dpp_f32<0x128>(acc[0]);
  activate_out(acc, ACT_SILU, BF16);
  if (lane >= 8) return;
  const int64_t at = (int64_t)slot * p.ldy + blockIdx.x * 8 + lane;
  if (BF16) ((uint16_t *)p.y)[at] = float_to_bf16(as_bf16(acc[0]) * as_bf16(u));
  else ((float *)p.y)[at] = acc[0] * u;
#endif
}

// ---- their down products and weighted sum in one launch
//
// A workgroup per token and tile of 16 columns, a wave per slot (in turns
// beyond eight): each streams its expert's tile with its one row of h,
// quantized to LDS, and the results, rounded to the output's type, are added in slot
// order by sixteen lanes (expert_combine_kernel's sum).  An expert that two
// tokens share is read twice.  Measured: 8 experts of [2560, 768], 17 MB, 6.8
// us: 160 workgroups that each read 104 KB at what a CU takes.

constexpr int kTokenWaves = 8;

// LDS of a wave: its row's values, natural order, and scales, each of a pair
// of steps more than the row may have.
__host__ __device__ inline int token_lds(int steps) { return ((steps + 1) & ~1) * (128 + 16); }

template <bool FMA, bool BF16>
__global__ __launch_bounds__(64 * kTokenWaves) void expert_token_kernel(
    const ExpertArgs p, const float *__restrict__ weights, int32_t top_k, const void *residual,
    int64_t ldr, void *y, int64_t ldy) {
#ifdef __HIP_DEVICE_COMPILE__
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float sums[kMaxTopK][16];
  const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int64_t token = blockIdx.y;
  const int tile = blockIdx.x, steps = p.lay.steps;
  uint8_t *const mine = smem + wave * token_lds(steps);
  float *const ls = (float *)(mine + ((steps + 1) & ~1) * 128);
  // what the sum needs, on its way before the products
  const int64_t choice = token * top_k + min(lane, top_k - 1);
  const int ids = p.ids[choice];
  const float factors = weights ? weights[choice] : 1.0f;
  const int n = tile * 16 + li;
  uint32_t raw = 0;  // widened at the end: nothing waits for it here
  if (residual && wave == 0 && n < p.rows)
    raw = BF16 ? ((const uint16_t *)residual)[token * ldr + n] : ((const uint32_t *)residual)[token * ldr + n];
  for (int j = wave; j < top_k; j += waves) {
    const int64_t slot = token * top_k + j;
    TokenRow<BF16 ? ROW_BF16 : ROW_F32, 3> x;  // on its way before the weights
    x.start(p, slot, 0);
    const int id = __builtin_amdgcn_readfirstlane(p.ids[slot]);
    if ((unsigned)id >= (unsigned)p.experts) continue;  // uniform per wave
    const uint8_t *const wexp = p.w0 + (int64_t)id * p.lay.expert_bytes();
    const uint32_t at = (uint32_t)tile * (uint32_t)p.lay.tile_bytes();
    FewRing ring;
    static_for<kFewRing>([&](auto Q) __attribute__((always_inline)) {
      constexpr int q = decltype(Q)::value;
      few_load(ring, q, wexp, at, q, steps, steps, lane, li * 8 + lq * 2);
      // (the later loads wait for room in the CU's queue as it is)
      if constexpr (q == 2) x.store(p, slot, 0, 4 * ((steps + 1) & ~1), mine, ls);
    });
    // every MFMA row reads the one row: eights 0, 2, 1, 3 of a block
    const uint8_t *const a = mine + ((lq & 1) * 2 + (lq >> 1)) * 8;
    auto read_rows = [&](FewRows &x, int st) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2i v = *(const v2i *)(a + st * 128 + i * 32);
        x.x[i >> 1][2 * (i & 1)] = v[0], x.x[i >> 1][2 * (i & 1) + 1] = v[1];
      }
      x.s = ls[4 * st + lq];
    };
    FewRows first;
    read_rows(first, 0);
    float acc[1];
    few_tile<1, FMA>(ring, wexp, at, at, 0, steps, first, read_rows, acc);
    if (lq == 0) sums[j][li] = BF16 ? as_bf16(acc[0]) : acc[0];
  }
  __syncthreads();
  if (wave != 0) return;
  float v = BF16 ? bf16_to_float(raw) : __uint_as_float(raw);
  constexpr int K = 8;  // read together
  for (int j0 = 0; j0 < top_k; j0 += K) {
    float o[K];
#pragma unroll
    for (int k = 0; k < K; ++k) o[k] = sums[(j0 + k) & (kMaxTopK - 1)][li];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = j0 + k;
      if (j >= top_k || (unsigned)__builtin_amdgcn_readlane(ids, j) >= (unsigned)p.experts) continue;
      const int w = __builtin_amdgcn_readlane(__builtin_bit_cast(int, factors), j);
      v = __builtin_fmaf(__builtin_bit_cast(float, w), o[k], v);
    }
  }
  if (lane >= 16 || n >= p.rows) return;
  if (BF16) ((uint16_t *)y)[token * ldy + n] = float_to_bf16(v);
  else ((float *)y)[token * ldy + n] = v;
#endif
}

// ---- many slots per expert: up to 64, on 32 x 32 tiles
//
// Bound by the exact epilogue, a convert and an FMA per result and block,
// and by the MFMAs, which do not run under it.  The weights are the A
// operand: two tiles of 16 rows side by side, for a SwiGLU 16 columns of
// gate and of up, whose results land in the same lane.
// v_mfma_i32_32x32x32_i8 gives a block's dots; v_mfma_f32_32x32x1_2b_f32 two
// scale tiles, of the two tiles of 32 slots (TT = 2) or of two blocks (TT =
// 1): a unit is two dots and their scales.  Three waves per SIMD cover each
// other's latencies.  The rows pass through an LDS ring of three steps of four
// blocks, loaded a step before they are stored there, one barrier a step; a
// workgroup takes `repeat` column ranges without a pause in either stream.
// Measured with 128 experts of [768, 2560], 8 per token: 4096 tokens, gate and
// up 439 us and down 262 us (258 + 129 GFLOP, 590 and 490 TOPS, where
// convert, FMA and MFMAs alone reach 880); 333 tokens, TT = 1, 102 and 59 us
// (538 and 269 MB of weights, 5.3 and 4.6 TB/s).

template <int TT>
struct ManyLds {
  // of a step: [tile of 32 slots][block][half][slot][16 B], halves 16 B apart
  // modulo 256 B and scales [block][slot], blocks 64 B apart modulo 256 B, so
  // that the stores, eight pieces of a row or four scales side by side, lie
  // in different banks
  static constexpr int HALF = 528, BLOCK = 2 * HALF, TILE = 4 * BLOCK;
  static constexpr int SBLOCK = TT * 128 + 64;
  static constexpr int A = TT * TILE, BUF = A + 4 * SBLOCK;
  static constexpr int RING = 3 * BUF;
  static constexpr int HLD = 68;
  static constexpr int H = TT * 32 * HLD * 4;
};

template <int TT, bool FMA, bool DUAL>
__device__ __forceinline__ void many_run(const ExpertArgs &p, int ng, int group, int count,
                                         const int *rows, uint8_t *smem, float *hb) {
  typedef ManyLds<TT> L;
  constexpr int U = TT == 2 ? 4 : 2;  // units per step
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int steps = p.lay.steps;
  // ---- weights: the lane's row of 32 (lanes 16-31 and 48-63: of the second
  // tile) and half of each block, a step in registers, each block replaced
  // by the next step's once its MFMA has taken it.  (Two steps ahead, with
  // two waves per SIMD or with spills, four waves, and non-temporal loads
  // were all slower for tiles of 32 slots bound by this stream: 333 tokens
  // over 128 experts, 102 + 59 us, 105 + 64, 133 + 90, 125 + 72, 103 + 68.)
  const int64_t expert = (int64_t)group * p.lay.expert_bytes();
  const int second = lane >> 4 & 1;
  const uint8_t *const wbase = (DUAL && second ? p.w1 : p.w0) + expert;
  const uint32_t tile_bytes = (uint32_t)p.lay.tile_bytes();
  // the first of the wave's tiles in column range r
  auto tile_of = [&](int r) { return DUAL ? r * 4 + wave : r * 8 + wave * 2; };
  const uint8_t *wp, *dp;  // of the step to load next
  auto seek = [&](int r) __attribute__((always_inline)) {
    const int t = min(tile_of(r) + (DUAL ? 0 : second), p.lay.tiles - 1);
    wp = wbase + (uint32_t)t * tile_bytes + hi * 256 + (lane & 15) * 16;
    dp = wbase + (uint32_t)t * tile_bytes + (uint32_t)steps * 2048u + (lane & 15) * 8;
  };
  v4i wq[4];
  uint2 wd;
  auto load_block = [&](int b) __attribute__((always_inline)) { wq[b] = *(const v4i *)(wp + b * 512); };
  // ---- rows: thread (slot tid / 8, 16 B piece tid % 8 of a step's 128 B) and
  // (slot tid / 4, scale tid % 4): a row's bytes of a step side by side in a
  // wave, so that it asks for few lines.  Past a row's last block they read
  // the next row's data or (past the last row) zeros, against weights of zero.
  const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<int8_t *>(p.qa), 0, (int)(uint32_t)(p.in_rows * p.blocks * kBlock), 0x00020000);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float *>(p.sa), 0, (int)(uint32_t)(p.in_rows * p.blocks * 4), 0x00020000);
  const int piece = tid & 7, sblock = tid & 3;
  uint32_t src[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t)
    src[t] = (uint32_t)(rows[min(32 * t + (tid >> 3), count - 1)] / p.per_row) * (uint32_t)(p.blocks * kBlock) +
             16 * piece;
  const int sslot = (tid >> 2) & (32 * TT - 1);  // (TT = 1: the upper threads repeat)
  const uint32_t ssrc =
      (uint32_t)(rows[min(sslot, count - 1)] / p.per_row) * (uint32_t)(p.blocks * 4) + 4 * sblock;
  v4u xv[TT];
  float xs;
  auto load_rows = [&](int step) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TT; ++t) xv[t] = __builtin_amdgcn_raw_buffer_load_b128(rq, src[t], step * 128, 0);
    xs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, ssrc, step * 16, 0));
    xs = 4 * step + sblock < p.blocks ? xs : 0.0f;  // (no inf against a weight of zero)
  };
  uint8_t *const to = smem + piece * L::HALF + (tid >> 3) * 16;
  uint8_t *const sto = smem + L::A + sblock * L::SBLOCK + sslot * 4;
  auto store_rows = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TT; ++t) *(v4u *)(to + buf * L::BUF + t * L::TILE) = xv[t];
    *(float *)(sto + buf * L::BUF) = xs;
  };
  // ---- a unit's operands
  v4i x0, x1;  // TT = 2: the block's two slot tiles, TT = 1: two blocks
  float sx;
  const uint8_t *const from = smem + hi * L::HALF + l32 * 16;
  const uint8_t *const sfrom = smem + L::A + (TT == 2 ? lane * 4 : hi * L::SBLOCK + l32 * 4);
  auto read_rows = [&](int buf, int u) __attribute__((always_inline)) {
    const uint8_t *const at = from + buf * L::BUF;
    x0 = *(const v4i *)(at + (TT == 2 ? u : 2 * u) * L::BLOCK);
    x1 = *(const v4i *)(at + (TT == 2 ? L::TILE + u * L::BLOCK : (2 * u + 1) * L::BLOCK));
    sx = *(const float *)(sfrom + buf * L::BUF + (TT == 2 ? u : 2 * u) * L::SBLOCK);
  };
  auto scale = [&](int b) __attribute__((always_inline)) -> float {
    const uint32_t d = b < 2 ? wd.x : wd.y;
    return half_bits_to_float((b & 1) ? d >> 16 : d & 0xffffu);
  };
  float acc[TT][16];
  const v16i zi = {};
  const v32f zf = {};
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[t][v] = 0.0f;
  };

  // the steps of all column ranges in one sequence: `step` of `range` is
  // computed, `ahead` the step of the rows that are loaded next (they start
  // over with each range), `wstep` of `wrange` that of the weights (the last
  // range again behind the last)
  const int r0 = ng * p.repeat;
  const int ranges = min(p.repeat, (p.lay.tiles + (DUAL ? 4 : 8) - 1) / (DUAL ? 4 : 8) - r0);
  int range = 0, step = 0, ahead = 0, wstep = 0, wrange = 0;
  int buf = 0, buf1 = 1, buf2 = 2;  // the ring's places of steps 0, + 1, + 2
  auto advance = [&]() { ahead = ahead + 1 == steps ? 0 : ahead + 1; };
  auto next_weights = [&]() __attribute__((always_inline)) {
    if (++wstep == steps) {
      wstep = 0;
      wrange = min(wrange + 1, ranges - 1);
      seek(r0 + wrange);
    } else {
      wp += 2048;
      dp += 128;
    }
  };
  load_rows(ahead);
  advance();
  seek(r0);
#pragma unroll
  for (int b = 0; b < 4; ++b) load_block(b);
  wd = *(const uint2 *)dp;
  next_weights();
  store_rows(0);
  load_rows(ahead);
  advance();
  store_rows(1);
  load_rows(ahead);
  advance();
  lds_barrier();
  read_rows(0, 0);
  clear();
  for (;;) {
    // (that place's last read, of the step before, lies behind a barrier)
    store_rows(buf2);
    load_rows(ahead);
    advance();
    float dw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      dw[u] = TT == 2 ? scale(u) : hi ? scale(2 * u + 1) : scale(2 * u);
    wd = *(const uint2 *)dp;
    static_for<U>([&](auto UU) __attribute__((always_inline)) {
      constexpr int u = decltype(UU)::value;
      constexpr int b0 = TT == 2 ? u : 2 * u, b1 = TT == 2 ? u : 2 * u + 1;
      const v16i d0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(wq[b0], x0, zi, 0, 0, 0);
      const v32f f = __builtin_amdgcn_mfma_f32_32x32x1f32(dw[u], sx, zf, 0, 0, 0);
      const v16i d1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(wq[b1], x1, zi, 0, 0, 0);
      load_block(b0);
      if constexpr (b1 != b0) load_block(b1);
      // (or the MFMAs, pure operations, are moved down to their first use)
      asm volatile("" ::"v"(d0), "v"(f), "v"(d1));
      read_rows(u + 1 == U ? buf1 : buf, (u + 1) % U);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[0][v] = chain<FMA>(d0[v], f[v], acc[0][v]);
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[TT - 1][v] = chain<FMA>(d1[v], f[16 + v], acc[TT - 1][v]);
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) asm volatile("" : "+v"(acc[t][v]));
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (u == U - 2) lds_barrier();
    });
    next_weights();
    const int free = buf;
    buf = buf1, buf1 = buf2, buf2 = free;
    if (++step < steps) continue;
    const int tile0 = tile_of(r0 + range);
    if constexpr (!DUAL) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int i = 32 * t + l32;
        const int64_t base = (int64_t)rows[min(i, count - 1)] * p.ldy;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float o[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = acc[t][4 * j + v];
          activate_out(o, p.act, p.y_bf16);
          const int n = tile0 * 16 + 8 * j + 4 * hi;
          if (i >= count || n >= p.rows) continue;
          if (p.y_bf16) {
            uint16_t h[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) h[v] = float_to_bf16(o[v]);
            uint16_t *const y = (uint16_t *)p.y + base + n;
            if (p.vec) {
              *(uint2 *)y = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
            } else {
#pragma unroll
              for (int v = 0; v < 4; ++v) y[v] = h[v];
            }
          } else {
            float *const y = (float *)p.y + base + n;
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
      // h through LDS, then its Q8_1 by rows
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float o[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) o[v] = acc[t][4 * j + v];
          activate_out(o, ACT_SILU, p.y_bf16);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float u = acc[t][8 + 4 * j + v];
            o[v] = p.y_bf16 ? as_bf16(as_bf16(o[v]) * as_bf16(u)) : o[v] * u;
          }
          *(float4 *)(hb + (32 * t + l32) * L::HLD + 16 * wave + 8 * j + 4 * hi) =
              make_float4(o[0], o[1], o[2], o[3]);
        }
      lds_barrier();
      store_h(p, hb, L::HLD, 2, (r0 + range) * 64, count, rows);
      // (the next write of hb lies behind the barriers of the next range)
    }
    if (++range == ranges) break;
    step = 0;
    clear();
  }
}

template <int TT, bool FMA, bool DUAL>
__global__ __launch_bounds__(256, 3) void expert_many_kernel(const ExpertArgs p) {
#ifdef __HIP_DEVICE_COMPILE__
  __shared__ __align__(1024) uint8_t smem[ManyLds<TT>::RING];
  __shared__ __align__(16) float hb[DUAL ? ManyLds<TT>::H / 4 : 4];
  __shared__ int rows[32 * TT];
  int ng, group;
  const int count = planned_tile(p, ng, group, rows);
  if (count == 0) return;
  lds_barrier();
  if (group >= p.experts) {
    if constexpr (!DUAL) expert_zero_rows(p, ng * 128 * p.repeat, 128 * p.repeat, count, rows);
    return;
  }
  if (TT == 1 || count <= 32) many_run<1, FMA, DUAL>(p, ng, group, count, rows, smem, hb);
  else many_run<TT, FMA, DUAL>(p, ng, group, count, rows, smem, hb);
#endif
}

// ----------------------------------------------------------- combine ---- //

// y[t] = residual[t] + sum over its slots j, in order, of w[t, j] * o[t, j]:
// an f32 FMA chain from the residual (or zero), rounded once; slots without
// an expert add nothing.  V columns per thread; eight slots' loads go out
// together (a slot without an expert loads its row as well and does not use
// it).  Bound by reading the rows.
template <bool BF16, int V>
__global__ __launch_bounds__(256) void expert_combine_kernel(
    const void *__restrict__ o, const int32_t *__restrict__ ids, const float *__restrict__ w,
    int32_t top_k, int32_t experts, int64_t m, int32_t cols, const void *residual, int64_t ldr,
    int raligned, void *y, int64_t ldy, int yaligned) {
  // (fewer than 2^32 threads)
  const uint32_t pieces = cols / V, i = blockIdx.x * 256u + threadIdx.x, row = i / pieces;
  const int64_t t = row;
  if (t >= m) return;
  const int c = V * (int)(i - row * pieces);
  float v[V];
#pragma unroll
  for (int n = 0; n < V; n += 4) {
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (residual) r = load_act4(residual, t * ldr + c + n, BF16, raligned != 0);
    v[n] = r.x, v[n + 1] = r.y, v[n + 2] = r.z, v[n + 3] = r.w;
  }
  constexpr int K = 8;
  for (int j0 = 0; j0 < top_k; j0 += K) {
    int id[K];
    float f[K];
    uint4 x[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t s = t * top_k + min(j0 + k, top_k - 1);
      id[k] = j0 + k < top_k ? ids[s] : -1;
      f[k] = w ? w[s] : 1.0f;
      if constexpr (V == 8) x[k] = *(const uint4 *)((const uint16_t *)o + s * cols + c);
      else x[k] = load_raw4<BF16, true>(o, s * cols + c);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((unsigned)id[k] >= (unsigned)experts) continue;
#pragma unroll
      for (int n = 0; n < V; ++n) {
        const uint32_t u = word(x[k], BF16 ? n / 2 : n);
        const float a = BF16 ? bf16_to_float(n & 1 ? u >> 16 : u & 0xffffu) : __uint_as_float(u);
        v[n] = __builtin_fmaf(f[k], a, v[n]);
      }
    }
  }
  if (BF16) {
    uint16_t *const to = (uint16_t *)y + t * ldy + c;
    uint16_t b[V];
#pragma unroll
    for (int n = 0; n < V; ++n) b[n] = float_to_bf16(v[n]);
#pragma unroll
    for (int n = 0; n < V; n += 4) {
      if (yaligned) {
        *(uint2 *)(to + n) = make_uint2(b[n] | (uint32_t)b[n + 1] << 16, b[n + 2] | (uint32_t)b[n + 3] << 16);
      } else {
        to[n] = b[n], to[n + 1] = b[n + 1], to[n + 2] = b[n + 2], to[n + 3] = b[n + 3];
      }
    }
  } else {
    float *const to = (float *)y + t * ldy + c;
    if (yaligned) {
      *(float4 *)to = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int n = 0; n < V; ++n) to[n] = v[n];
    }
  }
}

// ------------------------------------------------------------- route ---- //

// Order of f32 logits as unsigned: NaN and -inf (never chosen) 0, then
// ascending with the value (zeros of both signs alike); and back.
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
  return !(v > -__builtin_inff()) ? 0u : (v == 0.0f ? 0x80000000u : k);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __builtin_bit_cast(float, (k >> 31) ? k & 0x7FFFFFFFu : ~k);
}

// The wave's largest v, in scalar registers (row shifts and row broadcasts; a
// lane without a source keeps its own).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
  return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x111>(v);  // row_shr:1, 2, 4, 8
  v = dpp_max<0x112>(v);
  v = dpp_max<0x114>(v);
  v = dpp_max<0x118>(v);
  v = dpp_max<0x142>(v);  // row_bcast:15, 31
  v = dpp_max<0x143>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The wave's sum, in a scalar register.
template <int CTRL>
__device__ __forceinline__ float dpp_sum(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
  return v + __builtin_bit_cast(float, o);
}
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_sum<0x111>(v);
  v = dpp_sum<0x112>(v);
  v = dpp_sum<0x114>(v);
  v = dpp_sum<0x118>(v);
  v = dpp_sum<0x142>(v);
  v = dpp_sum<0x143>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// One wave per row, PER logits per lane (logit i in lane i % 64): top_k
// rounds, each the wave's largest key and the lowest index that has it; then
// the chosen ones' exponentials side by side, one per lane.  Latency bound
// for few rows: a round is six lane moves and a ballot per 64 logits.
// Measured: the 8 largest of 128, one row 3.6 us, 4096 rows 5.3.
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
  uint32_t first = 0, mine = 0;  // the largest key, and this lane's round's
  int id = -1;
  for (int j = 0; j < top_k; ++j) {
    uint32_t most = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) most = key[i] > most ? key[i] : most;
    most = wave_max(most);
    if (most == 0) break;  // only masked logits are left
    if (j == 0) first = most;
    int e = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint64_t hit = __ballot(key[i] == most);
      const bool here = e < 0 && hit != 0;
      e = here ? 64 * i + __builtin_ctzll(hit | 1ull << 63) : e;
      if (here && lane == (e & 63)) key[i] = 0;
    }
    if (lane == j) id = e, mine = most;
  }
  const float top = key_logit(first);
  // (the maximum itself gives 1, also where it is infinite)
  auto weight = [&](float v) { return v == top ? 1.0f : exp_f32(v - top); };
  const float p = id >= 0 ? weight(key_logit(mine)) : 0.0f;
  float total = p;
  if (!normalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (l[i] > -__builtin_inff()) total += weight(l[i]);
  }
  total = wave_sum(total);
  if (lane < top_k) {
    ids[row * top_k + lane] = id;
    weights[row * top_k + lane] = id >= 0 ? p / total * scale : 0.0f;
  }
}

}  // namespace

hipError_t launch_repack_experts(const uint8_t *p4, uint8_t *out, int64_t experts, int64_t rows,
                                 int64_t cols, hipStream_t s) {
  const ExpertLayout lay = expert_layout(rows, cols);
  // a launch holds fewer than 2^32 threads: experts in as many as it takes
  const int64_t per = (int64_t)lay.tiles * lay.steps * 64;
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

hipError_t launch_selftest_silu(unsigned long long *out, hipStream_t s) {
  for (uint32_t half = 0; half < 2; ++half) {
    hipLaunchKernelGGL(selftest_silu_kernel, dim3(1u << 23), dim3(256), 0, s, half << 31, out);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

int32_t expert_tile_rows(int64_t slots, int64_t experts, int64_t widest) {
  const int64_t some = std::max<int64_t>(1, std::min(slots, experts));
  const int64_t mean = slots / some;
  int32_t rows = slots * 2 <= 3 * some ? 4 : mean <= 4 ? 8 : mean <= 10 ? 16 : mean <= 28 ? 32 : 64;
  // the few-slot kernel keeps its rows in LDS
  const FewLds lds = FewLds::of((int)((widest / kBlock + 3) / 4));
  while (rows > 4 && rows <= 16 && lds.bytes(rows) + kFewBox > kFewLdsMost / 2) rows /= 2;
  return rows <= 16 && lds.bytes(rows) + kFewBox > kFewLdsMost ? 32 : rows;
}

bool expert_planned(int64_t slots, int64_t experts, int32_t tile_rows) {
  return slots > kDirectSlots || tile_rows > 16 || (tile_rows > 4 && experts >= kDirectSlots);
}

int64_t expert_max_tiles(int64_t slots, int64_t experts, int32_t tile_rows) {
  return (slots / tile_rows + std::min(slots, experts + 1) + 7) / 8 * 8;
}

int64_t expert_plan_ints(int64_t slots, int64_t experts, int32_t tile_rows) {
  return 4 * expert_max_tiles(slots, experts, tile_rows) + (slots + 3) / 4 * 4;
}

hipError_t launch_expert_prepare(const int32_t *ids, int64_t slots, int32_t experts,
                                 int32_t tile_rows, int32_t *plan, int32_t *err_flag, const void *x, bool bf16, int64_t m, int64_t ldx,
                                 int64_t cols, int8_t *qa, float *sa, hipStream_t s) {
  // one unit per thread as long as that leaves CUs without a workgroup
  const int64_t units = x ? m * (cols / kBlock) : 0;
  const int32_t per = units <= 128 * (int64_t)cu_count() ? 1 : kQuantUnits;
  const int64_t wgs = 1 + (units + 128 * per - 1) / (128 * per);
  if (wgs * 1024 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  const int aligned = (uintptr_t)x % (bf16 ? 8 : 16) == 0 && ldx % 4 == 0;
  hipLaunchKernelGGL(expert_prepare_kernel, dim3((unsigned)wgs), dim3(1024), 0, s, ids, (int32_t)slots,
                     experts, tile_rows, (int32_t)expert_max_tiles(slots, experts, tile_rows), plan,
                     err_flag, x, bf16 ? 1 : 0, aligned, ldx, m, (int32_t)(cols / kBlock), per, qa, sa);
  return hipGetLastError();
}

// Column ranges of 32 to 128 columns, `repeat` of them per workgroup: as many as
// leave 8 workgroups (few slots) or 20 (many) per CU for about as many tiles as
// there is work for.
void expert_ranges(int64_t slots, int64_t experts, int32_t tile_rows, int64_t rows, bool dual,
                   int32_t test_repeat, int32_t *n_groups, int32_t *repeat) {
  const bool few = tile_rows <= 16;
  const int64_t cols = (dual ? 32 : 64) * (few ? 1 : 2), groups = (rows + cols - 1) / cols;
  const int64_t some = std::min(slots, experts), tiles = few ? some : std::max(slots / tile_rows, some);
  int64_t want = std::max<int64_t>(1, tiles * groups / ((few ? 8 : 20) * (int64_t)cu_count()));
  if (test_repeat > 0) want = test_repeat;
  *n_groups = (int32_t)((groups + std::min(want, groups) - 1) / std::min(want, groups));
  *repeat = (int32_t)((groups + *n_groups - 1) / *n_groups);
}

template <int NV, bool DUAL>
static hipError_t launch_few(ExpertArgs &a, bool fma, hipStream_t s) {
  const int64_t tiles = a.plan ? a.max_tiles
                        : NV == 1 ? a.slots
                                  : a.slots / (4 * NV) + std::min(a.slots, a.experts + 1);
  const int64_t wgs = tiles * a.n_groups;
  // HIP bounds a grid's work-items by 2^32 - 1
  if (wgs * 256 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  const size_t lds = FewLds::of(a.lay.steps).bytes(std::min(4 * NV, a.slots)) + (DUAL ? kFewBox : 0);
  if (fma)
    hipLaunchKernelGGL((expert_few_kernel<NV, true, DUAL>), dim3((unsigned)wgs), dim3(256), lds, s, a);
  else
    hipLaunchKernelGGL((expert_few_kernel<NV, false, DUAL>), dim3((unsigned)wgs), dim3(256), lds, s, a);
  return hipGetLastError();
}

template <int TT, bool DUAL>
static hipError_t launch_many(ExpertArgs &a, bool fma, hipStream_t s) {
  const int64_t wgs = (int64_t)a.max_tiles * a.n_groups;
  if (wgs * 256 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  if (fma)
    hipLaunchKernelGGL((expert_many_kernel<TT, true, DUAL>), dim3((unsigned)wgs), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((expert_many_kernel<TT, false, DUAL>), dim3((unsigned)wgs), dim3(256), 0, s, a);
  return hipGetLastError();
}

static ExpertArgs expert_args(const ExpertLaunch &l) {
  ExpertArgs a = {};
  a.qa = l.qa;
  a.sa = l.sa;
  a.x = l.x;
  a.ldx = l.ldx;
  a.x_type = l.x ? (l.bf16 ? 2 : 1) : 0;
  a.x_aligned = (uintptr_t)l.x % (l.bf16 ? 8 : 16) == 0 && l.ldx % 4 == 0 ? 1 : 0;
  a.per_row = l.per_row;
  a.in_rows = l.in_rows;
  a.ids = l.ids;
  a.err = l.err_flag;
  a.slots = (int32_t)l.slots;
  a.experts = l.experts;
  a.plan = l.plan;
  a.max_tiles = (int32_t)expert_max_tiles(l.slots, l.experts, l.tile_rows);
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
  return a;
}

hipError_t launch_experts(const ExpertLaunch &l, hipStream_t s) {
  ExpertArgs a = expert_args(l);
  const bool dual = l.up != nullptr;
  expert_ranges(l.slots, l.experts, l.tile_rows, l.rows, dual, l.test_repeat, &a.n_groups, &a.repeat);
  switch (l.tile_rows) {
    case 4:
      return dual ? launch_few<1, true>(a, l.fma, s) : launch_few<1, false>(a, l.fma, s);
    case 8:
      return dual ? launch_few<2, true>(a, l.fma, s) : launch_few<2, false>(a, l.fma, s);
    case 16:
      return dual ? launch_few<4, true>(a, l.fma, s) : launch_few<4, false>(a, l.fma, s);
    case 32:
      return dual ? launch_many<1, true>(a, l.fma, s) : launch_many<1, false>(a, l.fma, s);
    default:
      return dual ? launch_many<2, true>(a, l.fma, s) : launch_many<2, false>(a, l.fma, s);
  }
}

bool expert_token_takes(int64_t m, int32_t top_k, int64_t experts, int64_t cols, int64_t width) {
  // An expert's weight read once per slot: as long as few tokens share one.  8
  // of 128 experts of [768, 2560] per token, against the kernels that share:
  // 2 tokens 26 us against 32, 4 42 / 46, 6 57 / 61, 8 73 / 71, 12 108 / 91.
  return (m == 1 || m * top_k * 5 <= experts * 2) && token_up_lds(expert_layout(16, cols).steps) <= 150 * 1024 &&
         std::min(top_k, kTokenWaves) * token_lds(expert_layout(16, width).steps) <= 150 * 1024;
}

template <bool FMA, bool BF16>
static hipError_t launch_token_up(const ExpertArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows / 8), (unsigned)a.slots), wg(256);
  const size_t lds = (size_t)token_up_lds(a.lay.steps);
  if (!a.x_type)
    hipLaunchKernelGGL((expert_token_up_kernel<FMA, BF16, ROW_Q8>), grid, wg, lds, s, a);
  else
    hipLaunchKernelGGL((expert_token_up_kernel<FMA, BF16, BF16 ? ROW_BF16 : ROW_F32>), grid, wg, lds, s, a);
  return hipGetLastError();
}

hipError_t launch_expert_token_up(const ExpertLaunch &l, hipStream_t s) {
  const ExpertArgs a = expert_args(l);
  if (l.fma) return l.bf16 ? launch_token_up<true, true>(a, s) : launch_token_up<true, false>(a, s);
  return l.bf16 ? launch_token_up<false, true>(a, s) : launch_token_up<false, false>(a, s);
}

hipError_t launch_expert_token(const ExpertLaunch &l, const float *weights, int32_t top_k, int64_t m,
                               const void *residual, int64_t ldr, void *y, int64_t ldy, hipStream_t s) {
  const ExpertArgs a = expert_args(l);
  const int waves = std::min(top_k, kTokenWaves);
  const dim3 grid((unsigned)a.lay.tiles, (unsigned)m), wg(64 * waves);
  const size_t lds = (size_t)waves * token_lds(a.lay.steps);
  if (l.fma && l.bf16)
    hipLaunchKernelGGL((expert_token_kernel<true, true>), grid, wg, lds, s, a, weights, top_k, residual, ldr, y, ldy);
  else if (l.fma)
    hipLaunchKernelGGL((expert_token_kernel<true, false>), grid, wg, lds, s, a, weights, top_k, residual, ldr, y, ldy);
  else if (l.bf16)
    hipLaunchKernelGGL((expert_token_kernel<false, true>), grid, wg, lds, s, a, weights, top_k, residual, ldr, y, ldy);
  else
    hipLaunchKernelGGL((expert_token_kernel<false, false>), grid, wg, lds, s, a, weights, top_k, residual, ldr, y, ldy);
  return hipGetLastError();
}

hipError_t launch_expert_combine(const void *o, const int32_t *ids, const float *w, int32_t top_k,
                                 int32_t experts, int64_t m, int64_t cols, const void *residual,
                                 int64_t ldr, void *y, int64_t ldy, bool bf16, hipStream_t s) {
  // Eight bf16 columns (16 B) per thread once that fills the chip (2048 lanes
  // per CU), four before: 4096 rows of 8 x 2560 35.1 us (6.0 TB/s) against 41,
  // 333 rows 7.0 against 6.4, 16 rows 5.2 against 4.5.
  const int v = bf16 && m * (cols / 8) >= (int64_t)cu_count() * 2048 ? 8 : 4;
  const int64_t wgs = (m * (cols / v) + 255) / 256;
  if (wgs * 256 > 0xFFFFFFFFll) return hipErrorInvalidConfiguration;
  const int64_t a = bf16 ? 8 : 16;
  const int ra = (uintptr_t)residual % a == 0 && ldr % 4 == 0;
  const int ya = (uintptr_t)y % a == 0 && ldy % 4 == 0;
  const auto kernel = !bf16 ? expert_combine_kernel<false, 4>
                      : v == 8 ? expert_combine_kernel<true, 8> : expert_combine_kernel<true, 4>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, s, o, ids, w, top_k, experts, m,
                     (int32_t)cols, residual, ldr, ra, y, ldy, ya);
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
