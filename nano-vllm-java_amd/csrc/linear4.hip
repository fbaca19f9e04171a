// y = x W^T (+ bias) with W in the 4-bit form (nva_linear4_forward).
//
// W is laid out once for the matrix cores (16 x 16 x 32 bf16; outs are rows, rows of x are columns): tiles
// of 16 outs and 128 inputs, lane l = 16 w + r of a tile holding out r's inputs 32 j + 8 w .. + 7 in word j
// of its 16 bytes, and the four scale bytes of an out's inputs as one word, 16 words a tile.  So a wave
// reads a tile as 1 KB in one load and x's rows in whole lines.  Codes times their scale are exact in bf16
// and x goes in as three bf16 parts whose sum it is, so products are those of fp32 and sums are fp32.
// Inputs are padded to 128 and outs to 16 with zeros.
#include "mx4.h"
#include "nva_internal.h"
#include "row_lanes.h"

namespace nva {

namespace {

__host__ __device__ constexpr int in_tiles(int in) { return (in + 127) / 128; }
__host__ __device__ constexpr int out_tiles(int out) { return (out + 15) / 16; }
__host__ __device__ constexpr size_t code_bytes(int out, int in) {
  return (size_t)out_tiles(out) * in_tiles(in) * 1024;
}

// Four outs o .. o + 3 of a row, in one store where all are there and 16-byte aligned (`whole`).
__device__ __forceinline__ void store4(float *y, size_t row, int o, int out, bool whole, const float *bias,
                                       f32x4 v) {
  float *at = y + row * out + o;
  if (bias)
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] += o + r < out ? bias[o + r] : 0.f;
  if (whole) {
    if (o < out) *reinterpret_cast<f32x4 *>(at) = v;
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; r++)
    if (o + r < out) at[r] = v[r];
}

// The scale of step j's inputs.
__device__ __forceinline__ float unit_of(uint32_t scales, int j) {
  return mx4_unit((scales >> (8 * j)) & 0xffu);
}

}  // namespace

__global__ void __launch_bounds__(256) linear4_layout_kernel(const uint8_t *codes, const uint8_t *scales,
                                                             int out, int in, uint8_t *weight) {
  const int kt = in_tiles(in);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)out_tiles(out) * kt * 64) return;
  const int lane = (int)(i & 63), r = lane & 15, w = lane >> 4;
  const int64_t tile = i >> 6;
  const int ot = (int)(tile / kt), s = (int)(tile - (int64_t)ot * kt), o = ot * 16 + r;
  uint8_t *dst = weight + tile * 1024 + lane * 16;
  uint8_t *unit = weight + code_bytes(out, in) + (tile * 16 + r) * 4;
  for (int j = 0; j < 4; j++) {
    const int k = s * 128 + 32 * j;
    const bool there = o < out && k < in;
    const uint8_t *src = codes + (size_t)o * (in / 2) + k / 2 + 4 * w;
    for (int b = 0; b < 4; b++) dst[4 * j + b] = there ? src[b] : 0;
    if (w == 0) unit[j] = there ? scales[(size_t)o * (in / 32) + k / 32] : 0;
  }
}

// A few rows (CG groups of 16): a wave takes NT out tiles and every waves-th input tile of them, and
// makes x's parts in registers; the waves' sums join in LDS.  The contraction is split over blockIdx.y too
// where `sums` is given, a plane for each part.  x comes in lines of RP pairs of rows a group (8, or fewer
// where there are fewer rows) and turns in the wave's own part of LDS: read from memory in the operands'
// order, 16 rows a load, 16 rows took 15 us instead of 10.
// What bounds it is not W's bytes but the launch (2.1 us empty), one trip to memory and the splitting of
// x, which every workgroup does for its own outs.  4096 inputs and 2560 outs (5.6 MB): 1 row 5.1 us, 5 rows
// 7.3, 16 rows 9.5, 48 rows 12.1 and 3.9 for the sum of the planes.
constexpr int kRowFloats = 128 + 4;  // of a row in LDS: 16 rows' 16 bytes lie in different banks

constexpr int kRowHalves = 128 + 8;  // the same of a row's parts

// Few enough rows that x is split before it turns, not after: a lane then splits 4 RP values, not 32.
__host__ __device__ constexpr bool rows_split_first(int cg, int rp) { return cg == 1 && rp <= 4; }
template <int NT, int CG, int RP> __host__ __device__ constexpr int rows_wave_floats() {
  const int x = rows_split_first(CG, RP) ? 3 * RP * kRowHalves : 2 * RP * kRowFloats;
  return NT * CG * 256 > x ? NT * CG * 256 : x;
}

template <int NT, int CG, int RP>
__global__ void __launch_bounds__(NT * CG == 1 ? 1024 : 512)
    linear4_rows_kernel(Linear4Launch a, int per, float *sums) {
  extern __shared__ float4 smem[];
  constexpr int kWave = rows_wave_floats<NT, CG, RP>();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int c = lane & 15, w = lane >> 4;
  const int kt = in_tiles(a.in), ots = out_tiles(a.out);
  const int ot0 = blockIdx.x * NT, s1 = min(kt, ((int)blockIdx.y + 1) * per);
  float *own = reinterpret_cast<float *>(smem) + wave * kWave;
  uint16_t *halves = reinterpret_cast<uint16_t *>(own);
  const u32x4 *codes = reinterpret_cast<const u32x4 *>(a.weight);
  const uint32_t *scales = reinterpret_cast<const uint32_t *>(a.weight + code_bytes(a.out, a.in));
  // What is loaded a tile ahead: W, and x's rows where they are few (else a group ahead).
  constexpr bool AHEAD = rows_split_first(CG, RP);
  struct Loads {
    u32x4 code[NT];
    uint32_t unit[NT];
    f32x4 x[RP];
  };
  f32x4 acc[NT][CG];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int g = 0; g < CG; g++) acc[n][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Behind the rows and the inputs: the last ones again.
  auto load_x = [&](int g, int s, Loads &t) {
    const int k = min(s * 128 + 4 * (lane & 31), a.in - 4);
#pragma unroll
    for (int i = 0; i < RP; i++)
      t.x[i] = *reinterpret_cast<const f32x4 *>(
          a.x + (size_t)min(16 * g + 2 * i + (lane >> 5), a.rows - 1) * a.in + k);
  };
  auto load = [&](int s, Loads &t) {
    if constexpr (AHEAD) load_x(0, s, t);
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const size_t at = (size_t)min(ot0 + n, ots - 1) * kt + s;
      t.code[n] = __builtin_nontemporal_load(codes + at * 64 + lane);
      t.unit[n] = scales[at * 16 + c];
    }
  };
  auto multiply = [&](int s, const Loads &t, Loads &x) {
    bf16x8 wf[4][NT];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int n = 0; n < NT; n++) wf[j][n] = mx4_frag(t.code[n][j], unit_of(t.unit[n], j));
#pragma unroll
    for (int g = 0; g < CG; g++) {
      // (One wave's accesses to LDS keep their order.)
#pragma unroll
      for (int i = 0; i < RP; i++) {
        const int r = 2 * i + (lane >> 5), k = 4 * (lane & 31);
        if constexpr (AHEAD) {
          const float v[4] = {x.x[i][0], x.x[i][1], x.x[i][2], x.x[i][3]};
          uint32_t part[3][2];
          split3_pairs<false, 2>(v, part);
#pragma unroll
          for (int q = 0; q < 3; q++)
            *reinterpret_cast<u32x2 *>(halves + (q * 2 * RP + r) * kRowHalves + k) =
                u32x2{part[q][0], part[q][1]};
        } else {
          *reinterpret_cast<f32x4 *>(own + r * kRowFloats + k) = x.x[i];
        }
      }
      __builtin_amdgcn_wave_barrier();
      if constexpr (!AHEAD) load_x(g + 1 < CG ? g + 1 : 0, g + 1 < CG ? s : min(s + waves, s1 - 1), x);
      const int r = min(c, 2 * RP - 1);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (s * 128 + 32 * j >= a.in) break;
        bf16x8 p[3];
        if constexpr (AHEAD) {
#pragma unroll
          for (int q = 0; q < 3; q++)
            p[q] = *reinterpret_cast<const bf16x8 *>(halves + (q * 2 * RP + r) * kRowHalves + 32 * j + 8 * w);
        } else {
          const float *row = own + r * kRowFloats + 32 * j + 8 * w;
          const f32x4 lo = *reinterpret_cast<const f32x4 *>(row);
          const f32x4 hi = *reinterpret_cast<const f32x4 *>(row + 4);
          const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          split3<false>(v, p);
        }
#pragma unroll
        for (int i = 0; i < 3; i++)
#pragma unroll
          for (int n = 0; n < NT; n++)
            acc[n][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[j][n], p[i], acc[n][g], 0, 0, 0);
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  int s = blockIdx.y * per + wave;
  if (s < s1) {
    Loads even, odd;
    load(s, even);
    if constexpr (!AHEAD) load_x(0, s, even);
    while (true) {
      load(min(s + waves, s1 - 1), odd);
      multiply(s, even, even);
      if ((s += waves) >= s1) break;
      load(min(s + waves, s1 - 1), even);
      multiply(s, odd, AHEAD ? odd : even);
      if ((s += waves) >= s1) break;
    }
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int g = 0; g < CG; g++)
      *(reinterpret_cast<f32x4 *>(own) + (n * CG + g) * 64 + lane) = acc[n][g];
  __syncthreads();
  float *y = sums ? sums + (size_t)blockIdx.y * a.rows * a.out : a.y;
  const float *bias = sums ? nullptr : a.bias;
  const bool whole = a.out % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
  // Four outs of one row a thread: entry (n, g, lane) of every wave, in the waves' order.
  for (int i = threadIdx.x; i < NT * CG * 64; i += blockDim.x) {
    const int l = i & 63, g = (i >> 6) % CG, n = (i >> 6) / CG;
    const int row = 16 * g + (l & 15), o = (ot0 + n) * 16 + 4 * (l >> 4);
    if (row >= a.rows) continue;
    const f32x4 *at = reinterpret_cast<const f32x4 *>(smem) + i;
    f32x4 sum = at[0];
    int v = 1;
    for (; v + 2 < waves; v += 3) {
      const f32x4 p0 = at[v * (kWave / 4)], p1 = at[(v + 1) * (kWave / 4)], p2 = at[(v + 2) * (kWave / 4)];
      sum += p0;
      sum += p1;
      sum += p2;
    }
    for (; v < waves; v++) sum += at[v * (kWave / 4)];
    store4(y, row, o, a.out, whole, bias, sum);
  }
}

// x's parts in the order that the matrix cores read them: [step of 32 inputs][16 rows][part][lane] of 16
// bytes, rows padded to whole groups and inputs to whole tiles with zeros.
__global__ void __launch_bounds__(256) linear4_parts_kernel(const float *x, int rows, int in,
                                                            int row_groups, bf16x8 *parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = (int64_t)in_tiles(in) * 4 * row_groups * 64;
  if (i >= n) return;
  const int lane = (int)(i & 63);
  const int64_t at = i >> 6;  // step * row_groups + group
  const int step = (int)(at / row_groups), g = (int)(at - (int64_t)step * row_groups);
  const int row = g * 16 + (lane & 15), k = step * 32 + (lane >> 4) * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (row < rows && k < in) {
    const float4 *src = reinterpret_cast<const float4 *>(x + (size_t)row * in + k);
    *reinterpret_cast<float4 *>(v) = src[0];
    *reinterpret_cast<float4 *>(v + 4) = src[1];
  }
  bf16x8 p[3];
  split3<false>(v, p);
#pragma unroll
  for (int q = 0; q < 3; q++) parts[(at * 3 + q) * 64 + lane] = p[q];
}

// Many rows: 128 outs x 128 rows a workgroup of eight waves, 64 outs x 32 rows each, over the input tiles
// of one plane.  x's parts come through a ring of kStages steps in LDS and W's codes and scales through
// one of two tiles, copied kStages - 1 steps and one tile ahead; a wave reads its operands of a step from
// LDS while the matrix cores are at the step before.
// 1500 rows, 4096 inputs and 2560 outs: 81 us, 1.16 PFLOP/s of bf16 products (a library product of 8192
// cubed makes 1.22 here), and 11 us for the parts, 5.6 TB/s.  With four waves of 64 x 64, W loaded from
// memory as it was needed and operands read as they were needed it was 173.
constexpr int kTileOuts = 128, kTileRows = 128, kStages = 5;
constexpr int kStageBytes = (kTileRows / 16) * 3 * 1024;
constexpr int kWeightBytes = (kTileOuts / 16) * 2048;  // 1 KB of codes and of scales an out tile
constexpr int kTilesLds = kStages * kStageBytes + 2 * kWeightBytes;

__global__ void __launch_bounds__(512, 2) linear4_tiles_kernel(Linear4Launch a, int row_groups, int per,
                                                               int out_blocks, int row_blocks,
                                                               float *sums) {
  extern __shared__ float4 smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wo = wave & 1, wr = wave >> 1;
  const int kt = in_tiles(a.in), ots = out_tiles(a.out);
  // Workgroups go to the eight XCDs in turn: each takes a run of blocks, the rows' parts in its L2 shared
  // by the outs.
  const int blocks = gridDim.x, eighth = blocks / 8, more = blocks % 8, xcd = blockIdx.x & 7;
  const int id = xcd * eighth + min(xcd, more) + (blockIdx.x >> 3);
  const int z = id / (out_blocks * row_blocks), block = id - z * out_blocks * row_blocks;
  const int s0 = z * per, s1 = min(kt, s0 + per);
  const int row_block = block / out_blocks;
  const int ot0 = (block - row_block * out_blocks) * (kTileOuts / 16), rg0 = row_block * (kTileRows / 16);
  const int steps = (s1 - s0) * 4;
  const uint32_t lds0 = lds_address(smem), ldsw = lds0 + kStages * kStageBytes;
  const float *parts = static_cast<const float *>(a.work);
  // A stage's bytes are contiguous in memory up to the last row group, behind which zeros are read.
  const int stage_bytes = min(kTileRows / 16, row_groups - rg0) * 3 * 1024;
  constexpr int kCopies = kStageBytes / 8192, kWeightCopies = 2;  // a wave's
  auto copy = [&](int step) {  // behind the last step: that one again, to keep the counts of copies
    const int at = s0 * 4 + min(step, steps - 1);
    const float *src = parts + ((size_t)at * row_groups + rg0) * (3 * 256);
    const uint32_t dst = lds0 + (step % kStages) * kStageBytes;
#pragma unroll
    for (int i = 0; i < kCopies; i++) {
      const int off = (i * 8 + wave) * 1024;
      copy16_to_lds_async(src, stage_bytes, off + lane * 16, dst + off);
    }
  };
  const int ot = min(ot0 + wave, ots - 1);  // the out tile that this wave copies
  auto copy_weight = [&](int s) {
    const size_t at = (size_t)ot * kt + min(s, s1 - 1);
    const uint32_t dst = ldsw + (s & 1) * kWeightBytes + wave * 2048;
    copy16_to_lds_async(reinterpret_cast<const float *>(a.weight + at * 1024), 1024, lane * 16, dst);
    // (Only the first 64 bytes are this tile's; lanes behind them read zeros.)
    copy16_to_lds_async(reinterpret_cast<const float *>(a.weight + code_bytes(a.out, a.in) + at * 64), 64,
                        lane * 16, dst + 1024);
  };
  f32x4 acc[4][2];
#pragma unroll
  for (int n = 0; n < 4; n++)
#pragma unroll
    for (int g = 0; g < 2; g++) acc[n][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  copy_weight(s0);
#pragma unroll
  for (int i = 0; i < kStages - 1; i++) copy(i);
  const bf16x8 *xs = reinterpret_cast<const bf16x8 *>(smem) + wr * 2 * 3 * 64 + lane;
  const char *ws = reinterpret_cast<const char *>(smem) + kStages * kStageBytes + wo * 4 * 2048;
  u32x4 code[2][4];
  uint32_t unit[2][4];
  bf16x8 p[2][2][3];
  auto read_weight = [&](int s, u32x4 *code, uint32_t *unit) {
    const char *tile = ws + (s & 1) * kWeightBytes;
#pragma unroll
    for (int n = 0; n < 4; n++) {
      code[n] = *(reinterpret_cast<const u32x4 *>(tile + n * 2048) + lane);
      unit[n] = *(reinterpret_cast<const uint32_t *>(tile + n * 2048 + 1024) + (lane & 15));
    }
  };
  auto read_x = [&](int step, bf16x8 (*p)[3]) {
    const bf16x8 *stage = xs + (step % kStages) * (kStageBytes / 16);
#pragma unroll
    for (int g = 0; g < 2; g++)
#pragma unroll
      for (int i = 0; i < 3; i++) p[g][i] = stage[(g * 3 + i) * 64];
  };
  wait_copies<(kStages - 2) * kCopies>();
  lds_barrier();
  read_weight(s0, code[0], unit[0]);
  read_x(0, p[0]);
  wait_lds_reads();
  auto tile_of = [&](int s, const u32x4 *code, const uint32_t *unit, u32x4 *next, uint32_t *next_unit) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int step = (s - s0) * 4 + j;
      // The next step's copies have landed once at most those of the kStages - 3 steps behind it are
      // outstanding, and those of the next tile of W where they were issued after them.
      if (j == 1 || j == 2) wait_copies<(kStages - 3) * kCopies + kWeightCopies>();
      else wait_copies<(kStages - 3) * kCopies>();
      lds_barrier();  // every wave's copies, and every wave has read what the next ones overwrite
      if (j == 0) copy_weight(s + 1);
      copy(step + kStages - 1);
      if (j == 3) read_weight(s + 1, next, next_unit);
      read_x(step + 1, p[(j + 1) & 1]);
      bf16x8 wf[4];
#pragma unroll
      for (int n = 0; n < 4; n++) wf[n] = mx4_frag(code[n][j], unit_of(unit[n], j));
#pragma unroll
      for (int i = 0; i < 3; i++)
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int g = 0; g < 2; g++)
            acc[n][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[n], p[j & 1][g][i], acc[n][g], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      wait_lds_reads();
    }
  };
  for (int s = s0; s < s1; s += 2) {
    tile_of(s, code[0], unit[0], code[1], unit[1]);
    if (s + 1 < s1) tile_of(s + 1, code[1], unit[1], code[0], unit[0]);
  }
  wait_copies<0>();
  const int c = lane & 15, w = lane >> 4;
  float *dst = sums ? sums + (size_t)z * a.rows * a.out : a.y;
  const float *bias = sums ? nullptr : a.bias;
  const bool whole = a.out % 4 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
#pragma unroll
  for (int g = 0; g < 2; g++) {
    const int row = (rg0 + wr * 2 + g) * 16 + c;
    if (row >= a.rows) continue;
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const int o = (ot0 + 4 * wo + n) * 16 + 4 * w;
      store4(dst, row, o, a.out, whole, bias, acc[n][g]);
    }
  }
}

// The planes of a split contraction, added in order (four planes of 48 rows of 2560: 3.9 us, half of it the
// launch).
__global__ void __launch_bounds__(256) linear4_sum_kernel(const float *sums, int planes, int64_t n,
                                                          int out, const float *bias, float *y) {
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    float s = sums[i];
    for (int p = 1; p < planes; p++) s += sums[p * n + i];
    y[i] = s + (bias ? bias[i % out] : 0.f);
  }
}

size_t linear4_bytes(int out, int in) {
  return code_bytes(out, in) + (size_t)out_tiles(out) * in_tiles(in) * 64;
}

hipError_t launch_linear4_layout(const uint8_t *codes, const uint8_t *scales, int out, int in,
                                 uint8_t *weight, hipStream_t s) {
  const int64_t lanes = (int64_t)out_tiles(out) * in_tiles(in) * 64;
  hipLaunchKernelGGL(linear4_layout_kernel, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, s,
                     codes, scales, out, in, weight);
  return hipGetLastError();
}

namespace {

// 64 rows of 4096 inputs and 2560 outs: 18.6 us, and 22 as 128 x 128 tiles.
constexpr int kFewRows = 64;
struct Plan4 {
  bool few;
  int groups;  // of 16 rows
  int outs;    // out tiles of a workgroup of the few-rows kernel
  int waves;
  int planes, per;
  size_t parts_bytes, sums_bytes;
};

Plan4 plan_of(const Linear4Launch &a, int num_cus) {
  Plan4 p{};
  const int kt = in_tiles(a.in), ots = out_tiles(a.out);
  p.few = a.rows <= kFewRows;
  p.groups = (a.rows + 15) / 16;
  int planes = 1;
  if (p.few) {
    // More than 16 rows: more outs a wave, for each splits x anew (17 rows: 12.3 us with 4 out tiles, 14.6
    // with 2; 64 rows 18.6 with 2 and 23.7, for the registers, with 4), and the contraction split as far as
    // one workgroup a CU and one tile a wave go.
    p.outs = p.groups == 1 ? 1 : p.groups == 2 ? 4 : 2;
    p.waves = std::min(p.groups == 1 ? 16 : 8, kt);
    if (p.groups > 1)
      planes = std::max(1, std::min(num_cus / ((ots + p.outs - 1) / p.outs), kt / p.waves));
  } else {
    // The contraction is split while the 128 x 128 blocks leave CUs idle and a part keeps 4 input tiles.
    const int64_t blocks = (int64_t)((a.out + kTileOuts - 1) / kTileOuts) *
                           ((a.rows + kTileRows - 1) / kTileRows);
    planes = (int)std::max<int64_t>(1, std::min<int64_t>(num_cus / blocks, kt / 4));
    p.parts_bytes = ((size_t)kt * 4 * p.groups * 3 * 1024 + 255) / 256 * 256;
  }
  p.per = (kt + planes - 1) / planes;
  p.planes = (kt + p.per - 1) / p.per;
  p.sums_bytes = p.planes > 1 ? (size_t)p.planes * a.rows * a.out * 4 : 0;
  return p;
}

template <int NT, int CG, int RP>
hipError_t rows_kernel(const Linear4Launch &a, const Plan4 &p, float *sums, hipStream_t s) {
  const int lds = p.waves * rows_wave_floats<NT, CG, RP>() * 4;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&linear4_rows_kernel<NT, CG, RP>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((linear4_rows_kernel<NT, CG, RP>), dim3((out_tiles(a.out) + NT - 1) / NT, p.planes),
                     dim3(64 * p.waves), lds, s, a, p.per, sums);
  return hipGetLastError();
}

}  // namespace

size_t linear4_work_bytes(const Linear4Launch &a, int num_cus) {
  const Plan4 p = plan_of(a, num_cus);
  return p.parts_bytes + p.sums_bytes;
}

hipError_t launch_linear4(const Linear4Launch &a, int num_cus, hipStream_t s) {
  const Plan4 p = plan_of(a, num_cus);
  float *sums = p.sums_bytes ? reinterpret_cast<float *>(static_cast<char *>(a.work) + p.parts_bytes)
                             : nullptr;
  hipError_t e;
  if (p.few) {
    switch (p.groups) {
      case 1:
        e = a.rows <= 2   ? rows_kernel<1, 1, 1>(a, p, sums, s)
            : a.rows <= 8 ? rows_kernel<1, 1, 4>(a, p, sums, s)
                          : rows_kernel<1, 1, 8>(a, p, sums, s);
        break;
      case 2: e = rows_kernel<4, 2, 8>(a, p, sums, s); break;
      case 3: e = rows_kernel<2, 3, 8>(a, p, sums, s); break;
      default: e = rows_kernel<2, 4, 8>(a, p, sums, s); break;
    }
  } else {
    const int64_t n = (int64_t)in_tiles(a.in) * 4 * p.groups * 64;
    hipLaunchKernelGGL(linear4_parts_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.x,
                       a.rows, a.in, p.groups, static_cast<bf16x8 *>(a.work));
    e = hipGetLastError();
    if (e == hipSuccess)
      e = hipFuncSetAttribute(reinterpret_cast<const void *>(&linear4_tiles_kernel),
                              hipFuncAttributeMaxDynamicSharedMemorySize, kTilesLds);
    if (e != hipSuccess) return e;
    const int out_blocks = (a.out + kTileOuts - 1) / kTileOuts;
    const int row_blocks = (a.rows + kTileRows - 1) / kTileRows;
    hipLaunchKernelGGL(linear4_tiles_kernel, dim3((unsigned)out_blocks * row_blocks * p.planes), dim3(512),
                       kTilesLds, s, a, p.groups, p.per, out_blocks, row_blocks, sums);
    e = hipGetLastError();
  }
  if (e != hipSuccess || !sums) return e;
  const int64_t entries = (int64_t)a.rows * a.out;
  hipLaunchKernelGGL(linear4_sum_kernel, dim3((unsigned)std::min<int64_t>((entries + 255) / 256, 4096)),
                     dim3(256), 0, s, sums, p.planes, entries, a.out, a.bias, a.y);
  return hipGetLastError();
}

}  // namespace nva
