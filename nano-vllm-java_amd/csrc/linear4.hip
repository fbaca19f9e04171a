// y = x W^T (+ bias) with W in the 4-bit form (nva_linear4_forward).
//
// W is laid out once for the matrix cores (16 x 16 x 32 bf16; outs are rows, rows of x are columns): tiles
// of 16 outs and 128 inputs, lane l = 16 w + r of a tile holding out r's inputs 32 w .. 32 w + 31, one
// 4-bit block (16 bytes and one scale byte), so a wave reads a tile as 1 KB in one load and a lane's
// scale is its own; step j of a tile's four contracts inputs 32 w + 8 j .. + 7 of every quarter w.  Codes
// are exact in bf16 and x goes in as three bf16 parts whose sum it is, so products are those of fp32 and
// sums are fp32.  Inputs are padded to 128 and outs to 16 with zeros.
#include "mx4.h"
#include "nva_internal.h"
#include "row_lanes.h"

namespace nva {

namespace {

__host__ __device__ constexpr int in_tiles(int in) { return (in + 127) / 128; }
__host__ __device__ constexpr int out_tiles(int out) { return (out + 15) / 16; }
// Scale bytes of four tiles along the inputs lie together: one 32-bit word a lane.
__host__ __device__ constexpr int scale_groups(int in) { return (in_tiles(in) + 3) / 4; }
__host__ __device__ constexpr size_t code_bytes(int out, int in) {
  return (size_t)out_tiles(out) * in_tiles(in) * 1024;
}

// x[row, k .. k + 8) as three parts; zeros behind the inputs.
__device__ __forceinline__ void load_parts(const float *x, int k, int in, bf16x8 *parts) {
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (k < in) {
    *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x + k);
    *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(x + k + 4);
  }
  split3<false>(v, parts);
}

}  // namespace

__global__ void __launch_bounds__(256) linear4_layout_kernel(const uint8_t *codes, const uint8_t *scales,
                                                             int out, int in, uint8_t *weight) {
  const int kt = in_tiles(in);
  const int64_t lanes = (int64_t)out_tiles(out) * scale_groups(in) * 4 * 64;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= lanes) return;
  const int lane = (int)(i & 63);
  const int64_t tile = i >> 6;
  const int per = scale_groups(in) * 4;
  const int ot = (int)(tile / per), s = (int)(tile - (int64_t)ot * per);
  const int o = ot * 16 + (lane & 15), k = s * 128 + (lane >> 4) * 32;
  const bool there = o < out && k < in;
  if (s < kt) {
    uint8_t *dst = weight + ((size_t)ot * kt + s) * 1024 + lane * 16;
    const uint8_t *src = codes + (size_t)o * (in / 2) + k / 2;
    for (int b = 0; b < 16; b++) dst[b] = there ? src[b] : 0;
  }
  weight[code_bytes(out, in) + (((size_t)ot * scale_groups(in) + (s >> 2)) * 64 + lane) * 4 + (s & 3)] =
      there ? scales[(size_t)o * (in / 32) + k / 32] : 0;
}

// A few rows: a workgroup takes NT out tiles, its waves every WV-th input tile of them, and x's parts are
// made in registers, CG groups of 16 rows.  W is read once from HBM; the waves' sums join in LDS.
template <int NT, int CG>
__global__ void __launch_bounds__(1024) linear4_rows_kernel(Linear4Launch a) {
  extern __shared__ f32x4 lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int c = lane & 15, w = lane >> 4;
  const int kt = in_tiles(a.in), groups = scale_groups(a.in), ots = out_tiles(a.out);
  const int ot0 = blockIdx.x * NT;
  const uint8_t *scales = a.weight + code_bytes(a.out, a.in);
  f32x4 acc[NT][CG];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int g = 0; g < CG; g++) acc[n][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float *x[CG];
#pragma unroll
  for (int g = 0; g < CG; g++) x[g] = a.x + (size_t)min(16 * g + c, a.rows - 1) * a.in;
  for (int s = wave; s < kt; s += waves) {
    u32x4 code[NT];
    float unit[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int ot = min(ot0 + n, ots - 1);
      code[n] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4 *>(a.weight + ((size_t)ot * kt + s) * 1024) + lane);
      unit[n] = mx4_unit(scales[(((size_t)ot * groups + (s >> 2)) * 64 + lane) * 4 + (s & 3)]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      bf16x8 wf[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) wf[n] = mx4_frag(code[n][j], unit[n]);
#pragma unroll
      for (int g = 0; g < CG; g++) {
        bf16x8 p[3];
        load_parts(x[g], s * 128 + w * 32 + 8 * j, a.in, p);
#pragma unroll
        for (int i = 0; i < 3; i++)
#pragma unroll
          for (int n = 0; n < NT; n++)
            acc[n][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[n], p[i], acc[n][g], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int g = 0; g < CG; g++) lds[((wave * NT + n) * CG + g) * 64 + lane] = acc[n][g];
  __syncthreads();
  // Four outs of one row a thread: entry (n, g, lane) of every wave, in the waves' order.
  for (int i = threadIdx.x; i < NT * CG * 64; i += blockDim.x) {
    f32x4 sum = lds[i];
    for (int v = 1; v < waves; v++) sum += lds[v * NT * CG * 64 + i];
    const int l = i & 63, g = (i >> 6) % CG, n = (i >> 6) / CG;
    const int row = 16 * g + (l & 15), o = (ot0 + n) * 16 + 4 * (l >> 4);
    if (row >= a.rows) continue;
    float *y = a.y + (size_t)row * a.out + o;
#pragma unroll
    for (int r = 0; r < 4; r++)
      if (o + r < a.out) y[r] = sum[r] + (a.bias ? a.bias[o + r] : 0.f);
  }
}

// x's parts in the order that the matrix cores read them: [step (128-input tile, j)][16 rows][part][lane]
// of 16 bytes, rows padded to whole groups.
__global__ void __launch_bounds__(256) linear4_parts_kernel(const float *x, int rows, int in,
                                                            int row_groups, bf16x8 *parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = (int64_t)in_tiles(in) * 4 * row_groups * 64;
  if (i >= n) return;
  const int lane = (int)(i & 63);
  const int64_t at = i >> 6;  // step * row_groups + group
  const int step = (int)(at / row_groups), g = (int)(at - (int64_t)step * row_groups);
  const int row = g * 16 + (lane & 15), k = (step >> 2) * 128 + (lane >> 4) * 32 + (step & 3) * 8;
  bf16x8 p[3];
  load_parts(x + (size_t)min(row, rows - 1) * in, row < rows ? k : in, in, p);
#pragma unroll
  for (int q = 0; q < 3; q++) parts[(at * 3 + q) * 64 + lane] = p[q];
}

// Many rows: 128 outs x 128 rows a workgroup, four waves of 64 x 64, over the input tiles
// [blockIdx.z * per, + per); W goes from memory to registers, x's parts through LDS.
constexpr int kTileOuts = 128, kTileRows = 128, kStages = 3;
constexpr int kStageBytes = (kTileRows / 16) * 3 * 1024;

__global__ void __launch_bounds__(256, 2) linear4_tiles_kernel(Linear4Launch a, int row_groups, int per,
                                                               float *sums) {
  extern __shared__ float4 smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wo = wave & 1, wr = wave >> 1;
  const int kt = in_tiles(a.in), groups = scale_groups(a.in), ots = out_tiles(a.out);
  const int s0 = blockIdx.z * per, s1 = min(kt, s0 + per);
  const int ot0 = blockIdx.x * (kTileOuts / 16) + 4 * wo, rg0 = blockIdx.y * (kTileRows / 16);
  const uint8_t *scales = a.weight + code_bytes(a.out, a.in);
  const int steps = (s1 - s0) * 4;
  const uint32_t lds0 = lds_address(smem);
  const float *parts = static_cast<const float *>(a.work);
  // A stage's bytes are contiguous in memory up to the last row group, behind which zeros are read.
  const int stage_bytes = min(kTileRows / 16, row_groups - rg0) * 3 * 1024;
  auto copy = [&](int step) {  // stage of one contraction step
    const float *src = parts + ((size_t)(s0 * 4 + step) * row_groups + rg0) * (3 * 256);
    const uint32_t dst = lds0 + (step % kStages) * kStageBytes;
#pragma unroll
    for (int i = 0; i < kStageBytes / 4096; i++) {
      const int at = (i * 4 + wave) * 1024;
      copy16_to_lds_async(src, stage_bytes, at + lane * 16, dst + at);
    }
  };
  constexpr int kCopies = kStageBytes / 4096;  // a wave's copies of a stage
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int g = 0; g < 4; g++) acc[i][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 code[4];
  float unit[4];
  auto load_w = [&](int s, u32x4 *cd, float *un) {
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const int ot = min(ot0 + n, ots - 1);
      cd[n] = *(reinterpret_cast<const u32x4 *>(a.weight + ((size_t)ot * kt + s) * 1024) + lane);
      un[n] = mx4_unit(scales[(((size_t)ot * groups + (s >> 2)) * 64 + lane) * 4 + (s & 3)]);
    }
  };
  copy(0);
  if (steps > 1) copy(1);
  const bf16x8 *xs = reinterpret_cast<const bf16x8 *>(smem);
  for (int step = 0; step < steps; step++) {
    if ((step & 3) == 0) load_w(s0 + (step >> 2), code, unit);
    // This step's copies have landed once only those of the next are outstanding (W's loads are waited
    // for by the compiler, before or after).
    if (step + 1 < steps && (step & 3) != 0) wait_copies<kCopies>(); else wait_copies<0>();
    lds_barrier();  // every wave's copies, and every wave is done with the stage two steps back
    if (step + 2 < steps) copy(step + 2);
    const bf16x8 *stage = xs + (step % kStages) * (kStageBytes / 16) + wr * 4 * 3 * 64 + lane;
    bf16x8 wf[4];
    const int j = step & 3;
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const uint32_t word = j == 0 ? code[n].x : j == 1 ? code[n].y : j == 2 ? code[n].z : code[n].w;
      wf[n] = mx4_frag(word, unit[n]);
    }
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
      for (int i = 0; i < 3; i++) {
        const bf16x8 p = stage[(g * 3 + i) * 64];
#pragma unroll
        for (int n = 0; n < 4; n++)
          acc[n][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[n], p, acc[n][g], 0, 0, 0);
      }
    wait_lds_reads();
  }
  const int c = lane & 15, w = lane >> 4;
  float *dst = sums ? sums + (size_t)blockIdx.z * a.rows * a.out : a.y;
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const int row = (rg0 + wr * 4 + g) * 16 + c;
    if (row >= a.rows) continue;
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const int o = (ot0 + n) * 16 + 4 * w;
#pragma unroll
      for (int r = 0; r < 4; r++)
        if (o + r < a.out)
          dst[(size_t)row * a.out + o + r] = acc[n][g][r] + (!sums && a.bias ? a.bias[o + r] : 0.f);
    }
  }
}

// The planes of a split contraction, added in order.
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
  return code_bytes(out, in) + (size_t)out_tiles(out) * scale_groups(in) * 256;
}

hipError_t launch_linear4_layout(const uint8_t *codes, const uint8_t *scales, int out, int in,
                                 uint8_t *weight, hipStream_t s) {
  const int64_t lanes = (int64_t)out_tiles(out) * scale_groups(in) * 4 * 64;
  hipLaunchKernelGGL(linear4_layout_kernel, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, s,
                     codes, scales, out, in, weight);
  return hipGetLastError();
}

namespace {

constexpr int kFewRows = 64;

struct TilePlan {
  int row_groups, planes, per;
  size_t parts_bytes, sums_bytes;
};

// The contraction is split while the 128 x 128 blocks leave CUs idle and a part keeps 4 input tiles.
TilePlan tile_plan(const Linear4Launch &a, int num_cus) {
  TilePlan p{};
  p.row_groups = (a.rows + 15) / 16;
  const int64_t blocks = (int64_t)((a.out + kTileOuts - 1) / kTileOuts) *
                         ((a.rows + kTileRows - 1) / kTileRows);
  const int kt = in_tiles(a.in);
  int planes = (int)std::max<int64_t>(1, std::min<int64_t>(num_cus / blocks, kt / 4));
  p.per = (kt + planes - 1) / planes;
  p.planes = (kt + p.per - 1) / p.per;
  p.parts_bytes = ((size_t)kt * 4 * p.row_groups * 3 * 1024 + 255) / 256 * 256;
  p.sums_bytes = p.planes > 1 ? (size_t)p.planes * a.rows * a.out * 4 : 0;
  return p;
}

template <int NT, int CG> hipError_t rows_kernel(const Linear4Launch &a, hipStream_t s) {
  const int kt = in_tiles(a.in);
  int waves = 64 / (NT * CG);  // 64 KB of sums
  waves = std::max(1, std::min({16, waves, kt}));
  hipLaunchKernelGGL((linear4_rows_kernel<NT, CG>), dim3((out_tiles(a.out) + NT - 1) / NT),
                     dim3(64 * waves), (size_t)waves * NT * CG * 1024, s, a);
  return hipGetLastError();
}

}  // namespace

size_t linear4_work_bytes(const Linear4Launch &a, int num_cus) {
  if (a.rows <= kFewRows) return 0;
  const TilePlan p = tile_plan(a, num_cus);
  return p.parts_bytes + p.sums_bytes;
}

hipError_t launch_linear4(const Linear4Launch &a, int num_cus, hipStream_t s) {
  if (a.rows <= kFewRows) {
    const int cg = (a.rows + 15) / 16;
    switch (cg) {
      case 1: return rows_kernel<1, 1>(a, s);
      case 2: return rows_kernel<1, 2>(a, s);
      case 3: return rows_kernel<1, 3>(a, s);
      default: return rows_kernel<1, 4>(a, s);
    }
  }
  const TilePlan p = tile_plan(a, num_cus);
  bf16x8 *parts = static_cast<bf16x8 *>(a.work);
  float *sums = p.sums_bytes ? reinterpret_cast<float *>(static_cast<char *>(a.work) + p.parts_bytes)
                             : nullptr;
  const int64_t n = (int64_t)in_tiles(a.in) * 4 * p.row_groups * 64;
  hipLaunchKernelGGL(linear4_parts_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.x, a.rows,
                     a.in, p.row_groups, parts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int lds = kStages * kStageBytes;
  e = hipFuncSetAttribute(reinterpret_cast<const void *>(&linear4_tiles_kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(linear4_tiles_kernel,
                     dim3((a.out + kTileOuts - 1) / kTileOuts, (a.rows + kTileRows - 1) / kTileRows,
                          p.planes),
                     dim3(256), lds, s, a, p.row_groups, p.per, sums);
  e = hipGetLastError();
  if (e != hipSuccess || !sums) return e;
  const int64_t entries = (int64_t)a.rows * a.out;
  hipLaunchKernelGGL(linear4_sum_kernel, dim3((unsigned)std::min<int64_t>((entries + 255) / 256, 4096)),
                     dim3(256), 0, s, sums, p.planes, entries, a.out, a.bias, a.y);
  return hipGetLastError();
}

}  // namespace nva
