// Attention of runs of query rows that all see one whole key range, for runs of few columns: the
// rows of a step under a shared prefix, or those that read one encoder's states (a row of a step
// alone, too).  Runs of many columns are span tiles (prefill.hip).
//
// Mathematics: column c of a run is query row r = c / H and query head h of one KV head
// (H = col_heads heads of it).  For the keys t of the item,
//   s_ct = q_rh . k_t * scale,  m_c = max_t s_ct,  l_c = sum_t e^(s_ct - m_c),
//   a_c = sum_t e^(s_ct - m_c) v_t;
// an item over the whole range writes a_c / l_c (0 where l_c = 0), a split one or one of a prefix
// leaves (m_c, l_c, a_c), and the merge joins what a row has from its prefix and from its own keys.
//
// Mapping onto CDNA4.  A key costs 8 D bytes of K and V and 4 D operations a column, 8 operations a byte
// on the 16 columns of a matrix instruction: fp32 matrix instructions (which need no scaling and take
// any value; 155 TFLOP/s) keep up with HBM to 32 columns.  Measured: 128 single tokens over 300-1500
// encoder rows (16 heads, d = 64, 0.96 GB) 172 us, 5.6 TB/s; 40 x 5 beams over 500-4000 rows (32 q / 8
// KV heads, d = 128, 0.73 GB) 151 us, 4.9 TB/s.  Short runs of more columns are bound by latency (33 rows
// of 4 heads under 6144 tokens, d = 256: 26 us, 36% of the matrix unit, 5.5 turns a wave).  One workgroup
// of 4 waves per (item, KV head, head group); each wave takes 16-key blocks of the item in turn, so that
// 4 waves read 64 consecutive keys at a time, with no barrier and no LDS until the end:
//   S^T[key][col] = K Q^T    D/4 v_mfma_f32_16x16x4_f32 per block and 16 columns: at step 4v + c
//                            lane (i, g) supplies K[t0 + i][16v + 4g + c] (A) and
//                            Q[col i][16v + 4g + c] (B), i = lane % 16, g = lane / 16;
//                            lane (j, g) then holds column j's scores of keys t0 + 4g + r;
//   O^T[dim][col] += V^T P^T 4 x D/16 per block: step s contracts key t0 + 4g + s, whose
//                            probability is the lane's own (B), against V[key][64w + 4i + c] (A) in
//                            block b = 4w + c, so P never leaves the registers.
// From D = 256 on, 2 or 4 waves share a block by 128 dims each and add their partial scores in LDS.
// K and V have one register buffer, so that two waves share a SIMD on items of 32 columns and three on
// those of 16 (a second buffer leaves one on 32: beams 189 -> 219 us).  K operands serve both blocks of
// 16 columns.  The waves' states meet in LDS in wave order.
#include "nva_internal.h"
#include "nva_device.h"
#include "row_lanes.h"

namespace nva {

namespace {
__device__ __forceinline__ float4 ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ void st4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
// This wave's LDS writes, then the workgroup: unlike __syncthreads(), the loads in flight stay so.
__device__ __forceinline__ void lds_writes_barrier() {
  wait_lds_reads();
  lds_barrier();
}
}  // namespace

template <int D, int NCB, bool PAGED>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
span_kernel(SpanLaunch a) {
  constexpr int DW = D < 128 ? D : 128;  // dims of a wave
  constexpr int DS = D / DW;             // waves that share a key block, by dims
  constexpr int KG = 4 / DS;             // key blocks in turn
  constexpr int DQ = DW / 4;   // QK steps per block
  constexpr int NB = DW / 16;  // O^T blocks; block b = 4w + c, row i is dim 64w + 4i + c of the wave's
  constexpr int NQ = DQ / 4;   // float4 loads of a K row part per lane
  constexpr int NV = NB / 4;   // float4 loads of a V row part per lane per key (one per 64 dims)
  constexpr int COLS = 16 * NCB;
  __shared__ float sm_m[KG][COLS];
  __shared__ float sm_l[KG][COLS];
  __shared__ float4 sm_acc[KG][COLS][D / 4];
  __shared__ int32_t stab[kRowTablePages];

  // Partial scores [turn][wave][column block][lane], until the waves' results meet.
  float4 *const spart = &sm_acc[0][0][0];
  static_assert(DS == 1 || 2 * 4 * NCB * 64 <= KG * COLS * (D / 4), "spart lies in sm_acc");

  const int rep = a.hq / a.hkv;
  const int groups = rep / a.col_heads;
  const int per_item = a.hkv * groups;
  const int item = blockIdx.x / per_item;
  const int gy = blockIdx.x - item * per_item;
  const SpanItem it = a.items[item];
  const int kvh = gy / groups;
  const int h0 = kvh * rep + (gy - kvh * groups) * a.col_heads;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / DS, ds = wave % DS;
  const int i = lane & 15;
  const int g = lane >> 4;

  const size_t rs = (size_t)a.kv.ld;
  const int bs_shift = a.kv.bs_shift;
  const int blk0 = PAGED ? it.kbeg >> bs_shift : 0;
  // An item within at most two pages carries their block ids: no table read before its first loads.
  const bool inl = PAGED && it.blk_a != 0;
  if (PAGED && !inl) {
    const int32_t *table = a.kv.table + (size_t)it.seq * a.kv.bt_stride;
    const int npages = ((it.kend - 1) >> bs_shift) - blk0 + 1;
    for (int j = threadIdx.x; j < npages; j += blockDim.x) stab[j] = table[blk0 + j];
    __syncthreads();
  }
  const float *kbase_h = a.kv.k + (size_t)kvh * D + DW * ds;
  const float *vbase_h = a.kv.v + (size_t)kvh * D + DW * ds;
  const int tfirst = it.kbeg & ~15;  // blocks of pages start at multiples of 16
  // Fixed lane offsets (floats) from a block's first row: K row i, dims 16v + 4g; V rows
  // 4g + s, dims 64w + 4i.
  const uint32_t koff = (uint32_t)(i * rs + 4 * g);
  const uint32_t voff = (uint32_t)(4 * g * rs + 4 * i);

  // The wave's block t0: its rows' base, and this lane's offsets in it (floats).
  struct Block {
    const float *k, *v;
    uint32_t ko, vo[4];
  };
  auto locate = [&](int t0) {
    Block b;
    // A block past the item's end is the item's first: never used up to d = 128, multiplied by weights
    // of 0 from d = 256 on, where the waves of a key group make the same turns.
    const int tb = t0 < it.kend ? t0 : tfirst;
    int64_t row;
    if constexpr (PAGED) {
      const int p = tb >> bs_shift;
      const int id = inl ? (p == blk0 ? it.blk_a - 1 : it.blk_b)
                         : __builtin_amdgcn_readfirstlane(stab[p - blk0]);
      row = (int64_t)id * a.kv.block_size + (tb - (p << bs_shift));
    } else {
      row = (int64_t)it.kbase + tb;
    }
    b.k = kbase_h + row * (int64_t)rs;
    b.v = vbase_h + row * (int64_t)rs;
    b.ko = koff;
#pragma unroll
    for (int s = 0; s < 4; s++) b.vo[s] = voff + (uint32_t)(s * rs);
    if (t0 < it.kbeg || t0 + 16 > it.kend) {
      // A partial block (what lies outside the item could hold any bits, NaN included): K is the block's
      // key nearest the lane's own inside the item, whose score is masked, V is zero.
      const int tk = min(max(tb + i, it.kbeg), it.kend - 1);
      b.ko = (uint32_t)((tk - tb) * (int64_t)rs + 4 * g);
#pragma unroll
      for (int s = 0; s < 4; s++) {
        const int tv = t0 + 4 * g + s;
        if (tv < it.kbeg || tv >= it.kend) b.vo[s] = kOutside;
      }
    }
    return b;
  };
  float kr[DQ], vr[4][NB];
  auto load_k = [&](const Block &b) {
#pragma unroll
    for (int v = 0; v < NQ; v++) {
      const float4 x = ld4_at(b.k, b.ko + 16 * v);
      kr[4 * v] = x.x;
      kr[4 * v + 1] = x.y;
      kr[4 * v + 2] = x.z;
      kr[4 * v + 3] = x.w;
    }
  };
  auto load_v = [&](const Block &b) {
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const float4 x = ld4_at(b.v, b.vo[s] + 64 * v);
        vr[s][4 * v] = x.x;
        vr[s][4 * v + 1] = x.y;
        vr[s][4 * v + 2] = x.z;
        vr[s][4 * v + 3] = x.w;
      }
  };

  // The first block's loads are in flight before Q is read, so that a short item waits once for both
  // (28 requests of up to 408 keys 16.7 -> 16.2 us; two column blocks, whose items are long, lose 2%).
  int t0 = tfirst + 16 * kg;
  const Block at = locate(t0);
  if constexpr (NCB == 1) {
    load_k(at);
    load_v(at);
  }

  // B operand of QK: this lane's columns i and 16 + i, dims 16v + 4g + [0, 4), in log2 units.
  const float sl2 = a.scale * 1.4426950408889634f;
  float q[NCB][DQ];
#pragma unroll
  for (int n = 0; n < NCB; n++) {
    const int c = 16 * n + i;
    if (c < it.cols) {
      const int r = c / a.col_heads;
      const float *qp = a.q + ((size_t)(it.row0 + r) * a.hq + h0 + c - r * a.col_heads) * D +
                        DW * ds + 4 * g;
#pragma unroll
      for (int v = 0; v < NQ; v++) {
        const float4 x = ld4(qp + 16 * v);
        q[n][4 * v] = x.x * sl2;
        q[n][4 * v + 1] = x.y * sl2;
        q[n][4 * v + 2] = x.z * sl2;
        q[n][4 * v + 3] = x.w * sl2;
      }
    } else {
#pragma unroll
      for (int s = 0; s < DQ; s++) q[n][s] = 0.0f;
    }
  }

  if constexpr (NCB > 1) {
    load_k(at);
    load_v(at);
  }

  f32x4 o[NCB][NB];
  float m_run[NCB], l_run[NCB];  // column's max (log2 units, the same in its 4 lanes), lane's sum
#pragma unroll
  for (int n = 0; n < NCB; n++) {
#pragma unroll
    for (int b = 0; b < NB; b++) o[n][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    m_run[n] = -INFINITY;
    l_run[n] = 0.0f;
  }

  // Waves that share a key block meet at every one, so all of the workgroup's make the same turns.
  const int tend = DS == 1 ? it.kend : it.kend + 16 * kg;
  for (int turn = 0; t0 < tend; t0 += 16 * KG, turn ^= 1) {
    f32x4 p[NCB];
#pragma unroll
    for (int n = 0; n < NCB; n++) p[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < DQ; s++)
#pragma unroll
      for (int n = 0; n < NCB; n++)
        p[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[s], q[n][s], p[n], 0, 0, 0);
    // The next block's K is in flight during the softmax and PV, its V during the next QK.
    const Block next = locate(t0 + 16 * KG);
    load_k(next);
    if constexpr (DS > 1) {
      // Scores of all dims, added in the waves' order (so that they hold the same bits).
#pragma unroll
      for (int n = 0; n < NCB; n++)
        spart[((turn * 4 + wave) * NCB + n) * 64 + lane] = make_float4(p[n][0], p[n][1], p[n][2], p[n][3]);
      lds_writes_barrier();
#pragma unroll
      for (int n = 0; n < NCB; n++) {
        const float4 x = spart[((turn * 4 + kg * DS) * NCB + n) * 64 + lane];
        p[n] = f32x4{x.x, x.y, x.z, x.w};
#pragma unroll
        for (int w = 1; w < DS; w++) {
          const float4 y = spart[((turn * 4 + kg * DS + w) * NCB + n) * 64 + lane];
          p[n] += f32x4{y.x, y.y, y.z, y.w};
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NCB; n++) {
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int key = t0 + 4 * g + r;
        p[n][r] = (key >= it.kbeg && key < it.kend) ? p[n][r] : -INFINITY;
        mx = fmaxf(mx, p[n][r]);
      }
      mx = max4_lanes(mx);
      // The max moves, and the sums with it, only where it grows by more than 2^8.
      const bool need = mx > m_run[n] + 8.0f;
      if (__any(need)) {
        const float mn = need ? mx : m_run[n];
        const float alpha = m_run[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - mn);
        l_run[n] *= alpha;
#pragma unroll
        for (int b = 0; b < NB; b++) o[n][b] *= alpha;
        m_run[n] = mn;
      }
      const float ms = m_run[n] == -INFINITY ? 0.0f : m_run[n];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[n][r] = __builtin_amdgcn_exp2f(p[n][r] - ms);
        l_run[n] += p[n][r];
      }
    }
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int n = 0; n < NCB; n++)
          o[n][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[s][b], p[n][s], o[n][b], 0, 0, 0);
    load_v(next);
  }

  if constexpr (DS > 1) __syncthreads();  // every wave is done with spart
#pragma unroll
  for (int n = 0; n < NCB; n++) {
    const int c = 16 * n + i;
    const float l_tot = sum4_lanes(l_run[n]);
    if (c < it.cols) {
      if (g == 0 && ds == 0) {
        sm_m[kg][c] = m_run[n];
        sm_l[kg][c] = l_tot;
      }
      // Lane (i, g) holds row 4g + r of block 4w + b: dim 64w + 16g + 4r + b of the wave's.
#pragma unroll
      for (int w = 0; w < NV; w++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          sm_acc[kg][c][DW / 4 * ds + 16 * w + 4 * g + r] = make_float4(
              o[n][4 * w][r], o[n][4 * w + 1][r], o[n][4 * w + 2][r], o[n][4 * w + 3][r]);
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < it.cols * (D / 4); idx += blockDim.x) {
    const int c = idx / (D / 4);
    const int cc = idx - c * (D / 4);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < KG; w++) M = fmaxf(M, sm_m[w][c]);
    const float Ms = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < KG; w++) {
      const float e = __builtin_amdgcn_exp2f(sm_m[w][c] - Ms);
      L = fmaf(sm_l[w][c], e, L);
      const float4 x = sm_acc[w][c][cc];
      A.x = fmaf(x.x, e, A.x);
      A.y = fmaf(x.y, e, A.y);
      A.z = fmaf(x.z, e, A.z);
      A.w = fmaf(x.w, e, A.w);
    }
    const int r = c / a.col_heads;
    const int h = h0 + c - r * a.col_heads;
    if (it.split < 0) {
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      st4(a.out + ((size_t)(it.row0 + r) * a.hq + h) * D + cc * 4,
          make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv));
    } else {
      const size_t pi = (size_t)(a.row_part[it.row0 + r] + it.split) * a.hq + h;
      st4(a.part_acc + pi * D + cc * 4, A);
      if (cc == 0) {
        a.part_m[pi] = M;
        a.part_l[pi] = L;
      }
    }
  }
}

namespace {

template <int D, int NCB>
void launch_span(const SpanLaunch &a, hipStream_t s) {
  const dim3 grid(a.num_items * (a.hkv * ((a.hq / a.hkv) / a.col_heads)));
  if (a.kv.paged)
    hipLaunchKernelGGL((span_kernel<D, NCB, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((span_kernel<D, NCB, false>), grid, dim3(256), 0, s, a);
}

}  // namespace

// Joins the partials of each row of a plan with spans: a workgroup per (row, head), whose groups of
// D / 4 lanes take every G-th partial, four of them in flight, and meet in LDS in order, so the result
// does not depend on timing.  (The decode merge gives a partial a wave of 64 lanes: of 97 partials at
// d = 64 three quarters of 16 waves idle, in two rounds of workgroups: 10 us for 20 rows of 32 heads,
// 5.0 here.  At d = 512, where two groups would be left, it is the faster one, 33 against 35 us a
// decode call, and so is the row-wide merge where it serves: 1280 rows of 32 heads and 8 partials 13
// against 26 us.)  Rows without partials are zero.
template <int D>
__global__ void __launch_bounds__(256) merge_spans_kernel(MergeLaunch a) {
  constexpr int D4 = D / 4, G = 256 / D4;
  __shared__ float sm[G], sl[G];
  __shared__ float4 sacc[G][D4];
  const MergeItem it = a.items[blockIdx.x];
  const int h = blockIdx.y;
  const int g = threadIdx.x / D4, c = threadIdx.x % D4;
  float4 *out = reinterpret_cast<float4 *>(a.out + ((size_t)it.qrow * a.hq + h) * D);
  float M = -INFINITY, L = 0.0f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = g; p0 < it.nparts; p0 += 4 * G) {
    float pm[4], pl[4];
    float4 x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int p = p0 + G * u;
      const bool ok = p < it.nparts;
      const size_t pi = (size_t)(it.first + (ok ? p : p0)) * a.hq + h;
      pm[u] = ok ? a.part_m[pi] : -INFINITY;
      pl[u] = ok ? a.part_l[pi] : 0.0f;
      x[u] = ok ? ld4(a.part_acc + pi * D + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float Mn = fmaxf(fmaxf(M, fmaxf(pm[0], pm[1])), fmaxf(pm[2], pm[3]));
    const float Ms = Mn == -INFINITY ? 0.0f : Mn;
    const float alpha = __builtin_amdgcn_exp2f(M - Ms);  // 0 while M is -inf
    L *= alpha;
    A = make_float4(A.x * alpha, A.y * alpha, A.z * alpha, A.w * alpha);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const float e = __builtin_amdgcn_exp2f(pm[u] - Ms);
      L = fmaf(pl[u], e, L);
      A.x = fmaf(x[u].x, e, A.x);
      A.y = fmaf(x[u].y, e, A.y);
      A.z = fmaf(x[u].z, e, A.z);
      A.w = fmaf(x[u].w, e, A.w);
    }
    M = Mn;
  }
  if (c == 0) {
    sm[g] = M;
    sl[g] = L;
  }
  sacc[g][c] = A;
  __syncthreads();
  float T = -INFINITY;
#pragma unroll
  for (int w = 0; w < G; w++) T = fmaxf(T, sm[w]);
  const float Ts = T == -INFINITY ? 0.0f : T;
  float LT = 0.0f;
#pragma unroll
  for (int w = 0; w < G; w++) LT = fmaf(sl[w], __builtin_amdgcn_exp2f(sm[w] - Ts), LT);
  const float inv = LT == 0.0f ? 0.0f : 1.0f / LT;
  for (int cc = threadIdx.x; cc < D4; cc += blockDim.x) {
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < G; w++) {
      const float e = __builtin_amdgcn_exp2f(sm[w] - Ts);
      const float4 x = sacc[w][cc];
      r.x = fmaf(x.x, e, r.x);
      r.y = fmaf(x.y, e, r.y);
      r.z = fmaf(x.z, e, r.z);
      r.w = fmaf(x.w, e, r.w);
    }
    out[cc] = make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv);
  }
}

bool span_kernel_supports(int head_dim, int paged, int block_size) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256 || head_dim == 512) &&
         (!paged || (block_size >= 16 && (block_size & (block_size - 1)) == 0));
}

hipError_t launch_spans(const SpanLaunch &a, int max_cols, hipStream_t s) {
  if (a.num_items <= 0) return hipSuccess;
  switch (a.head_dim * 2 + (max_cols > kSpanCols)) {
    case 64 * 2: launch_span<64, 1>(a, s); break;
    case 64 * 2 + 1: launch_span<64, 2>(a, s); break;
    case 128 * 2: launch_span<128, 1>(a, s); break;
    case 128 * 2 + 1: launch_span<128, 2>(a, s); break;
    case 256 * 2: launch_span<256, 1>(a, s); break;
    case 512 * 2: launch_span<512, 1>(a, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_merge_spans(const MergeLaunch &a, hipStream_t s) {
  if (a.num_items <= 0) return hipSuccess;
  const dim3 grid(a.num_items, a.hq);
  switch (a.head_dim) {
    case 64: hipLaunchKernelGGL(merge_spans_kernel<64>, grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL(merge_spans_kernel<128>, grid, dim3(256), 0, s, a); break;
    case 256: hipLaunchKernelGGL(merge_spans_kernel<256>, grid, dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace nva
