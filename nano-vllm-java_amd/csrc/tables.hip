// Block tables, slots and positions of a step from how many tokens of each sequence stay and how many
// follow (nva_step_extend).
//
// Row b holds have = ceil(len / bs) blocks, keeps stay = ceil(keep / bs) of them and wants want =
// ceil((keep + new) / bs).  Three exclusive prefix sums over the rows, of new, have - stay and
// want - stay, give every token, returned block and taken block its place: returned block e (in
// ascending order of row and column) goes to stack entry top + returned - 1 - e, and taken block e comes
// from entry top + returned - 1 - e of the stack as it is then.  So the order of threads decides
// nothing, and taking is the inverse of returning.
//
// What bounds it is latency: a decode step of 256 rows moves some 10 KB and takes 6.2 us (an empty launch
// 2.2).  One workgroup does all of a small step, as a second launch would cost more than the work; steps of
// more than kFillApart tokens write their slots and positions from a launch of many workgroups (61 prompts
// of 25 thousand tokens: 6.9 and 3.2 us).
#include "nva_internal.h"
#include "row_lanes.h"

namespace nva {

namespace {

constexpr int kThreads = 1024;
constexpr int kFillApart = 4096;

// The largest b with cu[b] <= e, for an e below cu[n]: the row (not an empty one) that e falls to.
__device__ __forceinline__ int row_of(const int32_t *cu, int n, int e) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= e) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int blocks_of(int64_t tokens, int bs) { return (int)((tokens + bs - 1) / bs); }

__device__ __forceinline__ void fill_token(const TablesLaunch &a, const int32_t *cu, int total, int t,
                                           const int32_t *keep) {
  int slot = -1, pos = 0;
  if (t < total) {
    const int b = row_of(cu, a.num_seqs, t);
    pos = keep[b] + (t - cu[b]);
    slot = a.table[(size_t)b * a.width + pos / a.block_size] * a.block_size + pos % a.block_size;
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

}  // namespace

__global__ void __launch_bounds__(kThreads) tables_extend_kernel(TablesLaunch a) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t wave_sum[3][kThreads / 64];
  __shared__ int32_t s_bad;
  const int n = a.num_seqs, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t *cu_t = lds, *cu_r = cu_t + n + 1, *cu_w = cu_r + n + 1, *kept = cu_w + n + 1;
  if (tid == 0) s_bad = INT32_MAX;
  __syncthreads();
  int64_t base[3] = {0, 0, 0};
  for (int b0 = 0; b0 < n; b0 += kThreads) {
    const int b = b0 + tid;
    int64_t v[3] = {0, 0, 0};
    if (b < n) {
      const int64_t len = a.lens[b], keep = a.keep ? a.keep[b] : len, fresh = a.fresh[b];
      if (keep < 0 || keep > len || fresh < 0 || fresh > a.max_new || keep + fresh > a.max_tokens) {
        atomicMin(&s_bad, b);  // (the order of rows does not matter to a minimum)
      } else {
        const int stay = blocks_of(keep, a.block_size);
        v[0] = fresh;
        v[1] = blocks_of(len, a.block_size) - stay;
        v[2] = blocks_of(keep + fresh, a.block_size) - stay;
      }
      kept[b] = (int32_t)keep;
    }
    const int64_t x[3] = {scan_wave(v[0]), scan_wave(v[1]), scan_wave(v[2])};
    if (lane == 63)
      for (int i = 0; i < 3; i++) wave_sum[i][wave] = x[i];
    __syncthreads();
    int64_t all[3];
    for (int i = 0; i < 3; i++) {
      int64_t before = base[i];
      all[i] = base[i];
      for (int w = 0; w < kThreads / 64; w++) {
        if (w < wave) before += wave_sum[i][w];
        all[i] += wave_sum[i][w];
      }
      // (Sums that pass 32 bits are refused below, before anything reads the entries.)
      if (b < n) lds[i * (n + 1) + b] = (int32_t)(before + x[i] - v[i]);
    }
    for (int i = 0; i < 3; i++) base[i] = all[i];
    __syncthreads();  // wave_sum is written again
  }
  const int64_t tokens = base[0], returned = base[1], taken = base[2];
  const int top = a.state[3];
  __syncthreads();  // every thread has read the stack's height and s_bad is settled
  int code = 0, what = 0;
  if (s_bad != INT32_MAX) {
    code = 1;
    what = s_bad;
  } else if (tokens > a.num_tokens) {
    code = 2;
    what = (int)min(tokens, (int64_t)INT32_MAX);
  } else if (taken > top + returned) {
    code = 3;
    what = (int)min(taken, (int64_t)INT32_MAX);
  }
  if (tid == 0) {
    const int left = code ? top : (int)(top + returned - taken);
    a.state[0] = code;
    a.state[1] = what;
    a.state[2] = left;
    a.state[3] = left;
  }
  if (code) {  // nothing is taken: the step has no tokens
    for (int b = tid; b <= n; b += kThreads) a.cu_q[b] = 0;
    if (!a.fill_apart)
      for (int t = tid; t < a.num_tokens; t += kThreads) a.slots[t] = -1, a.positions[t] = 0;
    return;
  }
  if (tid == 0) {
    cu_t[n] = (int32_t)tokens;
    cu_r[n] = (int32_t)returned;
    cu_w[n] = (int32_t)taken;
  }
  __syncthreads();
  const int end = top + (int)returned - 1;
  for (int e = tid; e < (int)returned; e += kThreads) {
    const int b = row_of(cu_r, n, e);
    int32_t *entry = a.table + (size_t)b * a.width + blocks_of(kept[b], a.block_size) + (e - cu_r[b]);
    a.free_pages[end - e] = *entry;
    *entry = -1;
  }
  if (returned) {
    __threadfence_block();
    __syncthreads();
  }
  for (int e = tid; e < (int)taken; e += kThreads) {
    const int b = row_of(cu_w, n, e);
    a.table[(size_t)b * a.width + blocks_of(kept[b], a.block_size) + (e - cu_w[b])] =
        a.free_pages[end - e];
  }
  for (int b = tid; b <= n; b += kThreads) {
    a.cu_q[b] = cu_t[b];
    if (b < n) a.lens[b] = kept[b] + cu_t[b + 1] - cu_t[b];
  }
  if (a.fill_apart) return;
  __threadfence_block();
  __syncthreads();
  for (int t = tid; t < a.num_tokens; t += kThreads) fill_token(a, cu_t, (int)tokens, t, kept);
}

// Slots and positions of a large step.
__global__ void __launch_bounds__(256) tables_fill_kernel(TablesLaunch a) {
  extern __shared__ int32_t lds[];
  const int n = a.num_seqs;
  int32_t *cu = lds, *kept = lds + n + 1;
  for (int b = threadIdx.x; b <= n; b += 256) cu[b] = a.cu_q[b];
  __syncthreads();
  for (int b = threadIdx.x; b < n; b += 256) kept[b] = a.lens[b] - (cu[b + 1] - cu[b]);
  __syncthreads();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < a.num_tokens) fill_token(a, cu, cu[n], t, kept);
}

// Empty tables and a full stack, whose last entry is handed out first.
__global__ void __launch_bounds__(256) tables_clear_kernel(TablesLaunch a, const int32_t *pages,
                                                           int num_pages, int64_t entries,
                                                           int max_seqs, int max_step_tokens) {
  const int64_t stride = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = i0; i < entries; i += stride) a.table[i] = -1;
  for (int64_t i = i0; i < num_pages; i += stride) {
    const int64_t j = num_pages - 1 - i;
    a.free_pages[i] = pages ? pages[j] : (int32_t)j;
  }
  for (int64_t i = i0; i < max_seqs; i += stride) a.lens[i] = 0;
  for (int64_t i = i0; i <= max_seqs; i += stride) a.cu_q[i] = 0;
  for (int64_t i = i0; i < max_step_tokens; i += stride) a.slots[i] = -1, a.positions[i] = 0;
  if (i0 == 0) {
    a.state[0] = a.state[1] = 0;
    a.state[2] = a.state[3] = num_pages;
  }
}

hipError_t launch_tables_clear(const TablesLaunch &a, const int32_t *pages, int num_pages,
                               int max_seqs, int max_step_tokens, hipStream_t s) {
  hipLaunchKernelGGL(tables_clear_kernel, dim3(256), dim3(256), 0, s, a, pages, num_pages,
                     (int64_t)max_seqs * a.width, max_seqs, max_step_tokens);
  return hipGetLastError();
}

hipError_t launch_tables_extend(const TablesLaunch &in, hipStream_t s) {
  TablesLaunch a = in;
  a.fill_apart = a.num_tokens > kFillApart ? 1 : 0;
  const size_t lds = (size_t)4 * (a.num_seqs + 1) * 4;
  hipLaunchKernelGGL(tables_extend_kernel, dim3(1), dim3(kThreads), lds, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.fill_apart) return e;
  hipLaunchKernelGGL(tables_fill_kernel, dim3((a.num_tokens + 255) / 256), dim3(256),
                     (size_t)2 * (a.num_seqs + 1) * 4, s, a);
  return hipGetLastError();
}

}  // namespace nva
