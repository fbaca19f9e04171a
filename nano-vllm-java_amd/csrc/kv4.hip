// Attention over the 4-bit arena (nva_attention4_forward): rounding rows into their slots, the work list,
// attention and the merge of split rows.
//
// Layout.  A layer is [block][KV head][tile of 32 keys][34 d bytes], a tile's bytes being
//   K codes   [key 32][d / 2]            dim 2j in the low bits of byte j
//   V codes   [quarter 4][row 16][slot 8][d / 32]
//   K scales  [key % 16][d / 32][key / 16]
//   V scales  [quarter 4][d / 32][slot 8]
// where slot s of quarter w is key 16 (s / 4) + 4 w + s % 4, and row r holds dims r d / 16 and on.  Lane
// l = 16 w + r of a wave thus reads its part of either product in one run of bytes, which neighbouring lanes
// continue, and a token's codes stay apart from its neighbours' (4-byte words at d = 128), so that tokens
// are stored independently.
//
// Products on the matrix cores (16 x 16 x 32 bf16): S^T = K Q^T with keys as rows and columns (query row,
// head of the KV head) as columns, then O^T += V^T P^T with dims as rows.  The order of the contraction is
// free, so that of the dims follows K's bytes (lane quarter w takes dims w d / 4 and on: its scale is its
// own), and that of the keys the accumulators of S^T: lane 16 w + c holds keys 4 w .. 4 w + 3 of both
// 16-key halves for column c, which is what the second product wants of P^T, given V's slots above.  No
// value crosses lanes but the column maxima.  The 4-bit values are exact in bf16; q and p go in as three
// bf16 parts whose sum they are (split3), so the products are those of fp32.
#include "mx4.h"
#include "nva_internal.h"
#include "row_lanes.h"

namespace nva {

namespace {

constexpr int kWaves = 4;
constexpr int kCols = kKv4Cols;

__device__ __forceinline__ size_t tile_at(const Kv4View &kv, int block, int head, int tile, int d) {
  return (((size_t)block * kv.hkv + head) * (kv.block_size >> 5) + tile) * (size_t)(34 * d);
}

// Where 8 dims (the i-th 8) of key `key` of a tile lie.
struct RowPlace {
  int k, v, ks, vs;  // byte offsets in the tile; v for d >= 128
};
__device__ __forceinline__ RowPlace row_place(int d, int key, int i) {
  const int nb = d >> 5, w = (key & 15) >> 2, slot = ((key >> 4) << 2) | (key & 3);
  RowPlace p;
  p.k = key * (d >> 1) + 4 * i;
  const int per = d >> 4, r = (8 * i) / per, within = (8 * i - r * per) >> 1;
  p.v = 16 * d + ((w * 16 + r) * 8 + slot) * nb + within;
  p.ks = 32 * d + ((key & 15) * nb + (i >> 2)) * 2 + (key >> 4);
  p.vs = 33 * d + (w * nb + (i >> 2)) * 8 + slot;
  return p;
}

// ---------------------------------------------------------------- rows in and out

// Rounds one row (8 dims a lane, D / 8 lanes) into its slot.
template <int D>
__device__ __forceinline__ void store_row(const Kv4View &kv, const float *src, int slot, int head,
                                          bool is_v, int i) {
  float x[8];
  *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(src + 8 * i);
  *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(src + 8 * i + 4);
  const uint32_t scale = mx4_scale(max_quad(mx4_top8(x)));
  const uint32_t word = mx4_codes8(x, scale);
  if (slot < 0 || slot >= kv.num_blocks * (int64_t)kv.block_size) return;
  const int block = slot / kv.block_size, in = slot - block * kv.block_size;
  uint8_t *tile = kv.pages + tile_at(kv, block, head, in >> 5, D);
  const RowPlace p = row_place(D, in & 31, i);
  if (!is_v) {
    *reinterpret_cast<uint32_t *>(tile + p.k) = word;
  } else if constexpr (D == 64) {  // two rows of 4 dims
    *reinterpret_cast<uint16_t *>(tile + p.v) = (uint16_t)word;
    *reinterpret_cast<uint16_t *>(tile + p.v + 16) = (uint16_t)(word >> 16);
  } else {
    *reinterpret_cast<uint32_t *>(tile + p.v) = word;
  }
  if ((i & 3) == 0) tile[is_v ? p.vs : p.ks] = (uint8_t)scale;
}

}  // namespace

// ---------------------------------------------------------------- the work list

// Column tiles: runs of kCols columns of one sequence, column c being query row c / rep and head c % rep
// of each KV head, over the 32-key tiles [kb, kb + n) that any of their rows sees.  Units are key tiles,
// numbered by column tile, KV head and tile; workgroup g of the attention takes units [g C, (g + 1) C), so
// every workgroup does the same work however lengths differ.  cum[t] is the units of one KV head before
// tile t.  The list is built from the lengths on the device, which a captured step's replays find there.
__device__ void build_list(const Kv4List &a) {
  __shared__ int64_t part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto scan = [&](int64_t v, int64_t &total) {  // exclusive, over the workgroup
    int64_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up((long long)x, d);
      if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < 4; w++) {
      if (w < wave) before += part[w];
      total += part[w];
    }
    return before + x - v;
  };
  const int rep = a.rep;
  // Column tiles before each sequence.
  int64_t tiles = 0;
  for (int b0 = 0; b0 < a.num_seqs; b0 += 256) {
    const int b = b0 + tid;
    int64_t mine = 0, all;
    if (b < a.num_seqs) {
      const int qlen = a.cu_q ? a.cu_q[b + 1] - a.cu_q[b] : 1;
      mine = ((int64_t)qlen * rep + kCols - 1) / kCols;
    }
    const int64_t at = tiles + scan(mine, all);
    if (b < a.num_seqs) a.before[b] = (int32_t)at;
    tiles += all;
  }
  if (tid == 0) a.before[a.num_seqs] = (int32_t)tiles;
  __threadfence_block();
  __syncthreads();
  // Their key tiles.
  int64_t units = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += 256) {
    const int t = (int)t0 + tid;
    Kv4Tile tile{0, 0, 0, 0};
    if (t < tiles) {
      int lo = 0, hi = a.num_seqs;  // before[lo] <= t < before[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.before[mid] <= t) lo = mid; else hi = mid;
      }
      const int row = a.cu_q ? a.cu_q[lo] : lo;
      const int qlen = a.cu_q ? a.cu_q[lo + 1] - row : 1;
      const int klen = a.lens ? a.lens[lo] : a.cu_k[lo + 1] - a.cu_k[lo];
      const int64_t col0 = (int64_t)(t - a.before[lo]) * kCols;
      const int first = (int)(col0 / rep);
      const int last = (int)min((int64_t)qlen - 1, (col0 + kCols - 1) / rep);
      const int end = min(klen, klen - qlen + last + 1);
      const int64_t beg = a.window > 0 ? (int64_t)klen - qlen + first + 1 - a.window : 0;
      tile.seq = lo;
      tile.col0 = (int)col0;
      tile.kb = beg > 0 ? (int)(beg >> 5) : 0;
      tile.n = end > max(beg, (int64_t)0) ? ((end + 31) >> 5) - tile.kb : 0;
    }
    int64_t all;
    const int64_t u = units + scan(tile.n, all);
    if (t < tiles) {
      a.tiles[t] = tile;
      a.cum[t] = u;
    }
    units += all;
  }
  if (tid == 0) {
    a.cum[tiles] = units;
    a.head->tiles = (int)tiles;
    // At least kKv4MinUnits a workgroup: fewer would be spent on joining their results.
    const int64_t all = units * a.hkv;
    const int64_t c = (all + a.workgroups - 1) / a.workgroups;
    a.head->chunk = max((c + kWaves - 1) / kWaves * kWaves, (int64_t)kKv4MinUnits);
    a.head->covered = a.cu_q ? a.cu_q[a.num_seqs] : a.num_seqs;
    a.head->first = a.cu_q ? a.cu_q[0] : 0;
  }
}

// Stores the step's rows and builds its list: workgroup 0 the list, the others 256 / (D / 8) rows of K or
// V each.
template <int D>
__global__ void __launch_bounds__(256) kv4_store_kernel(Kv4Store a) {
  if (blockIdx.x == 0) {
    if (a.list.head) build_list(a.list);
    return;
  }
  constexpr int LPR = D / 8, ROWS = 256 / LPR;
  const int64_t row = (int64_t)(blockIdx.x - 1) * ROWS + threadIdx.x / LPR;
  const int64_t half = (int64_t)a.tokens * a.kv.hkv;
  if (row >= 2 * half) return;  // (whole quads)
  const bool is_v = row >= half;
  const int64_t r = is_v ? row - half : row;
  const int t = (int)(r / a.kv.hkv), h = (int)(r - (int64_t)t * a.kv.hkv);
  store_row<D>(a.kv, (is_v ? a.v : a.k) + r * D, a.slots[t], h, is_v, threadIdx.x % LPR);
}

// The values of rows at slots.
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4View kv, const int32_t *slots, float *k,
                                                       float *v, int rows) {
  constexpr int LPR = D / 8, ROWS = 256 / LPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  const int64_t half = (int64_t)rows * kv.hkv;
  if (row >= 2 * half) return;
  const bool is_v = row >= half;
  float *out = is_v ? v : k;
  if (!out) return;
  const int64_t r = is_v ? row - half : row;
  const int t = (int)(r / kv.hkv), h = (int)(r - (int64_t)t * kv.hkv), i = threadIdx.x % LPR;
  const int slot = slots[t];
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < kv.num_blocks * (int64_t)kv.block_size) {
    const int block = slot / kv.block_size, in = slot - block * kv.block_size;
    const uint8_t *tile = kv.pages + tile_at(kv, block, h, in >> 5, D);
    const RowPlace p = row_place(D, in & 31, i);
    uint32_t word;
    if (!is_v)
      word = *reinterpret_cast<const uint32_t *>(tile + p.k);
    else if constexpr (D == 64)
      word = *reinterpret_cast<const uint16_t *>(tile + p.v) |
             ((uint32_t)*reinterpret_cast<const uint16_t *>(tile + p.v + 16) << 16);
    else
      word = *reinterpret_cast<const uint32_t *>(tile + p.v);
    mx4_values8(word, mx4_unit(tile[is_v ? p.vs : p.ks]), x);
  }
  float *o = out + r * D + 8 * i;
  *reinterpret_cast<float4 *>(o) = *reinterpret_cast<const float4 *>(x);
  *reinterpret_cast<float4 *>(o + 4) = *reinterpret_cast<const float4 *>(x + 4);
}

// ---------------------------------------------------------------- attention

namespace {

// One lane's part of a tile.
template <int D> struct Tile {
  uint32_t k[2][D / 32];
  uint32_t v[D / 16];
  uint32_t ks[D == 512 ? 2 : 1];
  u32x2 vs;
};

template <int N> __device__ __forceinline__ void load_words(const uint8_t *p, uint32_t *w) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
    }
  } else {
    static_assert(N == 2, "8 bytes");
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p));
    w[0] = x.x, w[1] = x.y;
  }
}

template <int D>
__device__ __forceinline__ void load_tile(const uint8_t *tile, int lane, Tile<D> &t) {
  constexpr int NB = D / 32;
  const int c = lane & 15, w = lane >> 4;
  load_words<D / 32>(tile + c * (D / 2) + w * (D / 8), t.k[0]);
  load_words<D / 32>(tile + (16 + c) * (D / 2) + w * (D / 8), t.k[1]);
  load_words<D / 16>(tile + 16 * D + lane * (D / 4), t.v);
  const uint8_t *ks = tile + 32 * D + (c * NB + (w * D) / 128) * 2;
  if constexpr (D == 512) {
    load_words<2>(ks, t.ks);
  } else if constexpr (D == 256) {
    t.ks[0] = *reinterpret_cast<const uint32_t *>(ks);
  } else {
    t.ks[0] = *reinterpret_cast<const uint16_t *>(ks);
  }
  t.vs = *reinterpret_cast<const u32x2 *>(tile + 33 * D + (w * NB + (c * D) / 512) * 8);
}

__device__ __forceinline__ uint32_t byte_of(uint32_t word, int i) { return (word >> (8 * i)) & 255u; }

template <int D> __device__ __forceinline__ float k_unit(const Tile<D> &t, int j, int half) {
  const int i = (j / 4) * 2 + half;
  return mx4_unit(byte_of(t.ks[i / 4], i % 4));
}

// Low halves, and high halves, of two words: neighbouring slots of one dim out of two dims of each slot.
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

__device__ __forceinline__ bf16x8 frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const u32x4 w = {a, b, c, d};
  return __builtin_bit_cast(bf16x8, w);
}

// Byte b of every slot: the dims 2 b and 2 b + 1 of the lane's row, over its 8 slots.
template <int D, int B>
__device__ __forceinline__ void v_frags(const Tile<D> &t, const float *unit, bf16x8 &even, bf16x8 &odd) {
  uint32_t p[8];
#pragma unroll
  for (int s = 0; s < 8; s++) {
    constexpr int NB = D / 32;
    const int at = s * NB + B;
    switch (at & 3) {
      case 0: p[s] = mx4_pair<0>(t.v[at >> 2], unit[s]); break;
      case 1: p[s] = mx4_pair<1>(t.v[at >> 2], unit[s]); break;
      case 2: p[s] = mx4_pair<2>(t.v[at >> 2], unit[s]); break;
      default: p[s] = mx4_pair<3>(t.v[at >> 2], unit[s]); break;
    }
  }
  even = frag(low_halves(p[0], p[1]), low_halves(p[2], p[3]), low_halves(p[4], p[5]),
              low_halves(p[6], p[7]));
  odd = frag(high_halves(p[0], p[1]), high_halves(p[2], p[3]), high_halves(p[4], p[5]),
             high_halves(p[6], p[7]));
}

template <int D, int B = 0>
__device__ __forceinline__ void add_values(const Tile<D> &t, const float *unit, const bf16x8 *p,
                                           f32x4 *o) {
  if constexpr (B < D / 32) {
    bf16x8 even, odd;
    v_frags<D, B>(t, unit, even, odd);
#pragma unroll
    for (int i = 0; i < 3; i++) {
      o[2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, p[i], o[2 * B], 0, 0, 0);
      o[2 * B + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, p[i], o[2 * B + 1], 0, 0, 0);
    }
    add_values<D, B + 1>(t, unit, p, o);
  }
}

// The 64-ary search for the last entry of cum that u reaches (times hkv), by a wave: tile of unit u.
__device__ __forceinline__ int find_tile(const int64_t *cum, int n, int64_t u, int hkv, int lane) {
  int lo = 0, hi = n;  // cum[lo] * hkv <= u < cum[hi] * hkv
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6;
    const int at = lo + lane * step;
    const uint64_t le = __ballot(at < hi && cum[min(at, hi - 1)] * hkv <= u);
    const int i = 63 - __builtin_clzll(le);  // lane 0 always holds
    lo += i * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

}  // namespace

// Workgroup g: its units' segments, each of one column tile and KV head.  The four waves take a segment's
// key tiles in turn, each with the running maximum and sum of a softmax, and join through LDS.  A segment
// that covers its keys is written out; others leave partials (slot 2 g for the workgroup's first, of keys
// another one began, 2 g + 1 for its last), which kv4_merge_kernel joins.
template <int D>
__global__ void __launch_bounds__(256, kv4_workgroups_per_cu(D)) kv4_attention_kernel(Kv4Attention a) {
  constexpr bool QLDS = D == 512;  // 192 registers of q's parts would leave none for the loads
  constexpr int NC = D / 32;       // contraction steps of a score
  extern __shared__ float4 smem[];
  float *lds_o = reinterpret_cast<float *>(smem);        // [wave][col][D + 4]
  float *lds_m = lds_o + kWaves * kCols * (D + 4), *lds_l = lds_m + kWaves * kCols;
  bf16x8 *lds_q = reinterpret_cast<bf16x8 *>(smem);      // (QLDS) [part][step][lane], before lds_o
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, w = lane >> 4;
  const int n_tiles = a.head->tiles;
  const int64_t chunk = a.head->chunk;
  const int64_t all = a.cum[n_tiles] * a.kv.hkv;
  int64_t u = (int64_t)blockIdx.x * chunk;
  const int64_t u_end = min(u + chunk, all);
  if (u >= u_end) return;
  const int rep = a.hq / a.kv.hkv;
  const int per_block = a.kv.block_size >> 5;
  int ct = find_tile(a.cum, n_tiles, u, a.kv.hkv, lane);
  while (u < u_end) {
    while (a.tiles[ct].n == 0 || u >= a.cum[ct + 1] * a.kv.hkv) ct++;  // (u is below the last entry's)
    const Kv4Tile tile = a.tiles[ct];
    const int64_t in = u - a.cum[ct] * a.kv.hkv;
    const int head = (int)(in / tile.n);
    const int t0 = (int)(in - (int64_t)head * tile.n);
    const int t1 = (int)min((int64_t)tile.n, t0 + (u_end - u));
    // The lane's column: its query row and head, and the keys [lo, hi) that it sees.
    const int seq = tile.seq;
    const int row0 = a.cu_q ? a.cu_q[seq] : seq;
    const int qlen = a.cu_q ? a.cu_q[seq + 1] - row0 : 1;
    const int klen = a.lens ? a.lens[seq] : a.cu_k[seq + 1] - a.cu_k[seq];
    const int64_t cols = (int64_t)qlen * rep;
    const int64_t col = min((int64_t)tile.col0 + c, cols - 1);  // (columns past the last repeat it)
    const int qrow = (int)(col / rep);
    const int hi = klen - qlen + qrow + 1;
    const int lo = a.window > 0 ? max(0, hi - a.window) : 0;
    const float *qp = a.q + ((size_t)(row0 + qrow) * a.hq + (size_t)head * rep + (col - (int64_t)qrow * rep)) * D;
    bf16x8 q[QLDS ? 1 : NC][3];
    if constexpr (QLDS) {
      __syncthreads();  // the last segment's results have been read
      for (int j = wave; j < NC; j += kWaves) {
        bf16x8 p[3];
        float x[8];
        *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(qp + w * (D / 4) + 8 * j);
        *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(qp + w * (D / 4) + 8 * j + 4);
        split3<false>(x, p);
        for (int i = 0; i < 3; i++) lds_q[(i * NC + j) * 64 + lane] = p[i];
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float x[8];
        *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(qp + w * (D / 4) + 8 * j);
        *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(qp + w * (D / 4) + 8 * j + 4);
        split3<false>(x, q[j]);
      }
    }
    // Tiles that every column sees whole need no mask.
    int all_hi = hi, all_lo = lo;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      all_hi = min(all_hi, __shfl_xor(all_hi, d));
      all_lo = max(all_lo, __shfl_xor(all_lo, d));
    }
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);

    f32x4 o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int32_t *table = a.table + (size_t)seq * a.bt_stride;
    auto address = [&](int t) {  // of key tile t
      const int kt = tile.kb + t;
      const int bi = a.tile_shift >= 0 ? kt >> a.tile_shift : kt / per_block;
      const int block = __builtin_amdgcn_readfirstlane(table[bi]);
      return a.kv.pages + tile_at(a.kv, block, head, kt - bi * per_block, D);
    };
    constexpr bool AHEAD = D < 512;  // the next tile's loads before this one's products
    Tile<D> cur, next;
    int t = t0 + wave;
    if (AHEAD && t < t1) load_tile<D>(address(t), lane, cur);
    for (; t < t1; t += kWaves) {
      if (!AHEAD) load_tile<D>(address(t), lane, cur);
      if (AHEAD && t + kWaves < t1) load_tile<D>(address(t + kWaves), lane, next);
      // Scores of the 32 keys.
      f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const bf16x8 k0 = mx4_frag(cur.k[0][j], k_unit<D>(cur, j, 0));
        const bf16x8 k1 = mx4_frag(cur.k[1][j], k_unit<D>(cur, j, 1));
#pragma unroll
        for (int i = 0; i < 3; i++) {
          bf16x8 qv;
          if constexpr (QLDS) qv = lds_q[(i * NC + j) * 64 + lane]; else qv = q[j][i];
          s[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qv, s[0], 0, 0, 0);
          s[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qv, s[1], 0, 0, 0);
        }
      }
      const int key0 = (tile.kb + t) * 32;
      const bool edge = key0 + 32 > all_hi || key0 < all_lo;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = s[i >> 2][i & 3] * a.scale2;
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int key = key0 + 16 * (i >> 2) + 4 * w + (i & 3);
          if (key >= hi || key < lo) x[i] = -INFINITY;
        }
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                        fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      top = max4_lanes(top);
      if (__any(top > m)) {
        const float grown = fmaxf(m, top);
        const float f = m == grown ? 1.f : __builtin_amdgcn_exp2f(m - grown);  // 0 from -infinity
        m = grown;
        l *= f;
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] *= f;
      }
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - base);
        l += x[i];
      }
      bf16x8 p[3];
      split3<true>(x, p);
      float unit[8];
#pragma unroll
      for (int i = 0; i < 8; i++) unit[i] = mx4_unit(byte_of(cur.vs[i >> 2], i & 3));
      if (edge) {
        // A block that is NaN reaches only the columns that see its key, though all of a wave's columns are
        // multiplied with it: its values are taken as 0 here, and NaN added where a column sees one.
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; i++) bad |= byte_of(cur.vs[i >> 2], i & 3) == 255u;
        if (__any(bad)) {
          uint32_t mark[8], see[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const bool nan = byte_of(cur.vs[i >> 2], i & 3) == 255u;
            const int key = key0 + 16 * (i >> 2) + 4 * w + (i & 3);
            mark[i] = nan ? 0x3f80u : 0u;  // 1 in bf16
            see[i] = key < hi && key >= lo ? 0x3f80u : 0u;
            if (nan) {
              unit[i] = 0.f;
              constexpr int NB = D / 32;  // the slot's codes to 0
#pragma unroll
              for (int b = 0; b < NB; b++) cur.v[(i * NB + b) >> 2] &= ~(255u << (8 * ((i * NB + b) & 3)));
            }
          }
          f32x4 n = {0.f, 0.f, 0.f, 0.f};
          n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              frag(low_halves(mark[0], mark[1]), low_halves(mark[2], mark[3]),
                   low_halves(mark[4], mark[5]), low_halves(mark[6], mark[7])),
              frag(low_halves(see[0], see[1]), low_halves(see[2], see[3]), low_halves(see[4], see[5]),
                   low_halves(see[6], see[7])),
              n, 0, 0, 0);
          // (A row's dims share one block, d / 16 of 32.)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (n[r] > 0.f)
#pragma unroll
              for (int i = 0; i < D / 16; i++) o[i][r] = NAN;
        }
      }
      add_values<D>(cur, unit, p, o);
      if (AHEAD) cur = next;
    }

    // Join the waves: column maxima, then sums and rows over the common maximum.
    l = sum4_lanes(l);
    if constexpr (QLDS) __syncthreads();  // q's parts have been read
    if (w == 0) {
      lds_m[wave * kCols + c] = m;
      lds_l[wave * kCols + c] = l;
    }
    float *mine = lds_o + (wave * kCols + c) * (D + 4);
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int i = 0; i < D / 16; i += 4)
        *reinterpret_cast<float4 *>(mine + (4 * w + r) * (D / 16) + i) =
            make_float4(o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]);
    __syncthreads();
    const int oc = threadIdx.x >> 4, part16 = threadIdx.x & 15;  // column, 16 lanes each
    float ms[kWaves], big = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      ms[i] = lds_m[i * kCols + oc];
      big = fmaxf(big, ms[i]);
    }
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const float li = lds_l[i * kCols + oc];
      // (No maximum: no keys, or scores that are NaN, which the sum holds.)
      ms[i] = ms[i] == -INFINITY ? (li == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(ms[i] - big);
      sum += ms[i] * li;
    }
    const bool whole = t0 == 0 && t1 == tile.n;
    const int64_t ocol = (int64_t)tile.col0 + oc;
    if (ocol < cols) {
      const int orow = (int)(ocol / rep);
      const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
      const size_t part = (size_t)(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * kCols + oc;
      float *dst = whole ? a.out + ((size_t)(row0 + orow) * a.hq + (size_t)head * rep +
                                    (ocol - (int64_t)orow * rep)) * D
                         : a.part_o + part * D;
#pragma unroll
      for (int i = 0; i < D / 64; i++) {
        const int e = 4 * (part16 + 16 * i);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < kWaves; v++)
          if (ms[v] != 0.f)  // (a wave without keys has nothing)
            acc += ms[v] * *reinterpret_cast<const f32x4 *>(lds_o + (v * kCols + oc) * (D + 4) + e);
        acc *= inv;
        *reinterpret_cast<f32x4 *>(dst + e) = acc;
      }
      if (!whole && part16 == 0) {
        a.part_m[part] = big;
        a.part_l[part] = sum;
      }
    }
    if constexpr (!QLDS) __syncthreads();  // lds_o is written again
    u += t1 - t0;
  }
}

// Joins the partials of column tiles that several workgroups shared, and zero-fills rows without keys:
// workgroup (column tile x KV head, four columns) or, behind them, rows that no sequence covers.
__global__ void __launch_bounds__(256) kv4_merge_kernel(Kv4Attention a) {
  const int n_tiles = a.head->tiles, D = a.head_dim, rep = a.hq / a.kv.hkv;
  const int64_t chunk = a.head->chunk;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int64_t item = blockIdx.x; item < (int64_t)n_tiles * a.kv.hkv; item += gridDim.x) {
    const int ct = (int)(item / a.kv.hkv), head = (int)(item - (int64_t)ct * a.kv.hkv);
    const Kv4Tile tile = a.tiles[ct];
    const int64_t u0 = a.cum[ct] * a.kv.hkv + (int64_t)head * tile.n;
    const int64_t g0 = u0 / chunk, g1 = tile.n ? (u0 + tile.n - 1) / chunk : g0;
    if (tile.n && g0 == g1) continue;
    const int row0 = a.cu_q ? a.cu_q[tile.seq] : tile.seq;
    const int qlen = a.cu_q ? a.cu_q[tile.seq + 1] - row0 : 1;
    const int64_t cols = (int64_t)qlen * rep;
    for (int c = wave + 4 * blockIdx.y; c < kCols; c += 4 * gridDim.y) {
      const int64_t col = (int64_t)tile.col0 + c;
      if (col >= cols) continue;
      const int row = (int)(col / rep);
      float *dst = a.out + ((size_t)(row0 + row) * a.hq + (size_t)head * rep + (col - (int64_t)row * rep)) * D;
      if (tile.n == 0) {
        for (int e = lane; e < D; e += 64) dst[e] = 0.f;
        continue;
      }
      // Partial of workgroup g: its last for the first one, its first for the others.
      auto slot = [&](int64_t g) { return (size_t)(2 * g + (g == g0 ? 1 : 0)) * kCols + c; };
      float big = -INFINITY;
      for (int64_t g = g0 + lane; g <= g1; g += 64) big = fmaxf(big, a.part_m[slot(g)]);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) big = fmaxf(big, __shfl_xor(big, d));
      float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int64_t g = g0; g <= g1; g++) {
        const float m = a.part_m[slot(g)], l = a.part_l[slot(g)];
        if (m == -INFINITY && l == 0.f) continue;  // no keys (a sum that is NaN stays)
        const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - big);
        sum += f * l;
        const float *src = a.part_o + slot(g) * D;
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (lane + 64 * i < D) acc[i] += f * src[lane + 64 * i];
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (lane + 64 * i < D) dst[lane + 64 * i] = acc[i] * inv;
    }
  }
  // Rows before the first sequence and behind the last one.
  if (blockIdx.y == 0) {
    const int first = a.head->first, covered = a.head->covered;
    const size_t width = (size_t)a.hq * D;
    const size_t rows = (size_t)first + (a.tokens - covered), n = rows * width;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
      const size_t r = i / width;
      a.out[(r < (size_t)first ? r : r - first + covered) * width + (i - r * width)] = 0.f;
    }
  }
}

// ---------------------------------------------------------------- quantize

__global__ void __launch_bounds__(256) quantize4_kernel(const float *x, int64_t words, uint32_t *codes,
                                                        uint8_t *scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // 8 values each; whole quads
  if (i >= words) return;
  float v[8];
  *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x + 8 * i);
  *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(x + 8 * i + 4);
  const uint32_t scale = mx4_scale(max_quad(mx4_top8(v)));
  codes[i] = mx4_codes8(v, scale);
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)scale;
}

hipError_t launch_quantize4(const float *x, int64_t values, uint8_t *codes, uint8_t *scales,
                            hipStream_t s) {
  const int64_t words = values / 8;
  for (int64_t at = 0; at < words;) {  // grids of at most 2^22 workgroups
    const int64_t n = std::min<int64_t>(words - at, (int64_t)256 << 22);
    hipLaunchKernelGGL(quantize4_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, x + 8 * at,
                       n, reinterpret_cast<uint32_t *>(codes) + at, scales + at / 4);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    at += n;
  }
  return hipSuccess;
}

// ---------------------------------------------------------------- launchers

bool kv4_supports(int head_dim) {
  return head_dim == 64 || head_dim == 128 || head_dim == 256 || head_dim == 512;
}

namespace {

template <int D> size_t attention_lds() {
  const size_t join = (size_t)kWaves * kCols * (D + 4 + 2) * 4;
  return D == 512 ? std::max<size_t>(join, (size_t)3 * (D / 32) * 64 * 16) : join;
}

template <int D> hipError_t store(const Kv4Store &a, hipStream_t s) {
  constexpr int ROWS = 256 / (D / 8);
  const int64_t rows = a.k ? 2 * (int64_t)a.tokens * a.kv.hkv : 0;
  const int64_t blocks = (rows + ROWS - 1) / ROWS;
  hipLaunchKernelGGL(kv4_store_kernel<D>, dim3((unsigned)(blocks + 1)), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int D>
hipError_t read(const Kv4View &kv, const int32_t *slots, float *k, float *v, int rows, hipStream_t s) {
  constexpr int ROWS = 256 / (D / 8);
  const int64_t blocks = (2 * (int64_t)rows * kv.hkv + ROWS - 1) / ROWS;
  hipLaunchKernelGGL(kv4_read_kernel<D>, dim3((unsigned)blocks), dim3(256), 0, s, kv, slots, k, v, rows);
  return hipGetLastError();
}

template <int D> hipError_t attention(const Kv4Attention &a, int workgroups, hipStream_t s) {
  const size_t lds = attention_lds<D>();
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&kv4_attention_kernel<D>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kv4_attention_kernel<D>, dim3(workgroups), dim3(256), lds, s, a);
  return hipGetLastError();
}

}  // namespace

#define NVA_BY_DIM(d, call)            \
  switch (d) {                         \
    case 64: return call<64> args;     \
    case 128: return call<128> args;   \
    case 256: return call<256> args;   \
    case 512: return call<512> args;   \
    default: return hipErrorInvalidValue; \
  }

hipError_t launch_kv4_store(const Kv4Store &a, int head_dim, hipStream_t s) {
#define args (a, s)
  NVA_BY_DIM(head_dim, store)
#undef args
}

hipError_t launch_kv4_read(const Kv4View &kv, int head_dim, const int32_t *slots, float *k, float *v,
                           int rows, hipStream_t s) {
  if (rows <= 0) return hipSuccess;
#define args (kv, slots, k, v, rows, s)
  NVA_BY_DIM(head_dim, read)
#undef args
}

hipError_t launch_kv4_attention(const Kv4Attention &a, int workgroups, hipStream_t s) {
#define args (a, workgroups, s)
  NVA_BY_DIM(a.head_dim, attention)
#undef args
}

hipError_t launch_kv4_merge(const Kv4Attention &a, int max_tiles, hipStream_t s) {
  const int64_t items = (int64_t)max_tiles * a.kv.hkv;
  hipLaunchKernelGGL(kv4_merge_kernel, dim3((unsigned)std::min<int64_t>(std::max<int64_t>(items, 1), 4096), 4),
                     dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace nva
