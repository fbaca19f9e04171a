// Attention over the 4-bit arena (nva_attention4_forward): rounding rows into their slots, the work list,
// attention and the merge of split rows.
//
// Layout.  A layer is [block][KV head][tile of 32 keys][34 d bytes], a tile's bytes being
//   K codes   [key % 2][run 64][d / 8]   run 16 w + c: of keys 2c and 2c + 1 the dims w d / 4 and on
//   V codes   [run 64][key % 8][d / 32]  run 16 w + c: of keys 8w .. 8w + 7 the dims c d / 16 and on
//   K scales  [key / 2][d / 32][key % 2]
//   V scales  [key / 8][d / 32][key % 8]
// a pair of dims a byte, the even one in its low bits.  Run l is what lane l of a wave needs for either
// product; runs of more than 16 bytes are cut into pieces of 16, [piece][run][16], so that each load of a
// wave is 1 KB in a row (with whole runs in a row a load touched every line of the tile, and 128 rows
// of up to 16K keys, d = 256, took 83 us instead of 53, and 8 columns of d = 512 141 instead of 97).  A
// token's codes stay apart from its neighbours' (4-byte words at d = 128), so that tokens are stored
// independently.
//
// Products on the matrix cores (16 x 16 x 32 bf16; operands hold 8 values of the contraction a lane,
// results rows 4 w .. 4 w + 3 of column c).  The order of the contraction is free: that of the dims follows
// K's bytes (lane quarter w takes dims w d / 4 and on, so its scale is its own), that of the keys gives
// quarter w keys 8 w .. 8 w + 7, and the two halves of a tile are its even and its odd keys.
//   Few columns (query rows times heads of a KV head): S = Q K^T with a column's three parts as three
//   rows, 4 h + part, so that lane (w, c) has all parts of column w and keys 2c and 2c + 1: no score is
//   computed twice.  P goes through 1 KB of LDS to be an operand of O = P V, whose rows again are parts.
//   Many: S^T = K Q^T, where lane (w, c) has column c and keys 8 w .. 8 w + 7, which is what O^T = V^T P^T
//   wants of P^T; nothing crosses lanes but the column maxima.
// The 4-bit values are exact in bf16; q and p go in as three bf16 parts whose sum they are (split3), so the
// products are those of fp32.
#include "mx4.h"
#include "nva_internal.h"
#include "row_lanes.h"

namespace nva {

namespace {

constexpr int kWaves = 4;

__device__ __forceinline__ size_t tile_at(const Kv4View &kv, int block, int head, int tile, int d) {
  return (((size_t)block * kv.hkv + head) * (kv.block_size >> 5) + tile) * (size_t)(34 * d);
}

// Where a byte of a lane's run lies among the wave's runs of `run` bytes.
__host__ __device__ constexpr int run_at(int lane, int byte, int run) {
  return run <= 16 ? lane * run + byte : (byte >> 4) * 1024 + lane * 16 + (byte & 15);
}

// Where 8 dims (the i-th 8) of key `key` of a tile lie.
struct RowPlace {
  int k, v, ks, vs;  // byte offsets in the tile; v for d >= 128
};
__device__ __forceinline__ RowPlace row_place(int d, int key, int i) {
  const int nb = d >> 5, w = key >> 3, slot = key & 7;
  RowPlace p;
  const int krun = d >> 3, kw = 4 * i / krun;
  p.k = (key & 1) * 8 * d + run_at(16 * kw + (key >> 1), 4 * i - kw * krun, krun);
  const int per = d >> 4, r = (8 * i) / per, within = (8 * i - r * per) >> 1;
  // (The quarters of the dims apart where waves share them.)
  const int byte = kv4_by_dims(d) ? (within >> 2) * 32 + slot * 4 + (within & 3) : slot * nb + within;
  p.v = 16 * d + run_at(w * 16 + r, byte, d >> 2);
  p.ks = 32 * d + ((key >> 1) * nb + (i >> 2)) * 2 + (key & 1);
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

// Column tiles: runs of a.cols columns of one sequence, column c being query row c / rep and head c % rep
// of each KV head, over the 32-key tiles [kb, kb + n) that any of their rows sees.  Units are key tiles,
// numbered by column tile, KV head and tile; workgroup g of the attention takes units [g C, (g + 1) C), so
// every workgroup does the same work however lengths differ.  cum[t] is the units of one KV head before
// tile t.  The list is built from the lengths on the device, which a captured step's replays find there.
//
// A workgroup's segment (its units of one column tile and KV head) costs some 4 us beside its units: q,
// the first keys and the join of its waves.  So where a few units more, a.slack, let every workgroup have
// one segment, each column tile's units are rounded up to whole chunks: with 96 rows of 1024 keys of one KV
// head, d = 256, the attention takes 17.5 us instead of 22.7, with 5 rows of up to 700 keys 7.5 instead of
// 12.2, with three of 60 to 120 thousand 33.4 instead of 35.6, and the list 1.2 more.  Elsewhere a segment
// counts a.over units more, so that a workgroup of many short ones gets fewer keys (20 more: 128 rows of up
// to 16K keys, four columns of d = 128, 208 -> 194 us, 64 of up to 8K, eight columns, 99 -> 67; 4 for tiles,
// where a unit is more work: 91 prompts of 147 rows of 40 heads 281 -> 260).
constexpr int kListThreads = 256, kListRounds = 4, kListNear = 1025;
static_assert(kListRounds * kListThreads == kKv4ListTiles);

__device__ void build_list(const Kv4List &a) {
  __shared__ int64_t part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto scan = [&](int64_t v, int64_t &total) {  // exclusive, over the workgroup
    const int64_t x = scan_wave(v);
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
  auto rows_of = [&](int b, Kv4Tile &t) {
    t.seq = b;
    t.row0 = a.cu_q ? a.cu_q[b] : b;
    t.qlen = a.cu_q ? a.cu_q[b + 1] - t.row0 : 1;
    t.klen = a.lens ? a.lens[b] : a.cu_k[b + 1] - a.cu_k[b];
  };
  // The key tiles that columns [col0, col0 + a.cols) of a sequence see.
  auto keys_of = [&](int col0, Kv4Tile &t) {  // (a step's rows times heads are below 2^30)
    const int first = col0 / rep;
    const int last = min(t.qlen - 1, (col0 + a.cols - 1) / rep);
    const int end = min(t.klen, t.klen - t.qlen + last + 1);
    const int64_t beg = a.window > 0 ? (int64_t)t.klen - t.qlen + first + 1 - a.window : 0;
    t.col0 = col0;
    t.kb = beg > 0 ? (int)(beg >> 5) : 0;
    t.n = t.qlen > 0 && end > max(beg, (int64_t)0) ? ((end + 31) >> 5) - t.kb : 0;
    t.units = t.n ? t.n + a.over : 0;
  };
  // Column tiles before each sequence, in LDS where they have room there: every column tile is looked up.
  __shared__ int32_t near[kListNear];
  int32_t *before = a.num_seqs < kListNear ? near : a.before;
  int64_t tiles = a.num_seqs;
  if (!a.one_each) {
    tiles = 0;
    for (int b0 = 0; b0 < a.num_seqs; b0 += kListThreads) {
      const int b = b0 + tid;
      int64_t mine = 0, all;
      if (b < a.num_seqs) {
        const int64_t cols = (int64_t)(a.cu_q ? a.cu_q[b + 1] - a.cu_q[b] : 1) * rep;
        if (cols >= a.min_cols && cols <= a.max_cols) mine = (cols + a.cols - 1) / a.cols;
      }
      const int64_t at = tiles + scan(mine, all);
      if (b < a.num_seqs) before[b] = (int32_t)at;
      tiles += all;
    }
    if (tid == 0) before[a.num_seqs] = (int32_t)tiles;
    __threadfence_block();
    __syncthreads();
  }
  // A thread's `per` column tiles from t0 + per * tid on: their sequences first, so that what is read of
  // those is on its way together.
  const int per = (int)min((tiles + kListThreads - 1) / kListThreads, (int64_t)kListRounds);
  auto take = [&](int64_t t0, Kv4Tile *mine) {
    const int64_t at = t0 + per * tid;
    int b[kListRounds];
    if (a.one_each) {  // no sequence has more than one: each gets one, of no keys where it has no rows
#pragma unroll
      for (int i = 0; i < kListRounds; i++) b[i] = (int)at + i;
    } else {
      int lo = 0, hi = a.num_seqs;  // before[lo] <= at < before[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= at) lo = mid; else hi = mid;
      }
#pragma unroll
      for (int i = 0; i < kListRounds; i++) {
        if (i < per && at + i < tiles)
          while (before[lo + 1] <= at + i) lo++;
        b[i] = lo;
      }
    }
#pragma unroll
    for (int i = 0; i < kListRounds; i++) {
      mine[i] = Kv4Tile{};
      if (i < per && at + i < tiles) rows_of(b[i], mine[i]);
    }
#pragma unroll
    for (int i = 0; i < kListRounds; i++)
      if (i < per && at + i < tiles)
        keys_of(a.one_each ? 0 : ((int)at + i - before[b[i]]) * a.cols, mine[i]);
  };
  int64_t units = 0, chunk = 0;
  int over = a.over;
  auto put = [&](int64_t t0, const Kv4Tile *mine) {
    int64_t own = 0, all;
#pragma unroll
    for (int i = 0; i < kListRounds; i++) own += mine[i].units;
    int64_t u = units + scan(own, all);
    const int64_t at = t0 + per * tid;
#pragma unroll
    for (int i = 0; i < kListRounds; i++) {
      if (i < per && at + i < tiles) {
        a.tiles[at + i] = mine[i];
        a.cum[at + i] = u;
      }
      u += mine[i].units;
    }
    units += all;
  };
  // A multiple of the waves that share a segment, and not so few units that joining costs more.
  auto chunk_of = [&](int64_t all) {
    if (all <= (int64_t)a.min_units * a.workgroups) return (int64_t)a.min_units;
    const int64_t c = (all + a.workgroups - 1) / a.workgroups;
    return (c + a.unit - 1) / a.unit * a.unit;
  };
  Kv4Tile mine[kListRounds];
  if (tiles <= kListRounds * kListThreads) {
    take(0, mine);
    int64_t own = 0, sums;  // key tiles, and 12 bits of column tiles that have some
#pragma unroll
    for (int i = 0; i < kListRounds; i++) own += ((int64_t)mine[i].n << 12) + (mine[i].n ? 1 : 0);
    scan(own, sums);
    const int64_t all = sums >> 12;
    chunk = chunk_of(all * a.hkv);
    // How many workgroups chunks of 0, 1, 2 and 3 thirds of the slack more would take, two counts a word.
    bool single = false;  // every workgroup has one segment
    if (a.slack > 0 && chunk < (1 << 28)) {
      int64_t need[2] = {0, 0}, total[2];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int c = (int)chunk + k * (a.slack / 3);
        int64_t n = 0;
#pragma unroll
        for (int i = 0; i < kListRounds; i++)
          if (i < per) n += (mine[i].n + c - 1) / c;
        need[k >> 1] |= min(n, (int64_t)1 << 20) << (32 * (k & 1));
      }
      scan(need[0], total[0]);
      scan(need[1], total[1]);
      for (int k = 0; k < 4; k++)
        if (((total[k >> 1] >> (32 * (k & 1))) & 0xffffffff) * a.hkv <= a.workgroups) {
          const int c = (int)chunk + k * (a.slack / 3);
#pragma unroll
          for (int i = 0; i < kListRounds; i++)
            if (i < per) mine[i].units = (mine[i].n + c - 1) / c * c;
          chunk = c;
          over = 0;
          single = true;
          break;
        }
    }
    if (!single) chunk = chunk_of((all + (sums & 0xfff) * a.over) * a.hkv);
    put(0, mine);
  } else {
    for (int64_t t0 = 0; t0 < tiles; t0 += kListRounds * kListThreads) {
      take(t0, mine);
      put(t0, mine);
    }
    chunk = chunk_of(units * a.hkv);
  }
  if (tid == 0) {
    a.cum[tiles] = units;
    a.head->tiles = (int)tiles;
    a.head->chunk = chunk;
    a.head->over = over;
    a.head->covered = a.cu_q ? a.cu_q[a.num_seqs] : a.num_seqs;
    a.head->first = a.cu_q ? a.cu_q[0] : 0;
  }
}

// Stores the step's rows and builds its lists: the first workgroups a list each, the others
// 256 / (D / 8) rows of K or V each.  A decode step of 128 rows takes 5.2 us, of which the list's chain of
// loads and scans is 3; 3300 tokens of 8 KV heads of 128 dims 12.6 (27 MB in, 2.2 TB/s: half of it is the
// launch and the scattered words of a token, which the caches put together).  The list is in this launch
// as one of its own would cost 2 us more.
template <int D>
__global__ void __launch_bounds__(256) kv4_store_kernel(Kv4Store a) {
  if ((int)blockIdx.x < a.lists) {
    build_list(a.list[blockIdx.x]);
    return;
  }
  constexpr int LPR = D / 8, ROWS = 256 / LPR;
  const int64_t row = (int64_t)(blockIdx.x - a.lists) * ROWS + threadIdx.x / LPR;
  const int64_t half = (int64_t)a.tokens * a.kv.hkv;
  if (row >= 2 * half) return;  // (whole quads)
  const bool is_v = row >= half;
  const int64_t r = is_v ? row - half : row;
  const int t = (int)(r / a.kv.hkv), h = (int)(r - (int64_t)t * a.kv.hkv);
  store_row<D>(a.kv, (is_v ? a.v : a.k) + r * D, a.slots[t], h, is_v, threadIdx.x % LPR);
}

// The values of rows at slots.  131072 rows of 8 KV heads of 128 dims, in random order: 373 us, 3.3 TB/s.
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

// One lane's part of a tile (of a quarter of the dims where waves share them).
template <int D> struct Tile {
  uint32_t k[2][D / 32];
  uint32_t v[D / 16];
  uint32_t ks;
  u32x2 vs;
};

// N words from byte `at` of a tile, 4 from each KB.  NT: keys read once (without the non-temporal bit a
// decode step's reads push everything else out).
template <int N, bool NT>
__device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t tile, uint32_t at, uint32_t *w) {
  constexpr int kPolicy = NT ? 2 : 0;
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(tile, at + 1024 * i, 0, kPolicy);
#pragma unroll
      for (int j = 0; j < 4; j++) w[4 * i + j] = x[j];
    }
  } else if constexpr (N == 2) {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(tile, at, 0, kPolicy);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(tile, at, 0, kPolicy);
  }
}

// Where a lane's parts lie in a tile: of all dims, or (DIMS) of wave's quarter.
struct TilePlaces {
  uint32_t k, v, ks, vs;
};
template <int D, bool DIMS> __device__ __forceinline__ TilePlaces tile_places(int lane, int wave) {
  constexpr int NB = D / 32;
  const int c = lane & 15, w = lane >> 4, quarter = DIMS ? wave : 0;
  return {(uint32_t)run_at(lane, 16 * quarter, D / 8), (uint32_t)(16 * D + run_at(lane, 32 * quarter, D / 4)),
          (uint32_t)(32 * D + (c * NB + (w * D) / 128 + quarter) * 2),
          (uint32_t)(33 * D + (w * NB + (c * D) / 512) * 8)};
}

// As buffer loads: the tile's address stays in scalar registers and the lane's places do not change, so that
// no address is computed in registers that loads in flight are still to be written to (which would wait for
// them).  D: the dims that are loaded, of FULL.
template <int D, int FULL, bool NT>
__device__ __forceinline__ void load_keys(__amdgpu_buffer_rsrc_t tile, const TilePlaces &p, Tile<D> &t) {
  load_words<D / 32, NT>(tile, p.k, t.k[0]);
  load_words<D / 32, NT>(tile, p.k + 8 * FULL, t.k[1]);
  if constexpr (D == 256)
    load_words<1, NT>(tile, p.ks, &t.ks);
  else
    t.ks = __builtin_amdgcn_raw_buffer_load_b16(tile, p.ks, 0, NT ? 2 : 0);
}
template <int D, bool NT>
__device__ __forceinline__ void load_values(__amdgpu_buffer_rsrc_t tile, const TilePlaces &p, Tile<D> &t) {
  load_words<D / 16, NT>(tile, p.v, t.v);
  uint32_t vs[2];
  load_words<2, NT>(tile, p.vs, vs);
  t.vs = u32x2{vs[0], vs[1]};
}

__device__ __forceinline__ uint32_t byte_of(uint32_t word, int i) { return (word >> (8 * i)) & 255u; }

template <int D> __device__ __forceinline__ float k_unit(const Tile<D> &t, int j, int half) {
  return mx4_unit(byte_of(t.ks, (j / 4) * 2 + half));
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

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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

// O += P V (FEW) or O^T += V^T P^T.
template <int D, int NG, int NP, bool FEW, int B = 0>
__device__ __forceinline__ void add_values(const Tile<D> &t, const float *unit, const bf16x8 (*p)[NP],
                                           f32x4 (*o)[D / 16]) {
  if constexpr (B < D / 32) {
    bf16x8 even, odd;
    v_frags<D, B>(t, unit, even, odd);
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
      for (int g = 0; g < NG; g++) {
        o[g][2 * B] = FEW ? mfma(p[g][i], even, o[g][2 * B]) : mfma(even, p[g][i], o[g][2 * B]);
        o[g][2 * B + 1] = FEW ? mfma(p[g][i], odd, o[g][2 * B + 1]) : mfma(odd, p[g][i], o[g][2 * B + 1]);
      }
    add_values<D, NG, NP, FEW, B + 1>(t, unit, p, o);
  }
}

// The maximum or sum over the 16 lanes of a row, in every lane.
__device__ __forceinline__ float max16(float x) {
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// A wave-uniform load of what earlier launches wrote, through the scalar cache: it waits on a counter of its
// own, where a vector load would wait for every key in flight.
template <typename T> __device__ __forceinline__ T uniform(const T *p) {
  typedef const T __attribute__((address_space(4))) * scalar;
  return *(scalar)(uintptr_t)p;
}

__device__ __forceinline__ Kv4Tile uniform_tile(const Kv4Tile *p) {
  typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
  static_assert(sizeof(Kv4Tile) == sizeof(i32x8), "one scalar load");
  return __builtin_bit_cast(Kv4Tile, uniform(reinterpret_cast<const i32x8 *>(p)));
}

// The 64-ary search for the last entry of cum that u reaches (times hkv), by a wave: tile of unit u.  Its first
// round covers the entries that the list has room for (those behind the n it has count as not reached), so
// that it need not wait for n.
__device__ __forceinline__ int find_tile(const int64_t *cum, int room, int n, int64_t u, int hkv, int lane) {
  int lo = 0, hi = room;
  do {
    const int step = (hi - lo + 63) >> 6;
    const int at = lo + lane * step;
    const int64_t before = cum[min(at, hi - 1)];
    const uint64_t le = __ballot(at < hi && at < n && before * hkv <= u);
    const int i = 63 - __builtin_clzll(le | 1);  // (lane 0 holds)
    lo += i * step;
    hi = min(hi, lo + step);
  } while (hi - lo > 1);
  return lo;
}

// Words between rows of P in LDS.
constexpr int kPRow = 20;

// How far scores may pass the reference that probabilities are taken relative to before it is raised:
// they are then at most 2^kSlack, which fp32 holds as exactly as those below 1.  Sums of probabilities times
// values stay finite where the values are below 2^67 (scale bytes below 192): 2^31 keys make less than 2^122.
// A tile with larger values, up to 6 * 2^125, raises the reference to kGuard above its highest score, so
// that its probabilities are at most 2^-31 and 2^31 of its keys sum to no more than the largest value.
// (Always taking probabilities that low would lose the small values instead.  Looking at the scales costs
// prompts of d = 64 3% and others less than 1%.)
constexpr float kSlack = 24.f, kGuard = 31.f;

// The weight of a partial beside those of the highest reference.  (No reference: no keys, or scores that are
// NaN, which the sum holds.)
__device__ __forceinline__ float weight_of(float m, float l, float big) {
  return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - big);
}

}  // namespace

// Workgroup g: its units' segments, each of one column tile and KV head, with the running reference and
// sum of a softmax.  A segment that covers its keys is written out; others leave partials (slot 2 g for
// the workgroup's first, of keys another one began, 2 g + 1 for its last), which kv4_merge_kernel joins.
//   KV4_FEW, KV4_EIGHT   NG groups of 4 columns, their parts as rows; the four waves take the key tiles in
//                        turn and join through LDS
//   KV4_ROWS             16 columns, three products; the waves as above
//   KV4_TILES            NG groups of 16 columns a wave, four waves of columns over the same key tiles
//   KV4_DIMS             16 columns, the four waves a quarter of the dims each over the same key tiles: their
//                        parts of the scores are added through LDS, and nothing joins at the end.  (d = 512 as
//                        KV4_ROWS has 128 registers of results a wave and q in LDS: one wave a SIMD, and
//                        prompts of 121 rows take 322 us instead of 196.)
//
// Decode is bound by reading the keys once: d = 128, 4 columns, 128 rows of up to 16K tokens (1.18 GB) take
// 194 us, 6.1 TB/s (the loads alone 186); 128 rows of d = 256 (295 MB) 52, 5.7 TB/s; 64 rows of eight
// columns (306 MB) 67 to 75, with both groups' softmax to do; 8 columns of d = 512 (307 MB) 81, half of its
// products on columns that are not there.  Few or short rows are bound by the chain of launch, list, q, keys
// and join: 5 rows of up to 700 tokens take 9.3 us whole and 7.5 split (an empty launch 2.2).  Prompts are
// bound by the matrix cores: 3 x 181 GFLOP of products (d = 128, chunks of up to 700 behind up to 4000
// tokens) take 500 us, 1.09 PFLOP/s (a library product of 8192 cubed makes 1.22 here).  Few columns as rows
// of three parts do no score twice: 16-column products for 4 columns were compute-bound at 242 us for the
// 128 rows.
template <int D, int MODE, int NG>
__global__ void __launch_bounds__(256, kv4_min_waves(D, MODE)) kv4_attention_kernel(Kv4Attention a) {
  constexpr bool FEW = MODE == KV4_FEW || MODE == KV4_EIGHT, TILES = MODE == KV4_TILES;
  constexpr bool DIMS = MODE == KV4_DIMS;
  constexpr int DW = DIMS ? D / kWaves : D;  // dims of a wave
  constexpr int NP = FEW ? 1 : 3;
  constexpr int NC = DW / 32;  // contraction steps of a score
  constexpr int COLS = kv4_cols(D, MODE);
  constexpr int E = DW / 16;   // the wave's dims of a row of V
  static_assert(COLS == (FEW ? 4 : TILES ? 64 : 16) * NG, "the columns of a tile");
  extern __shared__ float4 smem[];
  float *lds_o = reinterpret_cast<float *>(smem);  // [wave][col][D + 4]
  float *lds_m = lds_o + kWaves * COLS * (D + 4), *lds_l = lds_m + kWaves * COLS;
  f32x4 *lds_s = reinterpret_cast<f32x4 *>(smem);  // (DIMS) [turn][wave][group][half][lane]
  int turn = 0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, w = lane >> 4;
  // (FEW) the wave's P, [group][row 16][key 32] bf16, rows kPRow words apart (no bank conflicts in either
  // direction); rows of part 3 are zero.
  uint32_t *lds_p = reinterpret_cast<uint32_t *>(lds_l + kWaves * COLS) + wave * (NG * 16 * kPRow);
  if constexpr (FEW)
    for (int i = lane; i < NG * 16 * kPRow; i += 64) lds_p[i] = 0;
  const int n_tiles = uniform(&a.head->tiles);
  const int64_t chunk = uniform(&a.head->chunk);
  const int over = uniform(&a.head->over);
  const int64_t all = uniform(a.cum + n_tiles) * a.kv.hkv;
  int64_t u = (int64_t)blockIdx.x * chunk;
  const int64_t u_end = min(u + chunk, all);
  Kv4Border border{0, -1, 0, 0, 0, 0};
  if (u >= u_end) {
    if (threadIdx.x == 0) a.borders[blockIdx.x] = border;
    return;
  }
  const int rep = a.hq / a.kv.hkv;
  const int per_block = a.kv.block_size >> 5;
  const TilePlaces places = tile_places<D, DIMS>(lane, wave);
  int ct = __builtin_amdgcn_readfirstlane(find_tile(a.cum, a.room, n_tiles, u, a.kv.hkv, lane));
  while (u < u_end) {
    while (u >= uniform(a.cum + ct + 1) * a.kv.hkv) ct++;  // (u is below the last entry's)
    const Kv4Tile tile = uniform_tile(a.tiles + ct);
    const int64_t in = u - uniform(a.cum + ct) * a.kv.hkv;
    // (64-bit divisions cost hundreds of instructions: columns are below 2^30, chunks as good as never larger.)
    const int head = in <= UINT32_MAX ? (int)((uint32_t)in / (uint32_t)tile.units) : (int)(in / tile.units);
    // Units [v0, v1) of the KV head's, of which the first `over` are no keys.
    const int v0 = (int)(in - (int64_t)head * tile.units);
    const int v1 = (int)min((int64_t)tile.units, v0 + (u_end - u));
    const int t0 = max(v0 - over, 0), t1 = min(tile.n, v1 - over);
    u += v1 - v0;
    if (t1 <= t0) continue;
    const int seq = tile.seq;
    const int row0 = tile.row0, qlen = tile.qlen, klen = tile.klen;
    const int cols = qlen * rep;
    const int first_col = tile.col0 + (TILES ? wave * (16 * NG) : 0);
    const bool whole = t0 == 0 && t1 == tile.n;
    const int64_t part0 = (int64_t)(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * COLS;
    if (t0 > 0 && t0 <= chunk) {  // (its workgroup's first segment) the workgroup before began it
      border = Kv4Border{(int32_t)(blockIdx.x - 1),
                         (int32_t)blockIdx.x + (chunk < tile.n ? (tile.n - t0 - 1) / (int)chunk : 0), row0,
                         head * rep, tile.col0, min(COLS, cols - tile.col0)};
    }
    if (TILES && first_col >= cols) continue;  // (a wave by itself: these waves meet at no barrier)
    const int32_t *table = a.table + (size_t)seq * a.bt_stride;
    // Key tile t's place among its block's tiles, and its block.
    auto block_index = [&](int t) {
      const int kt = tile.kb + t;
      return a.tile_shift >= 0 ? kt >> a.tile_shift : kt / per_block;
    };
    auto block_of = [&](int t) { return uniform(table + block_index(t)); };
    auto buffer = [&](int t, int block) {
      const int in_block = tile.kb + t - block_index(t) * per_block;
      return __builtin_amdgcn_make_buffer_rsrc(a.kv.pages + tile_at(a.kv, block, head, in_block, D),
                                               (short)0, 34 * D, kBufferWord3);
    };
    auto load = [&](int t, int block, Tile<DW> &into) {
      const __amdgpu_buffer_rsrc_t from = buffer(t, block);
      load_keys<DW, D, !TILES>(from, places, into);
      load_values<DW, !TILES>(from, places, into);
      // The loads go out before the products of the tile at hand (the compiler would have them wait for
      // that tile, whose registers it could then use again).
      __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int STRIDE = TILES || DIMS ? 1 : kWaves;
    int t = t0 + (TILES || DIMS ? 0 : wave);
    // The columns whose scores the lane has see keys [lo, hi).  (Columns past the last repeat it.)
    int hi[NG], lo[NG], all_hi = INT32_MAX, all_lo = 0, any_hi = 0, any_lo = INT32_MAX;
#pragma unroll
    for (int g = 0; g < NG; g++) {
      hi[g] = klen - qlen + min(first_col + (FEW ? 4 * g + w : 16 * g + c), cols - 1) / rep + 1;
      lo[g] = a.window > 0 ? max(0, max(hi[g], 0) - a.window) : 0;
      all_hi = min(all_hi, hi[g]);
      any_hi = max(any_hi, hi[g]);
      all_lo = max(all_lo, lo[g]);
      any_lo = min(any_lo, lo[g]);
    }
    // Tiles that every column sees whole need no mask, those that none sees no work.
#pragma unroll
    for (int d = FEW ? 16 : 1; d < (FEW ? 64 : 16); d <<= 1) {
      all_hi = min(all_hi, __shfl_xor(all_hi, d));
      all_lo = max(all_lo, __shfl_xor(all_lo, d));
      any_hi = max(any_hi, __shfl_xor(any_hi, d));
      any_lo = min(any_lo, __shfl_xor(any_lo, d));
    }
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    any_hi = __builtin_amdgcn_readfirstlane(any_hi);
    any_lo = __builtin_amdgcn_readfirstlane(any_lo);
    // The wave's key tiles of the segment (each is below 2^26).
    int te = t1;
    if constexpr (TILES) {
      t = max(t, (any_lo >> 5) - tile.kb);
      te = min(te, (max(any_hi, 0) + 31) / 32 - tile.kb);
    }
    // (TILES) the first tile is on its way while q is loaded and split.  (Where the registers that hold it are
    // not there anyway, in the kernels of few columns, it cost 5%.)
    Tile<DW> one;
    if (TILES && t < te) load(t, block_of(t), one);
    bf16x8 q[NG][NC][NP];
#pragma unroll
    for (int g = 0; g < NG; g++) {
      // The column of q that the lane loads.
      const int col = min(first_col + (FEW ? 4 * g + (c >> 2) : 16 * g + c), cols - 1);
      const int qrow = col / rep;
      const float *qp = a.q + ((size_t)(row0 + qrow) * a.hq + head * rep + (col - qrow * rep)) * D +
                        w * (D / 4) + (DIMS ? wave * 32 : 0);
#pragma unroll
      for (int j = 0; j < NC; j++) {
        float x[8];
        *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(qp + 8 * j);
        *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(qp + 8 * j + 4);
        // Scores come out in units of log2 (one rounding of q more).
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] *= a.scale2;
        bf16x8 p[3];
        split3<false>(x, p);
        if constexpr (FEW) {
          const bf16x8 zero = {};
          q[g][j][0] = (c & 3) == 0 ? p[0] : (c & 3) == 1 ? p[1] : (c & 3) == 2 ? p[2] : zero;
        } else {
#pragma unroll
          for (int i = 0; i < 3; i++) q[g][j][i] = p[i];
        }
      }
    }
    f32x4 o[NG][E];
    float m[NG], l[NG];
    uint32_t nan[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
      nan[g] = 0;
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int i = 0; i < E; i++) o[g][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // Scores of the 32 keys, of either half of them.
    auto scores = [&](const Tile<DW> &cur, f32x4 (*s)[2]) {
#pragma unroll
      for (int g = 0; g < NG; g++) s[g][0] = s[g][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NC; j++) {
        const bf16x8 k0 = mx4_frag(cur.k[0][j], k_unit<DW>(cur, j, 0));
        const bf16x8 k1 = mx4_frag(cur.k[1][j], k_unit<DW>(cur, j, 1));
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
          for (int i = 0; i < NP; i++) {
            const bf16x8 qv = q[g][j][i];
            s[g][0] = FEW ? mfma(qv, k0, s[g][0]) : mfma(k0, qv, s[g][0]);
            s[g][1] = FEW ? mfma(qv, k1, s[g][1]) : mfma(k1, qv, s[g][1]);
          }
      }
      if constexpr (DIMS) {
        // The sum of the waves' parts, the same bits in each.  (The other half of the buffer was read before
        // the last barrier; loads in flight stay so.)
        f32x4 *buf = lds_s + (turn & 1) * (kWaves * NG * 2 * 64);
        turn++;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
          for (int h = 0; h < 2; h++) buf[((wave * NG + g) * 2 + h) * 64 + lane] = s[g][h];
        wait_lds_reads();
        lds_barrier();
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            f32x4 sum = buf[(g * 2 + h) * 64 + lane];
#pragma unroll
            for (int v = 1; v < kWaves; v++) sum += buf[((v * NG + g) * 2 + h) * 64 + lane];
            s[g][h] = sum;
          }
      }
    };
    // Their probabilities, and the values of their V.
    auto values = [&](int t, Tile<DW> &cur, f32x4 (*s)[2]) {
      const int key0 = (tile.kb + t) * 32;
      const bool edge = key0 + 32 > all_hi || key0 < all_lo;
      // Does any of its values pass 2^67: a scale byte with both upper bits, of a key that some column sees?
      // (All of the waves that share the dims hold the same scales.)
      const u32x2 both = cur.vs & (cur.vs << 1);
      bool large = __any(((both.x | both.y) & 0x80808080u) != 0);
      if (large) {
        const u32x2 upper = both & 0x80808080u;
        bool seen = false;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int key = key0 + 8 * w + i;
          seen |= (byte_of(upper[i >> 2], i & 3) != 0) & (key < any_hi) & (key >= any_lo);
        }
        large = __any(seen);
      }
      const float slack = large ? -kGuard : kSlack, guard = large ? kGuard : 0.f;
      constexpr int NX = FEW ? 2 : 8;  // scores of a lane and column: keys NX (lane's) .. + NX - 1
      const int mine = key0 + NX * (FEW ? c : w);
      bf16x8 p[NG][NP];
#pragma unroll
      for (int g = 0; g < NG; g++) {
        float x[NX];
#pragma unroll
        for (int i = 0; i < NX; i++) {
          if constexpr (FEW)
            x[i] = s[g][i][0] + (s[g][i][1] + s[g][i][2]);
          else
            x[i] = s[g][i & 1][i >> 1];
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < NX; i++)
            if (mine + i >= hi[g] || mine + i < lo[g]) x[i] = -INFINITY;
        }
        float top = fmaxf(x[0], x[1]);
#pragma unroll
        for (int i = 2; i < NX; i++) top = fmaxf(top, x[i]);
        if (__any(top > m[g] + slack)) {
          if constexpr (FEW) top = max16(top); else top = max4_lanes(top);
          const float grown = top > m[g] + slack ? top + guard : m[g];
          const float f = m[g] == grown ? 1.f : __builtin_amdgcn_exp2f(m[g] - grown);  // 0 from -infinity
          m[g] = grown;
          l[g] *= f;
#pragma unroll
          for (int i = 0; i < E; i++) o[g][i] *= f;
        }
        const float base = m[g] == -INFINITY ? 0.f : m[g];
#pragma unroll
        for (int i = 0; i < NX; i++) {
          x[i] = __builtin_amdgcn_exp2f(x[i] - base);
          l[g] += x[i];
        }
        if constexpr (FEW) {
          // Both keys' parts, one word each, to row 4 w + part.
          uint32_t *row = lds_p + (g * 16 + 4 * w) * kPRow + c;
#pragma unroll
          for (int i = 0; i < 3; i++) {
            row[i * kPRow] = high_halves(__float_as_uint(x[0]), __float_as_uint(x[1]));
            x[0] -= __uint_as_float(__float_as_uint(x[0]) & 0xffff0000u);
            x[1] -= __uint_as_float(__float_as_uint(x[1]) & 0xffff0000u);
          }
        } else {
          split3<true>(x, p[g]);
        }
      }
      if constexpr (FEW) {
        asm volatile("" ::: "memory");  // (a wave's LDS operations are in order; the compiler's are, too)
#pragma unroll
        for (int g = 0; g < NG; g++)
          p[g][0] = __builtin_bit_cast(
              bf16x8, *reinterpret_cast<const u32x4 *>(lds_p + (g * 16 + c) * kPRow + 4 * w));
        asm volatile("" ::: "memory");
      }
      float unit[8];
#pragma unroll
      for (int i = 0; i < 8; i++) unit[i] = mx4_unit(byte_of(cur.vs[i >> 2], i & 3));
      if (edge) {
        // A block that is NaN reaches only the columns that see its key, though all of a wave's columns are
        // multiplied with it: its values are taken as next to nothing here, and the rows of O that a column
        // sees one of become NaN at the end (bits of nan; a row's dims share one block, d / 16 of 32).
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; i++) bad |= unit[i] == INFINITY;
        if (__any(bad)) {
          uint32_t mark[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const bool is = unit[i] == INFINITY;
            mark[i] = is ? 0x3f80u : 0u;  // 1 in bf16
            unit[i] = is ? 0.f : unit[i];
          }
          const bf16x8 marks = frag(low_halves(mark[0], mark[1]), low_halves(mark[2], mark[3]),
                                    low_halves(mark[4], mark[5]), low_halves(mark[6], mark[7]));
#pragma unroll
          for (int g = 0; g < NG; g++) {
            // Which of keys 8 w and on the operand's row or column sees.
            const int ohi = FEW ? __shfl(hi[g], 16 * (c >> 2)) : hi[g];
            const int olo = FEW ? __shfl(lo[g], 16 * (c >> 2)) : lo[g];
            uint32_t see[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int key = key0 + 8 * w + i;
              see[i] = key < ohi && key >= olo ? 0x3f80u : 0u;
            }
            const bf16x8 sees = frag(low_halves(see[0], see[1]), low_halves(see[2], see[3]),
                                     low_halves(see[4], see[5]), low_halves(see[6], see[7]));
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            const f32x4 n = FEW ? mfma(sees, marks, zero) : mfma(marks, sees, zero);
#pragma unroll
            for (int r = 0; r < 4; r++) nan[g] |= n[r] > 0.f ? 1u << r : 0u;
          }
        }
      }
      add_values<DW, NG, NP, FEW>(cur, unit, p, o);
    };
    auto attend = [&](int t, Tile<DW> &cur) {
      f32x4 s[NG][2];
      scores(cur, s);
      values(t, cur, s);
    };
    if constexpr (TILES) {
      // One tile's registers: the next keys are loaded behind the scores, the next values behind the sums.
      // (The last turns load the last tile again: loads behind a condition would be waited for as if they
      // were needed at once.)
      if (t < te) {
        int next = min(t + STRIDE, te - 1), block = block_of(next);
        for (; t < te; t += STRIDE) {
          f32x4 s[NG][2];
          scores(one, s);
          const __amdgpu_buffer_rsrc_t from = buffer(next, block);
          __builtin_amdgcn_sched_barrier(0);
          load_keys<DW, D, !TILES>(from, places, one);
          next = min(t + 2 * STRIDE, te - 1);
          block = block_of(next);
          __builtin_amdgcn_sched_barrier(0);
          values(t, one, s);
          __builtin_amdgcn_sched_barrier(0);
          load_values<DW, !TILES>(from, places, one);
        }
      }
    } else {
      // The next tile loads into the other registers while this one is attended.  (The last turn loads the
      // last tile again: loads behind a condition would be waited for as if they were needed at once.)  Two
      // and three tiles ahead were 2 to 20% slower for the registers that they take.
      Tile<DW> even, odd;
      if (t < te) {
        int next = t, block = block_of(t);
        auto ahead = [&](Tile<DW> &into) {
          load(next, block, into);
          next = min(next + STRIDE, te - 1);
          block = block_of(next);
        };
        ahead(even);
        while (true) {
          ahead(odd);
          attend(t, even);
          if ((t += STRIDE) >= te) break;
          ahead(even);
          attend(t, odd);
          if ((t += STRIDE) >= te) break;
        }
      }
    }
    // NaN where a column saw one, then the lane's results: FEW has E dims of column 4 g + w (the sum of
    // its parts, in r = 0), the others E dims of four rows of V for column c.
#pragma unroll
    for (int g = 0; g < NG; g++) {
      if constexpr (FEW) {
        l[g] = sum16(l[g]);
#pragma unroll
        for (int i = 0; i < E; i++) {
          const float sum = o[g][i][0] + (o[g][i][1] + o[g][i][2]);
          o[g][i][0] = nan[g] & 1 ? NAN : sum;
        }
      } else {
        l[g] = sum4_lanes(l[g]);
        if (__any(nan[g] != 0))
#pragma unroll
          for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < E; i++) o[g][i][r] = (nan[g] >> r) & 1 ? NAN : o[g][i][r];
      }
    }

    if constexpr (TILES || DIMS) {  // every wave writes its own columns, or its own dims
#pragma unroll
      for (int g = 0; g < NG; g++) {
        const int col = first_col + 16 * g + c;
        if (col >= cols) continue;
        const int row = col / rep;
        const size_t part = (size_t)part0 + (TILES ? wave * (16 * NG) : 0) + 16 * g + c;
        const float inv = whole ? (l[g] == 0.f ? 0.f : 1.f / l[g]) : 1.f;
        float *dst = whole ? a.out + ((size_t)(row0 + row) * a.hq + head * rep + (col - row * rep)) * D
                           : a.part_o + part * D;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int i = 0; i < E; i += 4)
            *reinterpret_cast<float4 *>(dst + (4 * w + r) * (D / 16) + (DIMS ? wave * E : 0) + i) =
                make_float4(o[g][i][r] * inv, o[g][i + 1][r] * inv, o[g][i + 2][r] * inv,
                            o[g][i + 3][r] * inv);
        if (!whole && w == 0 && (TILES || wave == 0)) {
          a.part_m[part] = m[g];
          a.part_l[part] = l[g];
        }
      }
      continue;
    }

    // Join the waves: sums and rows over the highest reference.
#pragma unroll
    for (int g = 0; g < NG; g++) {
      const int at = wave * COLS + (FEW ? 4 * g + w : c);
      if (FEW ? c == 0 : w == 0) {
        lds_m[at] = m[g];
        lds_l[at] = l[g];
      }
      float *to = lds_o + at * (D + 4);
#pragma unroll
      for (int r = 0; r < (FEW ? 1 : 4); r++)
#pragma unroll
        for (int i = 0; i < E; i += 4)
          *reinterpret_cast<float4 *>(to + (FEW ? c : 4 * w + r) * E + i) =
              make_float4(o[g][i][r], o[g][i + 1][r], o[g][i + 2][r], o[g][i + 3][r]);
    }
    __syncthreads();
    constexpr int LANES = 256 / COLS;  // lanes of a column
    const int oc = threadIdx.x / LANES, ol = threadIdx.x % LANES;
    float ms[kWaves], big = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      ms[i] = lds_m[i * COLS + oc];
      big = fmaxf(big, ms[i]);
    }
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const float li = lds_l[i * COLS + oc];
      ms[i] = weight_of(ms[i], li, big);
      sum += ms[i] * li;
    }
    const int ocol = tile.col0 + oc;
    if (ocol < cols) {
      const int orow = ocol / rep;
      const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
      const size_t part = (size_t)part0 + oc;
      float *dst = whole ? a.out + ((size_t)(row0 + orow) * a.hq + head * rep + (ocol - orow * rep)) * D
                         : a.part_o + part * D;
#pragma unroll
      for (int i = 0; i < (D + 4 * LANES - 1) / (4 * LANES); i++) {
        const int e = 4 * (ol + LANES * i);
        if (e >= D) break;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < kWaves; v++)
          if (ms[v] != 0.f)  // (a wave without keys has nothing)
            acc += ms[v] * *reinterpret_cast<const f32x4 *>(lds_o + (v * COLS + oc) * (D + 4) + e);
        acc *= inv;
        *reinterpret_cast<f32x4 *>(dst + e) = acc;
      }
      if (!whole && ol == 0) {
        a.part_m[part] = big;
        a.part_l[part] = sum;
      }
    }
    __syncthreads();  // lds_o is written again
  }
  if (threadIdx.x == 0) a.borders[blockIdx.x] = border;
}

// Joins the partials of column tiles that several workgroups shared: workgroup x that of the first border
// between workgroups in it, which workgroup x of the attention left.  W waves a column, 4 / W columns a
// workgroup.  Then zeroes for rows without keys and rows that no sequence covers.  Bound by its chain of
// loads: 4 to 5 us for a decode step, 7 for rows of 43 partials, 25 for prompts (512 borders of 128
// columns, some 100 MB of partials; 34 with weights loaded before the rows).
template <int W>
__global__ void __launch_bounds__(256) kv4_merge_kernel(Kv4Attention a, int cols_of_tile) {
  const int D = a.head_dim, rep = a.hq / a.kv.hkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const Kv4Border b = a.borders[blockIdx.x];
  const int c = blockIdx.y * (4 / W) + wave / W;
  if (b.g1 >= 0 && c < b.cols) {  // (uniform over a column's waves)
    const int col = b.col0 + c, row = col / rep;
    float *dst = a.out + ((size_t)(b.row0 + row) * a.hq + b.head0 + (col - row * rep)) * D;
    // Partial of workgroup g: its last for the first one, its first for the others.
    auto slot = [&](int g) { return (size_t)(2 * g + (g == b.g0 ? 1 : 0)) * cols_of_tile + c; };
    if (W == 1 && b.g1 - b.g0 < 4) {  // few partials: all of their loads at once
      float m[4], l[4], big = -INFINITY, sum = 0.f;
      f32x2 row_of[4][4], acc[4] = {};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const size_t at = slot(min(b.g0 + j, b.g1));
        m[j] = a.part_m[at];
        l[j] = a.part_l[at];
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (2 * lane + 128 * k < D)
            row_of[j][k] = *reinterpret_cast<const f32x2 *>(a.part_o + at * D + 2 * lane + 128 * k);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) big = fmaxf(big, m[j]);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float f = b.g0 + j > b.g1 ? 0.f : weight_of(m[j], l[j], big);
        sum += f * l[j];
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (2 * lane + 128 * k < D && f != 0.f) acc[k] += f * row_of[j][k];
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (2 * lane + 128 * k < D) *reinterpret_cast<f32x2 *>(dst + 2 * lane + 128 * k) = acc[k] * inv;
    } else {
      float big = -INFINITY;
      for (int g = b.g0 + lane; g <= b.g1; g += 64) big = fmaxf(big, a.part_m[slot(g)]);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) big = fmaxf(big, __shfl_xor(big, d));
      float sum = 0.f;
      f32x2 acc[4] = {};  // dims 2 lane + 128 i
      for (int base = b.g0; base <= b.g1; base += 64) {
        // A lane a partial's weight, then all lanes the wave's rows.
        float f = 0.f;
        if (base + lane <= b.g1) {
          const float m = a.part_m[slot(base + lane)], l = a.part_l[slot(base + lane)];
          f = weight_of(m, l, big);
          sum += f * l;
        }
        const int n = min(64, b.g1 - base + 1);
        for (int i = W == 1 ? 0 : wave; i < n; i += 4 * W) {  // four rows' loads at once
          f32x2 row_of[4][4];
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int at = min(i + j * W, n - 1);
            w[j] = i + j * W < n ? __shfl(f, at) : 0.f;
            const float *src = a.part_o + slot(base + at) * D;
#pragma unroll
            for (int k = 0; k < 4; k++)
              if (2 * lane + 128 * k < D)
                row_of[j][k] = *reinterpret_cast<const f32x2 *>(src + 2 * lane + 128 * k);
          }
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int k = 0; k < 4; k++)  // (a row without weight saw nothing)
              if (2 * lane + 128 * k < D && w[j] != 0.f) acc[k] += w[j] * row_of[j][k];
        }
      }
      // (In a fixed order: a lane's sums, then lane by lane.)
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if constexpr (W == 1) {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (2 * lane + 128 * k < D)
            *reinterpret_cast<f32x2 *>(dst + 2 * lane + 128 * k) = acc[k] * inv;
      } else {
        __shared__ f32x2 sums[W][256];
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (2 * lane + 128 * k < D) sums[wave][lane + 64 * k] = acc[k];
        __syncthreads();
        for (int e = threadIdx.x; 2 * e < D; e += 256) {
          f32x2 all = sums[0][e];
#pragma unroll
          for (int i = 1; i < W; i++) all += sums[i][e];
          *reinterpret_cast<f32x2 *>(dst + 2 * e) = all * inv;
        }
      }
    }
  }
  if (blockIdx.y != 0) return;
  const int n_tiles = a.head->tiles;
  const int64_t stride = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const size_t width = (size_t)a.hq * D;
  // Rows whose column tile has no keys, a thread a column tile (there are few, and its rows are few).
  for (int64_t t = i0; t < n_tiles; t += stride) {
    const Kv4Tile tile = a.tiles[t];
    if (tile.n) continue;
    const int row0 = tile.row0;
    const int64_t end = min((int64_t)tile.qlen * rep, (int64_t)tile.col0 + cols_of_tile);
    for (int64_t col = tile.col0; col < end; col++) {
      const int64_t row = col / rep;
      for (int h = 0; h < a.kv.hkv; h++) {
        float *dst = a.out + (row0 + row) * width + ((size_t)h * rep + (col - row * rep)) * D;
        for (int e = 0; e < D; e += 4) *reinterpret_cast<float4 *>(dst + e) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  if (!a.zero_rest) return;
  // Rows before the first sequence and behind the last one.
  const int first = a.head->first, covered = a.head->covered;
  const size_t n = ((size_t)first + (a.tokens - covered)) * width;
  for (size_t i = i0; i < n; i += stride) {
    const size_t r = i / width;
    a.out[(r < (size_t)first ? r : r - first + covered) * width + (i - r * width)] = 0.f;
  }
}

// ---------------------------------------------------------------- quantize

// One pass: 8192 x 8192 values take 46 us, 6.6 TB/s.
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

template <int D, int MODE> size_t attention_lds() {
  if (MODE == KV4_TILES) return 0;
  constexpr int cols = kv4_cols(D, MODE);
  const size_t join = (size_t)kWaves * cols * (D + 4 + 2) * 4;
  if (MODE == KV4_ROWS) return join;
  if (MODE == KV4_DIMS) return (size_t)2 * kWaves * (cols / 16) * 2 * 64 * 16;
  return join + (size_t)kWaves * (cols / 4) * 16 * kPRow * 4;
}

template <int D, int MODE> constexpr int groups() {
  return kv4_cols(D, MODE) / (MODE == KV4_TILES ? 64 : MODE == KV4_ROWS || MODE == KV4_DIMS ? 16 : 4);
}

// Rows of K and V that a launch takes: its threads are counted in 32 bits, and those of a larger grid would be
// left out without an error.
template <int D> int rows_at_once(int hkv) {
  return (int)std::max<int64_t>(1, ((int64_t)1 << 31) / (2 * (int64_t)hkv * (D / 8)));
}

template <int D> hipError_t store(const Kv4Store &a, hipStream_t s) {
  constexpr int ROWS = 256 / (D / 8);
  Kv4Store piece = a;
  int t = 0;
  do {
    piece.tokens = a.k ? std::min(a.tokens - t, rows_at_once<D>(a.kv.hkv)) : 0;
    const int64_t blocks = (2 * (int64_t)piece.tokens * a.kv.hkv + ROWS - 1) / ROWS + piece.lists;
    if (blocks == 0) break;
    hipLaunchKernelGGL(kv4_store_kernel<D>, dim3((unsigned)blocks), dim3(256), 0, s, piece);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    t += piece.tokens;
    piece.lists = 0;
    if (a.k) {
      piece.k = a.k + (size_t)t * a.kv.hkv * D;
      piece.v = a.v + (size_t)t * a.kv.hkv * D;
      piece.slots = a.slots + t;
    }
  } while (a.k && t < a.tokens);
  return hipSuccess;
}

template <int D>
hipError_t read(const Kv4View &kv, const int32_t *slots, float *k, float *v, int rows, hipStream_t s) {
  constexpr int ROWS = 256 / (D / 8);
  for (int t = 0; t < rows;) {
    const int n = std::min(rows - t, rows_at_once<D>(kv.hkv));
    const int64_t blocks = (2 * (int64_t)n * kv.hkv + ROWS - 1) / ROWS;
    const size_t at = (size_t)t * kv.hkv * D;
    hipLaunchKernelGGL(kv4_read_kernel<D>, dim3((unsigned)blocks), dim3(256), 0, s, kv, slots + t,
                       k ? k + at : nullptr, v ? v + at : nullptr, n);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    t += n;
  }
  return hipSuccess;
}

template <int D, int MODE> hipError_t attention(const Kv4Attention &a, int workgroups, hipStream_t s) {
  constexpr int NG = groups<D, MODE>();
  const auto kernel = &kv4_attention_kernel<D, MODE, NG>;
  const size_t lds = attention_lds<D, MODE>();
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((kv4_attention_kernel<D, MODE, NG>), dim3(workgroups), dim3(256), lds, s, a);
  return hipGetLastError();
}

template <int D> hipError_t attention_of(const Kv4Attention &a, int mode, int workgroups, hipStream_t s) {
  if constexpr (kv4_by_dims(D)) {
    return attention<D, KV4_DIMS>(a, workgroups, s);
  } else {
    switch (mode) {
      case KV4_FEW: return attention<D, KV4_FEW>(a, workgroups, s);
      case KV4_EIGHT: return attention<D, KV4_EIGHT>(a, workgroups, s);
      case KV4_ROWS: return attention<D, KV4_ROWS>(a, workgroups, s);
      default: return attention<D, KV4_TILES>(a, workgroups, s);
    }
  }
}

template <int D, int MODE> int resident() {
  constexpr int NG = groups<D, MODE>();
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
          &n, reinterpret_cast<const void *>(&kv4_attention_kernel<D, MODE, NG>), 256,
          attention_lds<D, MODE>()) != hipSuccess)
    (void)hipGetLastError();
  return std::max(1, n);
}

template <int D> int resident_of(int mode) {
  if constexpr (kv4_by_dims(D)) {
    return resident<D, KV4_DIMS>();
  } else {
    switch (mode) {
      case KV4_FEW: return resident<D, KV4_FEW>();
      case KV4_EIGHT: return resident<D, KV4_EIGHT>();
      case KV4_ROWS: return resident<D, KV4_ROWS>();
      default: return resident<D, KV4_TILES>();
    }
  }
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

hipError_t launch_kv4_attention(const Kv4Attention &a, int mode, int workgroups, hipStream_t s) {
#define args (a, mode, workgroups, s)
  NVA_BY_DIM(a.head_dim, attention_of)
#undef args
}

int kv4_workgroups_per_cu(int head_dim, int mode) {
  switch (head_dim) {
    case 64: return resident_of<64>(mode);
    case 128: return resident_of<128>(mode);
    case 256: return resident_of<256>(mode);
    default: return resident_of<512>(mode);
  }
}

hipError_t launch_kv4_merge(const Kv4Attention &a, int mode, int workgroups, int items, hipStream_t s) {
  const int cols = kv4_cols(a.head_dim, mode);
  // Few column tiles and heads (items) leave many partials each, for which four waves share a column (three
  // rows of 60-120K tokens, 43 partials: 13.5 -> 7 us; 1024 items: 8.7 us against 6.5 with one wave).
  if (mode != KV4_TILES && items <= workgroups / 4)
    hipLaunchKernelGGL(kv4_merge_kernel<4>, dim3(workgroups, cols), dim3(256), 0, s, a, cols);
  else
    hipLaunchKernelGGL(kv4_merge_kernel<1>, dim3(workgroups, cols / 4), dim3(256), 0, s, a, cols);
  return hipGetLastError();
}

}  // namespace nva
