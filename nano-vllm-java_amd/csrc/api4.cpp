// C ABI of the steps that are built on the device and of what is held in 4 bits: scaled rotary positions,
// block tables, the 4-bit arena with its attention, and 4-bit projections.  See include/nva.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "context.h"

namespace {

int shift_of(int x) {  // log2, or -1
  return x > 0 && (x & (x - 1)) == 0 ? __builtin_ctz((unsigned)x) : -1;
}

// The frequencies of a scaled RoPE in 64 bits, and the factor of cos and sin.
double frequencies(const nva_rope_desc &d, std::vector<double> &f) {
  const int rd = d.rotary_dim, pairs = rd / 2;
  double base = d.base;
  if (d.scaling == NVA_ROPE_NTK && rd > 2) base *= std::pow((double)d.factor, rd / (rd - 2.0));
  f.resize(pairs);
  for (int i = 0; i < pairs; i++) f[i] = std::pow(base, -2.0 * i / rd);
  const double two_pi = 6.283185307179586476925286766559;
  if (d.scaling == NVA_ROPE_LINEAR || (d.scaling == NVA_ROPE_NTK && rd == 2)) {
    for (double &x : f) x /= d.factor;
  } else if (d.scaling == NVA_ROPE_YARN) {
    // The pair that turns t times within the trained context.
    auto pair = [&](double t) {
      return rd * std::log(d.original_max_pos / (t * two_pi)) / (2.0 * std::log((double)d.base));
    };
    const double lo = std::max(0.0, std::floor(pair(d.high)));
    const double hi = std::min(rd - 1.0, std::ceil(pair(d.low)));
    for (int i = 0; i < pairs; i++) {
      const double mix = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 1e-3)));
      f[i] = f[i] / d.factor * mix + f[i] * (1.0 - mix);
    }
  } else if (d.scaling == NVA_ROPE_BANDS) {
    for (double &x : f) {
      const double turns = d.original_max_pos * x / two_pi;
      const double keep =
          std::min(1.0, std::max(0.0, (turns - d.low) / ((double)d.high - d.low)));
      x = (1.0 - keep) * x / d.factor + keep * x;
    }
  }
  if (d.amplitude != 0.0f) return d.amplitude;
  return d.scaling == NVA_ROPE_YARN ? 0.1 * std::log((double)d.factor) + 1.0 : 1.0;
}

nva_status check_rope(nva_ctx *ctx, const nva_rope_desc &d) {
  if (d.max_pos <= 0 || d.head_size <= 0 || d.head_size % 2)
    return fail(ctx, NVA_E_ARG, "RoPE table needs maxPos > 0 and an even headSize");
  if (d.rotary_dim < 2 || d.rotary_dim > d.head_size || d.rotary_dim % 2)
    return fail(ctx, NVA_E_ARG, "rotaryDim %d must be even, in [2, headSize %d]", d.rotary_dim,
                d.head_size);
  if (!(d.base > 1.0f) || !std::isfinite(d.base))
    return fail(ctx, NVA_E_ARG, "RoPE base must be > 1");
  if (d.scaling < NVA_ROPE_NONE || d.scaling > NVA_ROPE_BANDS)
    return fail(ctx, NVA_E_ARG, "unknown RoPE scaling %d", d.scaling);
  if (d.scaling != NVA_ROPE_NONE && (!(d.factor >= 1.0f) || !std::isfinite(d.factor)))
    return fail(ctx, NVA_E_ARG, "RoPE scaling needs factor >= 1");
  if (d.scaling == NVA_ROPE_YARN || d.scaling == NVA_ROPE_BANDS) {
    if (d.original_max_pos <= 0)
      return fail(ctx, NVA_E_ARG, "this RoPE scaling needs originalMaxPos > 0");
    if (!(d.low > 0.0f) || !(d.high > d.low) || !std::isfinite(d.high))
      return fail(ctx, NVA_E_ARG, "this RoPE scaling needs 0 < low < high");
  }
  if (!std::isfinite(d.amplitude) || d.amplitude < 0.0f)
    return fail(ctx, NVA_E_ARG, "RoPE amplitude must be >= 0");
  return NVA_OK;
}

Kv4View view_of(const nva_kv4 *kv, int layer) {
  return Kv4View{kv->pages[layer], kv->num_blocks, kv->block_size, kv->num_kv_heads};
}

int64_t kv4_block_bytes(int block_size, int hkv, int d) {
  return (int64_t)(block_size / 32) * hkv * 34 * d;
}

nva_status check_arena4(nva_ctx *ctx, int num_layers, int block_size, int num_kv_heads,
                        const int32_t *head_dims, const uint8_t *allocate) {
  if (num_layers <= 0) return fail(ctx, NVA_E_ARG, "numLayers must be > 0");
  if (block_size <= 0 || num_kv_heads <= 0 || !head_dims)
    return fail(ctx, NVA_E_ARG, "blockSize, numKvHeads must be > 0 and headDims non-null");
  if (block_size % 32)
    return fail(ctx, NVA_E_UNSUPPORTED, "the 4-bit arena needs blockSize %% 32 == 0 (got %d)",
                block_size);
  for (int i = 0; i < num_layers; i++)
    if ((!allocate || allocate[i]) && !kv4_supports(head_dims[i]))
      return fail(ctx, NVA_E_UNSUPPORTED,
                  "the 4-bit arena holds head dims 64, 128, 256 and 512, not headDims[%d] = %d", i,
                  head_dims[i]);
  return NVA_OK;
}

nva_status check_layer(nva_kv4 *kv, int layer) {
  if (layer < 0 || layer >= kv->num_layers)
    return fail(kv->ctx, NVA_E_LAYER, "layerIndex out of range: %d (layers=%d)", layer,
                kv->num_layers);
  return NVA_OK;
}

// The host step's block tables against the arena, once per step and sequence: every block that a sequence's
// keys lie in exists.
nva_status check_tables4(nva_ctx *ctx, const nva_kv4 *kv, int num_tokens) {
  if (ctx->checked_blocks != kv->num_blocks || ctx->checked_block_size != kv->block_size)
    ctx->checked_seqs = 0;
  const int seqs = ctx->is_prefill ? ctx->num_seqs : std::min(ctx->num_seqs, num_tokens);
  for (int b = ctx->checked_seqs; b < seqs; b++) {
    const int klen = ctx->is_prefill ? ctx->cu_k[b + 1] - ctx->cu_k[b] : ctx->ctx_lens[b];
    const int64_t pages = ((int64_t)klen + kv->block_size - 1) / kv->block_size;
    if (klen <= 0 || (ctx->is_prefill && ctx->cu_q[b + 1] == ctx->cu_q[b])) continue;
    if (klen > INT32_MAX - 8192)
      return fail(ctx, NVA_E_UNSUPPORTED, "sequence %d has %d keys", b, klen);
    if (pages > ctx->bt_stride)
      return fail(ctx, NVA_E_ARG, "sequence %d has %d keys but a block table of %d blocks", b, klen,
                  ctx->bt_stride);
    const int32_t *t = ctx->tables.data() + (size_t)b * ctx->bt_stride;
    for (int64_t i = 0; i < pages; i++)
      if (t[i] < 0 || t[i] >= kv->num_blocks)
        return fail(ctx, NVA_E_ARG, "sequence %d: block %d outside the arena's %d", b, t[i],
                    kv->num_blocks);
  }
  ctx->checked_blocks = kv->num_blocks;
  ctx->checked_block_size = kv->block_size;
  ctx->checked_seqs = std::max(ctx->checked_seqs, seqs);  // (a call of fewer rows has looked at fewer)
  return NVA_OK;
}

// Whether a call's rows go to the step's slots.
bool stores(const nva_ctx *ctx, const nva_attn_desc &d, int num_tokens) {
  return d.write_kv && (ctx->dev_step || (ctx->has_slots && ctx->num_slots == num_tokens));
}

int ctx_kv4_workgroups_per_cu(nva_ctx *ctx, int head_dim, int mode) {
  const int key = -(head_dim + 1000 * (mode + 1));  // beside the other kernels' keys
  auto it = ctx->occupancy.find(key);
  if (it == ctx->occupancy.end())
    it = ctx->occupancy.emplace(key, kv4_workgroups_per_cu(head_dim, mode)).first;
  return it->second;
}

constexpr int64_t kJoinUnits = 3500;
// The key tiles up to which the rows of a decode step are not split where there are workgroups for all, so
// that nothing is to be merged (4 to 5 us, and a launch).  Items are rows times KV heads (and column tiles).
// Few of them split over idle CUs; where the pieces of eight would share CUs, splitting gains less.  A step's
// kernels, split and whole, us:
//   few    1 row of 32 / 8 heads of 128: 18.1, 17.9 with 32 tiles, 18.4, 19.7 with 40; 5 rows of 4 / 1 heads
//          of 256: 19.8, 20.3 with 28, 19.7, 21.8 with 36; 5 of 8 / 1 heads of 512: 22, 20.7 with 8, 23, 24.3
//          with 10
//   many   5 rows of 32 / 8 heads of 128: 20.4, 20.6 with 48, 21.5, 21.8 with 56 (32 rows 25, 21.9 and 26,
//          23); 96 of 4 / 1 heads of 256: 28.8, 26 with 48; 100 of 8 / 1 heads of 512: 30.4, 27.9 with 12
int whole_tiles(int head_dim, int64_t items, int num_cus) {
  const bool few = items * 8 < num_cus;
  return head_dim <= 128 ? (few ? 32 : 48) : head_dim <= 256 ? (few ? 28 : 48) : few ? 8 : 12;
}

// Growing a buffer of a call that may be captured.
nva_status reserve_for(nva_ctx *ctx, DevBuf &buf, size_t bytes, bool capturing, const char *what) {
  if (capturing) {
    if (buf.cap < bytes)
      return fail(ctx, NVA_E_ARG,
                  "a captured step must not be larger than every earlier one: run it once before the "
                  "capture");
    buf.captured = true;
    return NVA_OK;
  }
  HIP_TRY(ctx, buf.reserve(bytes), what);
  return NVA_OK;
}

}  // namespace

namespace nva {

// What attention4_rows could not serve (but for work areas under capture), before a fused call rotates.
nva_status check_forward4(nva_ctx *ctx, nva_kv4 *kv, const nva_attn_desc *desc, int num_tokens) {
  nva_status st = check_desc(ctx, desc);
  if (st != NVA_OK) return st;
  if (!kv) return fail(ctx, NVA_E_NO_ARENA, "KV cache arena not bound in Context");
  if (kv->ctx != ctx) return fail(ctx, NVA_E_ARG, "KV arena belongs to another context");
  const int layer = desc->kv_layer_index;
  st = check_layer(kv, layer);
  if (st != NVA_OK) return st;
  if (num_tokens < 0) return fail(ctx, NVA_E_ARG, "num_tokens < 0");
  if (!kv->pages[layer])
    return fail(ctx, NVA_E_ARG, "layer %d has no pages to attend over", layer);
  if (kv->head_dims[layer] != desc->head_dim || kv->num_kv_heads != desc->num_kv_heads)
    return fail(ctx, NVA_E_ARG, "layer %d pages are [.., %d, %d], attention wants [.., %d, %d]",
                layer, kv->num_kv_heads, kv->head_dims[layer], desc->num_kv_heads,
                desc->head_dim);
  if ((int64_t)num_tokens * desc->num_heads > INT32_MAX / 2)
    return fail(ctx, NVA_E_UNSUPPORTED, "%d tokens of %d heads", num_tokens, desc->num_heads);
  if (const nva_tables *t = ctx->dev_step) {
    if (t->block_size != kv->block_size || t->max_page >= kv->num_blocks)
      return fail(ctx, NVA_E_ARG,
                  "tables of blocks of %d up to block %d, but the arena has %d blocks of %d",
                  t->block_size, t->max_page, kv->num_blocks, kv->block_size);
    if (num_tokens != ctx->dev_tokens && num_tokens != 0)
      return fail(ctx, NVA_E_ARG, "%d tokens but the step has %d", num_tokens, ctx->dev_tokens);
    return NVA_OK;
  }
  if (!ctx->has_step) return fail(ctx, NVA_E_NO_STEP, "no step metadata set on the context");
  if (!ctx->is_prefill) {
    if (!ctx->has_ctx_lens || !ctx->has_tables)
      return fail(ctx, NVA_E_ARG, "decode needs context lengths and block tables");
    if (num_tokens > ctx->num_seqs)
      return fail(ctx, NVA_E_ARG, "decode has %d rows but %d context lengths", num_tokens,
                  ctx->num_seqs);
  } else {
    if (!ctx->has_cu) return fail(ctx, NVA_E_ARG, "prefill needs cu_seqlens");
    if (!ctx->has_tables)
      return fail(ctx, NVA_E_ARG, "attention over the 4-bit arena needs block tables");
    if (num_tokens > 0 && ctx->cu_q[ctx->num_seqs] > num_tokens)
      return fail(ctx, NVA_E_ARG, "cu_seqlens end at row %d of %d", ctx->cu_q[ctx->num_seqs],
                  num_tokens);
  }
  if (num_tokens == 0) return NVA_OK;
  if (stream_capturing(ctx->stream))
    return fail(ctx, NVA_E_ARG,
                "only steps of nva_step_extend may be captured over the 4-bit arena");
  if (stores(ctx, *desc, num_tokens) && ctx->slot_max >= (int64_t)kv->num_blocks * kv->block_size)
    return fail(ctx, NVA_E_ARG, "slot %lld outside the arena's %lld slots", (long long)ctx->slot_max,
                (long long)kv->num_blocks * kv->block_size);
  return check_tables4(ctx, kv, num_tokens);
}

nva_status attention4_rows(nva_ctx *ctx, nva_kv4 *kv, const nva_attn_desc &d, const float *q,
                           const float *k, const float *v, int num_tokens, float *out) {
  const nva_tables *dev = ctx->dev_step;
  const int layer = d.kv_layer_index, rep = d.num_heads / d.num_kv_heads;
  const bool capturing = stream_capturing(ctx->stream);
  const bool store = stores(ctx, d, num_tokens);
  if (store && (!k || !v)) return fail(ctx, NVA_E_ARG, "k and v are required to store");

  // The kernels: sequences of up to 16 columns on the first list, of more on the second.  What the host
  // knows of their rows bounds them: the lengths themselves, or the most tokens that follow.
  const int seqs = dev ? ctx->dev_seqs : ctx->is_prefill ? ctx->num_seqs : num_tokens;
  int64_t few = 0, many = 0;  // most columns of a sequence on either list
  int64_t whole = 0;          // key tiles of decode rows that are short enough for one workgroup a KV head
  int64_t limit = kv4_by_dims(d.head_dim) ? INT32_MAX : 16;
  auto count = [&](int64_t cols) {
    if (cols <= limit) few = std::max(few, cols); else many = std::max(many, cols);
  };
  if (dev) {
    const int64_t most = (int64_t)std::min(ctx->dev_max_new, num_tokens) * rep;
    if (most > limit) many = most;
    few = std::min(most, limit);
  } else if (ctx->is_prefill) {
    int64_t units = 0;  // key tiles of the sequences of few columns
    for (int b = 0; b < seqs; b++) {
      const int64_t cols = (int64_t)(ctx->cu_q[b + 1] - ctx->cu_q[b]) * rep;
      count(cols);
      if (cols > 0 && cols <= limit)
        units += (int64_t)((ctx->cu_k[b + 1] - ctx->cu_k[b] + 31) / 32) * d.num_kv_heads;
    }
    // A few of them among others join those: the tile kernel takes some 6.5 ns for a key tile of one column
    // tile and head, the kernels of few columns 0.9 and the 20 us of two more launches.
    if (many && units <= kJoinUnits) {
      limit = 0;
      few = 0;
    }
  } else {
    count(rep);
    int64_t most = 0;  // keys that a row sees, and those before them in its first tile
    int least = INT32_MAX;
    for (int b = 0; b < seqs; b++) {
      most = std::max<int64_t>(most, ctx->ctx_lens[b]);
      least = std::min(least, ctx->ctx_lens[b]);
    }
    if (d.sliding_window > 0) most = std::min(most, (int64_t)d.sliding_window + 31);
    if (least > 0 && !many) whole = (most + 31) / 32;
  }
  struct Run {
    int mode, workgroups, tiles;
    size_t off_head, off_tiles, off_cum, off_before, off_borders, off_part, parts;
  } runs[2];
  int n_runs = 0;
  size_t plan_bytes = 0, part_floats = 0;
  auto add = [&](int mode) {
    Run &r = runs[n_runs++];
    r.mode = mode;
    r.workgroups = ctx->num_cus * ctx_kv4_workgroups_per_cu(ctx, d.head_dim, mode);
    const int cols = kv4_cols(d.head_dim, mode);
    const int64_t tiles = (int64_t)num_tokens * rep / cols + seqs + 1;
    r.tiles = (int)tiles;
    r.off_head = plan_bytes;
    r.off_tiles = r.off_head + 256;
    r.off_cum = align256(r.off_tiles + tiles * sizeof(Kv4Tile));
    r.off_before = align256(r.off_cum + (tiles + 1) * 8);
    r.off_borders = align256(r.off_before + ((size_t)seqs + 1) * 4);
    plan_bytes = align256(r.off_borders + r.workgroups * sizeof(Kv4Border));
    r.parts = (size_t)2 * r.workgroups * cols;
    r.off_part = part_floats;
    part_floats += r.parts * (d.head_dim + 2);
  };
  if (many) add(KV4_TILES);
  // (One list at least: it knows the rows that no sequence covers.)
  if (few || !many)
    add(kv4_by_dims(d.head_dim) ? KV4_DIMS : few <= 4 ? KV4_FEW : few <= 8 ? KV4_EIGHT : KV4_ROWS);
  if (whole) {  // a workgroup for every column tile and KV head, by a list that gives them one each
    const int cols = kv4_cols(d.head_dim, runs[0].mode);
    const int64_t tiles = (int64_t)seqs * ((rep + cols - 1) / cols), items = tiles * d.num_kv_heads;
    if (tiles > kKv4ListTiles || items > runs[0].workgroups ||
        whole > whole_tiles(d.head_dim, items, ctx->num_cus))
      whole = 0;
  }
  nva_status st = reserve_for(ctx, ctx->d_plan4, plan_bytes, capturing, "attention work list");
  if (st != NVA_OK) return st;
  st = reserve_for(ctx, ctx->d_part4, part_floats * 4, capturing, "attention partials");
  if (st != NVA_OK) return st;
  char *plan = static_cast<char *>(ctx->d_plan4.ptr);

  Kv4Store s{};
  s.kv = view_of(kv, layer);
  s.k = store ? k : nullptr;
  s.v = v;
  s.slots = dev ? dev->slots : ctx->dev_i32(ctx->off_slots);
  s.tokens = num_tokens;
  s.lists = n_runs;
  Kv4Attention a{};
  a.kv = s.kv;
  a.q = q;
  a.out = out;
  Kv4List rows{};
  if (dev) {
    rows.cu_q = dev->cu_q;
    rows.lens = dev->lens;
  } else if (ctx->is_prefill) {
    rows.cu_q = ctx->dev_i32(ctx->off_cu_q);
    rows.cu_k = ctx->dev_i32(ctx->off_cu_k);
  } else {
    rows.lens = ctx->dev_i32(ctx->off_ctx);
  }
  a.table = dev ? dev->table : ctx->dev_i32(ctx->off_tables);
  a.bt_stride = dev ? dev->width : ctx->bt_stride;
  a.hq = d.num_heads;
  a.head_dim = d.head_dim;
  a.window = d.sliding_window;
  a.tokens = num_tokens;
  a.tile_shift = shift_of(kv->block_size / 32);
  a.scale2 = (float)((double)d.scale * 1.4426950408889634074);
  for (int i = 0; i < n_runs; i++) {
    const Run &r = runs[i];
    Kv4List &l = s.list[i];
    l.head = reinterpret_cast<Kv4Head *>(plan + r.off_head);
    l.tiles = reinterpret_cast<Kv4Tile *>(plan + r.off_tiles);
    l.cum = reinterpret_cast<int64_t *>(plan + r.off_cum);
    l.before = reinterpret_cast<int32_t *>(plan + r.off_before);
    l.cu_q = rows.cu_q;
    l.cu_k = rows.cu_k;
    l.lens = rows.lens;
    l.num_seqs = seqs;
    l.rep = rep;
    l.hkv = d.num_kv_heads;
    l.window = d.sliding_window;
    l.workgroups = r.workgroups;
    l.cols = kv4_cols(d.head_dim, r.mode);
    l.min_cols = r.mode == KV4_TILES ? (int)limit + 1 : 1;
    l.max_cols = r.mode == KV4_TILES ? INT32_MAX : (int)limit;
    l.one_each = n_runs == 1 && std::max(few, many) <= l.cols;
    l.unit = r.mode == KV4_TILES || r.mode == KV4_DIMS ? 1 : 4;
    l.min_units = std::max(4, (int)(whole + 3) / 4 * 4);
    l.slack = r.mode == KV4_TILES ? 0 : 12;
    l.over = r.mode == KV4_TILES ? 4 : r.mode == KV4_DIMS ? 6 : 20;
  }
  {
    Timed tm(ctx, "store4");
    HIP_TRY(ctx, launch_kv4_store(s, d.head_dim, ctx->stream), "4-bit store kernel launch");
    tm.done();
  }
  for (int i = 0; i < n_runs; i++) {
    const Run &r = runs[i];
    a.head = s.list[i].head;
    a.tiles = s.list[i].tiles;
    a.cum = s.list[i].cum;
    a.room = r.tiles;
    a.borders = reinterpret_cast<Kv4Border *>(plan + r.off_borders);
    float *part = static_cast<float *>(ctx->d_part4.ptr) + r.off_part;
    a.part_m = part;
    a.part_l = part + r.parts;
    a.part_o = part + 2 * r.parts;
    a.zero_rest = i == 0;
    Timed tm(ctx, "attention4");
    HIP_TRY(ctx, launch_kv4_attention(a, r.mode, r.workgroups, ctx->stream),
            "4-bit attention kernel launch");
    tm.done();
    if (whole) continue;  // every row has keys and one segment: nothing to join, none to zero
    Timed tg(ctx, "merge4");
    const int64_t items = (int64_t)std::min(seqs, num_tokens) * d.num_kv_heads;
    HIP_TRY(ctx, launch_kv4_merge(a, r.mode, r.workgroups, (int)std::min<int64_t>(items, INT32_MAX),
                                  ctx->stream),
            "4-bit merge kernel launch");
    tg.done();
  }
  return NVA_OK;
}

}  // namespace nva

extern "C" {

// ------------------------------------------------------------------------------- RoPE

nva_status nva_rope_create_scaled(nva_ctx *ctx, const nva_rope_desc *desc, nva_rope **out) try {
  if (!ctx || !out) return NVA_E_ARG;
  *out = nullptr;
  if (!desc) return fail(ctx, NVA_E_ARG, "RoPE descriptor is null");
  DeviceGuard dg(ctx);
  nva_status st = check_rope(ctx, *desc);
  if (st != NVA_OK) return st;
  std::vector<double> f;
  const double amplitude = frequencies(*desc, f);
  std::unique_ptr<nva_rope> r(new nva_rope());
  r->ctx = ctx;
  r->max_pos = desc->max_pos;
  r->head_size = desc->head_size;
  r->rotary_dim = desc->rotary_dim;
  r->interleaved = desc->interleaved != 0;
  void *table = nullptr, *freq = nullptr;
  hipError_t e = hipMalloc(&table, (size_t)desc->max_pos * desc->rotary_dim * 4);
  if (e == hipSuccess) e = hipMalloc(&freq, f.size() * sizeof(double));
  if (e == hipSuccess)
    e = hipMemcpy(freq, f.data(), f.size() * sizeof(double), hipMemcpyHostToDevice);
  if (e == hipSuccess)
    e = launch_rope_table(static_cast<double *>(freq), static_cast<float *>(table),
                          (int)f.size(), desc->max_pos, amplitude, ctx->stream);
  // The frequencies are freed here, and a table is used on whichever stream comes next.
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (freq) (void)hipFree(freq);
  if (e != hipSuccess) {
    if (table) (void)hipFree(table);
    return hip_fail(ctx, e, "RoPE table");
  }
  r->table = static_cast<float *>(table);
  *out = r.release();
  return NVA_OK;
} catch (const std::exception &) {
  return no_memory(ctx);
}

// ------------------------------------------------------------------------------- tables

static TablesLaunch launch_of(const nva_tables *t) {
  TablesLaunch a{};
  a.table = t->table;
  a.lens = t->lens;
  a.free_pages = t->free_pages;
  a.slots = t->slots;
  a.positions = t->positions;
  a.cu_q = t->cu_q;
  a.state = t->state;
  a.block_size = t->block_size;
  a.width = t->width;
  a.max_tokens = t->max_tokens;
  return a;
}

nva_status nva_tables_create(nva_ctx *ctx, int max_seqs, int max_tokens, int max_step_tokens,
                             int num_blocks, int block_size, const int32_t *pages,
                             nva_tables **out) try {
  if (!ctx || !out) return NVA_E_ARG;
  *out = nullptr;
  DeviceGuard dg(ctx);
  if (max_seqs <= 0 || max_tokens <= 0 || max_step_tokens < 0 || num_blocks <= 0 || block_size <= 0)
    return fail(ctx, NVA_E_ARG, "tables need maxSeqs, maxTokens, numBlocks and blockSize > 0");
  if (max_seqs > kTablesMaxSeqs)
    return fail(ctx, NVA_E_UNSUPPORTED, "tables hold at most %d sequences (got %d)", kTablesMaxSeqs,
                max_seqs);
  if (max_tokens > INT32_MAX - 8192)
    return fail(ctx, NVA_E_UNSUPPORTED, "tables of %d tokens a sequence", max_tokens);
  int max_page = num_blocks - 1;
  if (pages) {
    std::vector<int32_t> sorted(pages, pages + num_blocks);
    std::sort(sorted.begin(), sorted.end());
    if (sorted[0] < 0 ||
        std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
      return fail(ctx, NVA_E_ARG, "the block ids handed out must be distinct and >= 0");
    max_page = sorted.back();
  }
  if (((int64_t)max_page + 1) * block_size > INT32_MAX)
    return fail(ctx, NVA_E_UNSUPPORTED, "slots of block %d of %d tokens pass 32 bits", max_page,
                block_size);
  std::unique_ptr<nva_tables> t(new nva_tables());
  t->ctx = ctx;
  t->max_seqs = max_seqs;
  t->max_tokens = max_tokens;
  t->max_step_tokens = max_step_tokens;
  t->num_pages = num_blocks;
  t->block_size = block_size;
  t->width = (int)(((int64_t)max_tokens + block_size - 1) / block_size);
  t->max_page = max_page;
  size_t off = 0;
  auto place = [&](size_t entries) {
    const size_t at = off;
    off = align256(off + entries * 4);
    return at;
  };
  const size_t table = place((size_t)max_seqs * t->width), lens = place(max_seqs);
  const size_t free_pages = place(num_blocks), slots = place(max_step_tokens);
  const size_t positions = place(max_step_tokens), cu_q = place((size_t)max_seqs + 1);
  const size_t state = place(4), staged = place(pages ? num_blocks : 0);
  void *p = nullptr;
  HIP_TRY(ctx, hipMalloc(&p, off), "block tables");
  char *m = t->memory = static_cast<char *>(p);
  auto at = [&](size_t o) { return reinterpret_cast<int32_t *>(m + o); };
  t->table = at(table);
  t->lens = at(lens);
  t->free_pages = at(free_pages);
  t->slots = at(slots);
  t->positions = at(positions);
  t->cu_q = at(cu_q);
  t->state = at(state);
  hipError_t e = pages ? hipMemcpy(m + staged, pages, (size_t)num_blocks * 4, hipMemcpyHostToDevice)
                       : hipSuccess;
  if (e == hipSuccess)
    e = launch_tables_clear(launch_of(t.get()), pages ? at(staged) : nullptr, num_blocks, max_seqs,
                            max_step_tokens, ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    (void)hipFree(p);
    return hip_fail(ctx, e, "block tables");
  }
  *out = t.release();
  return NVA_OK;
} catch (const std::exception &) {
  return no_memory(ctx);
}

nva_status nva_tables_destroy(nva_tables *tables) {
  if (!tables) return NVA_OK;
  if (nva_ctx *ctx = tables->ctx) {
    if (ctx->dev_step == tables) ctx->dev_step = nullptr;
    (void)hipStreamSynchronize(ctx->stream);
  }
  (void)hipFree(tables->memory);
  delete tables;
  return NVA_OK;
}

nva_status nva_tables_array(nva_tables *t, int which, void **ptr, int64_t *count) {
  if (!t) return NVA_E_ARG;
  int32_t *p = nullptr;
  int64_t n = 0;
  switch (which) {
    case NVA_TABLES_BLOCKS: p = t->table, n = (int64_t)t->max_seqs * t->width; break;
    case NVA_TABLES_LENS: p = t->lens, n = t->max_seqs; break;
    case NVA_TABLES_SLOTS: p = t->slots, n = t->max_step_tokens; break;
    case NVA_TABLES_POSITIONS: p = t->positions, n = t->max_step_tokens; break;
    case NVA_TABLES_CU_Q: p = t->cu_q, n = (int64_t)t->max_seqs + 1; break;
    default: return fail(t->ctx, NVA_E_ARG, "no array %d", which);
  }
  if (ptr) *ptr = p;
  if (count) *count = n;
  return NVA_OK;
}

nva_status nva_tables_status(nva_tables *t, int32_t *status) {
  if (!t || !status) return NVA_E_ARG;
  nva_ctx *ctx = t->ctx;
  DeviceGuard dg(ctx);
  if (stream_capturing(ctx->stream))  // (waiting would end the capture)
    return fail(ctx, NVA_E_ARG, "the status of tables is not for a captured step");
  HIP_TRY(ctx, hipStreamSynchronize(ctx->stream), "stream synchronize");
  HIP_TRY(ctx, hipMemcpy(status, t->state, 12, hipMemcpyDeviceToHost), "tables status");
  return NVA_OK;
}

nva_status nva_step_extend(nva_ctx *ctx, nva_tables *t, const int32_t *keep,
                           const int32_t *new_tokens, int num_seqs, int num_tokens, int max_new) {
  if (!ctx) return NVA_E_ARG;
  DeviceGuard dg(ctx);
  if (!t) return fail(ctx, NVA_E_ARG, "block tables are null");
  if (t->ctx != ctx) return fail(ctx, NVA_E_ARG, "block tables belong to another context");
  if (num_seqs < 0 || num_seqs > t->max_seqs)
    return fail(ctx, NVA_E_ARG, "%d sequences of at most %d", num_seqs, t->max_seqs);
  if (num_tokens < 0 || num_tokens > t->max_step_tokens)
    return fail(ctx, NVA_E_ARG, "%d tokens in a step of at most %d", num_tokens, t->max_step_tokens);
  if (max_new < 0) return fail(ctx, NVA_E_ARG, "max_new < 0");
  if (num_seqs > 0 && !new_tokens) return fail(ctx, NVA_E_ARG, "new_tokens are required");
  TablesLaunch a = launch_of(t);
  a.keep = keep;
  a.fresh = new_tokens;
  a.num_seqs = num_seqs;
  a.num_tokens = num_tokens;
  a.max_new = max_new;
  ctx->has_step = false;
  ctx->dev_step = nullptr;
  Timed tm(ctx, "tables");
  HIP_TRY(ctx, launch_tables_extend(a, ctx->stream), "block tables kernel launch");
  tm.done();
  for (Plan *p : ctx->plans) p->valid = false;
  ctx->tile_choices.clear();
  ctx->groups.clear();
  ctx->has_encoder = false;
  ctx->dev_step = t;
  ctx->dev_seqs = num_seqs;
  ctx->dev_tokens = num_tokens;
  ctx->dev_max_new = max_new;
  return NVA_OK;
}

// ------------------------------------------------------------------------------- 4-bit arena

nva_status nva_quantize4(nva_ctx *ctx, const float *x, int64_t rows, int n, uint8_t *codes,
                         uint8_t *scales) {
  if (!ctx) return NVA_E_ARG;
  DeviceGuard dg(ctx);
  if (rows < 0 || n <= 0) return fail(ctx, NVA_E_ARG, "bad shape [%lld, %d]", (long long)rows, n);
  if (n % 32) return fail(ctx, NVA_E_UNSUPPORTED, "4-bit rows need n %% 32 == 0 (got %d)", n);
  if (rows == 0) return NVA_OK;
  if (rows > ((int64_t)1 << 46) / n)
    return fail(ctx, NVA_E_UNSUPPORTED, "%lld rows of %d values", (long long)rows, n);
  if (!x || !codes || !scales) return fail(ctx, NVA_E_ARG, "x, codes and scales are required");
  if (!aligned16(x) || (reinterpret_cast<uintptr_t>(codes) & 3u))
    return fail(ctx, NVA_E_ARG, "x must be 16-byte and codes 4-byte aligned");
  Timed tm(ctx, "quantize4");
  HIP_TRY(ctx, launch_quantize4(x, rows * n, codes, scales, ctx->stream), "quantize kernel launch");
  tm.done();
  return NVA_OK;
}

nva_status nva_kv4_create(nva_ctx *ctx, int num_layers, int num_blocks, int block_size,
                          int num_kv_heads, const int32_t *head_dims, const uint8_t *allocate,
                          nva_kv4 **out) try {
  if (!ctx || !out) return NVA_E_ARG;
  DeviceGuard dg(ctx);
  *out = nullptr;
  if (num_blocks <= 0) return fail(ctx, NVA_E_ARG, "numBlocks must be > 0");
  nva_status st = check_arena4(ctx, num_layers, block_size, num_kv_heads, head_dims, allocate);
  if (st != NVA_OK) return st;
  std::unique_ptr<nva_kv4> kv(new nva_kv4());
  kv->ctx = ctx;
  kv->num_layers = num_layers;
  kv->num_blocks = num_blocks;
  kv->block_size = block_size;
  kv->num_kv_heads = num_kv_heads;
  kv->head_dims.assign(head_dims, head_dims + num_layers);
  kv->pages.assign(num_layers, nullptr);
  kv->bytes.assign(num_layers, 0);
  hipError_t e = hipSuccess;
  for (int i = 0; i < num_layers && e == hipSuccess; i++) {
    if (allocate && !allocate[i]) continue;
    const int64_t bytes = num_blocks * kv4_block_bytes(block_size, num_kv_heads, head_dims[i]);
    void *p = nullptr;
    e = hipMalloc(&p, bytes);
    if (e != hipSuccess) break;
    kv->pages[i] = static_cast<uint8_t *>(p);
    kv->bytes[i] = bytes;
    e = hipMemsetAsync(p, 0, bytes, ctx->stream);
  }
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    const nva_status failed = hip_fail(ctx, e, "4-bit KV arena allocation");
    nva_kv4_destroy(kv.release());
    return failed;
  }
  *out = kv.release();
  return NVA_OK;
} catch (const std::exception &) {
  return no_memory(ctx);
}

nva_status nva_kv4_destroy(nva_kv4 *kv) {
  if (!kv) return NVA_OK;
  if (kv->ctx) (void)hipStreamSynchronize(kv->ctx->stream);
  for (uint8_t *p : kv->pages)
    if (p) (void)hipFree(p);
  delete kv;
  return NVA_OK;
}

nva_status nva_kv4_blocks_that_fit(nva_ctx *ctx, int num_layers, int block_size, int num_kv_heads,
                                   const int32_t *head_dims, const uint8_t *allocate,
                                   float fraction, int *blocks, int64_t *free_bytes) {
  if (!ctx || !blocks) return NVA_E_ARG;
  DeviceGuard dg(ctx);
  nva_status st = check_arena4(ctx, num_layers, block_size, num_kv_heads, head_dims, allocate);
  if (st != NVA_OK) return st;
  if (!(fraction > 0.0f && fraction <= 1.0f))
    return fail(ctx, NVA_E_ARG, "kvHeapFraction must be in (0, 1], got %g", (double)fraction);
  int64_t per_block = 0;
  for (int i = 0; i < num_layers; i++)
    if (!allocate || allocate[i])
      per_block += kv4_block_bytes(block_size, num_kv_heads, head_dims[i]);
  if (per_block <= 0) return fail(ctx, NVA_E_ARG, "no layer gets pages");
  size_t free_b = 0, total_b = 0;
  HIP_TRY(ctx, hipMemGetInfo(&free_b, &total_b), "device memory query");
  const int64_t cap = std::max<int64_t>(32, (int64_t)((double)free_b * (double)fraction) / per_block);
  *blocks = (int)std::min<int64_t>(cap, INT32_MAX);
  if (free_bytes) *free_bytes = (int64_t)free_b;
  return NVA_OK;
}

nva_status nva_kv4_layer(nva_kv4 *kv, int layer, void **pages, int64_t *bytes) {
  if (!kv) return NVA_E_ARG;
  nva_status st = check_layer(kv, layer);
  if (st != NVA_OK) return st;
  if (pages) *pages = kv->pages[layer];
  if (bytes) *bytes = kv->bytes[layer];
  return NVA_OK;
}

// Checks of the calls over rows at slots; *done: there is nothing to do.
static nva_status check_rows4(nva_kv4 *kv, int layer, const int32_t *slots, const float *k,
                              const float *v, int num_rows, bool *done) {
  nva_ctx *ctx = kv->ctx;
  nva_status st = check_layer(kv, layer);
  if (st != NVA_OK) return st;
  if (!kv->pages[layer]) return fail(ctx, NVA_E_ARG, "layer %d has no pages", layer);
  if (num_rows < 0) return fail(ctx, NVA_E_ARG, "num_rows < 0");
  if ((int64_t)num_rows * kv->num_kv_heads > INT32_MAX / 2)
    return fail(ctx, NVA_E_UNSUPPORTED, "%d rows of %d heads", num_rows, kv->num_kv_heads);
  *done = num_rows == 0;
  if (*done) return NVA_OK;
  if (!slots) return fail(ctx, NVA_E_ARG, "slots are required");
  if ((k && !aligned16(k)) || (v && !aligned16(v)))
    return fail(ctx, NVA_E_ARG, "device pointers must be 16-byte aligned");
  return NVA_OK;
}

nva_status nva_kv4_write_rows(nva_kv4 *kv, int layer, const int32_t *slots, const float *k,
                              const float *v, int num_rows) {
  if (!kv) return NVA_E_ARG;
  nva_ctx *ctx = kv->ctx;
  DeviceGuard dg(ctx);
  bool done = false;
  nva_status st = check_rows4(kv, layer, slots, k, v, num_rows, &done);
  if (st != NVA_OK || done) return st;
  if (!k || !v) return fail(ctx, NVA_E_ARG, "k and v are required to store");
  Kv4Store s{};
  s.kv = view_of(kv, layer);
  s.k = k;
  s.v = v;
  s.slots = slots;
  s.tokens = num_rows;
  Timed tm(ctx, "store4");
  HIP_TRY(ctx, launch_kv4_store(s, kv->head_dims[layer], ctx->stream), "4-bit store kernel launch");
  tm.done();
  return NVA_OK;
}

nva_status nva_kv4_read_rows(nva_kv4 *kv, int layer, const int32_t *slots, float *k, float *v,
                             int num_rows) {
  if (!kv) return NVA_E_ARG;
  nva_ctx *ctx = kv->ctx;
  DeviceGuard dg(ctx);
  bool done = false;
  nva_status st = check_rows4(kv, layer, slots, k, v, num_rows, &done);
  if (st != NVA_OK || done) return st;
  Timed tm(ctx, "read4");
  HIP_TRY(ctx, launch_kv4_read(view_of(kv, layer), kv->head_dims[layer], slots, k, v, num_rows,
                               ctx->stream),
          "4-bit read kernel launch");
  tm.done();
  return NVA_OK;
}

nva_status nva_attention4_forward(nva_ctx *ctx, nva_kv4 *kv, const nva_attn_desc *desc,
                                  const float *q, const float *k, const float *v, int num_tokens,
                                  float *out) try {
  if (!ctx) return NVA_E_ARG;
  DeviceGuard dg(ctx);
  nva_status st = check_forward4(ctx, kv, desc, num_tokens);
  if (st != NVA_OK) return st;
  if (num_tokens == 0) return NVA_OK;
  if (!q || !out) return fail(ctx, NVA_E_ARG, "q and out are required");
  if (!aligned16(q) || !aligned16(out) || (k && !aligned16(k)) || (v && !aligned16(v)))
    return fail(ctx, NVA_E_ARG, "device pointers must be 16-byte aligned");
  return attention4_rows(ctx, kv, *desc, q, k, v, num_tokens, out);
} catch (const std::exception &) {
  return no_memory(ctx);
}

// ------------------------------------------------------------------------------- 4-bit projections

nva_status nva_linear4_create(nva_ctx *ctx, const uint8_t *codes, const uint8_t *scales, int out,
                              int in, nva_linear4 **linear) try {
  if (!ctx || !linear) return NVA_E_ARG;
  *linear = nullptr;
  DeviceGuard dg(ctx);
  if (in <= 0 || out <= 0) return fail(ctx, NVA_E_ARG, "bad linear shape in=%d out=%d", in, out);
  if (in % 32) return fail(ctx, NVA_E_UNSUPPORTED, "4-bit linear needs in %% 32 == 0 (got %d)", in);
  if (in >= (1 << 22))
    return fail(ctx, NVA_E_UNSUPPORTED, "linear needs in < 4194304 (got %d)", in);
  // A launch's threads are counted in 32 bits: a thread a lane of 16 x 128 tiles lays out, and up to 1024 a tile
  // of outs multiply.
  const int64_t out_tiles = ((int64_t)out + 15) / 16, in_tiles = ((int64_t)in + 127) / 128;
  if (out_tiles >= 1 << 22 || out_tiles * in_tiles >= 1 << 26)
    return fail(ctx, NVA_E_UNSUPPORTED, "4-bit linear of in=%d out=%d", in, out);
  if (!codes || !scales) return fail(ctx, NVA_E_ARG, "codes and scales are required");
  std::unique_ptr<nva_linear4> l(new nva_linear4());
  l->device = ctx->device;
  l->in = in;
  l->out = out;
  void *p = nullptr;
  HIP_TRY(ctx, hipMalloc(&p, linear4_bytes(out, in)), "4-bit weight");
  hipError_t e = launch_linear4_layout(codes, scales, out, in, static_cast<uint8_t *>(p), ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    (void)hipFree(p);
    return hip_fail(ctx, e, "4-bit weight layout");
  }
  l->weight = static_cast<uint8_t *>(p);
  *linear = l.release();
  return NVA_OK;
} catch (const std::exception &) {
  return no_memory(ctx);
}

nva_status nva_linear4_destroy(nva_linear4 *linear) {
  if (!linear) return NVA_OK;
  (void)hipFree(linear->weight);  // (waits for the device)
  delete linear;
  return NVA_OK;
}

nva_status nva_linear4_forward(nva_ctx *ctx, const nva_linear4 *l, const float *x, int rows,
                               const float *bias, float *y) try {
  if (!ctx) return NVA_E_ARG;
  DeviceGuard dg(ctx);
  if (!l) return fail(ctx, NVA_E_ARG, "4-bit linear is null");
  if (l->device != ctx->device)
    return fail(ctx, NVA_E_ARG, "4-bit linear belongs to another device");
  if (rows < 0) return fail(ctx, NVA_E_ARG, "rows < 0");
  if (rows == 0) return NVA_OK;
  if (rows > INT32_MAX - 128) return fail(ctx, NVA_E_UNSUPPORTED, "4-bit linear of %d rows", rows);
  if (!x || !y) return fail(ctx, NVA_E_ARG, "x and y are required");
  if (!aligned16(x)) return fail(ctx, NVA_E_ARG, "x must be a 16-byte aligned device pointer");
  Linear4Launch a{};
  a.weight = l->weight;
  a.bias = bias;
  a.in = l->in;
  a.out = l->out;
  // Rows at a time: the parts of x, half as large again as x, stay within bounds.
  constexpr int kRows = 16384;
  a.rows = std::min(rows, kRows);
  // (The last rows may be few, whose work area is another.)
  Linear4Launch rest = a;
  rest.rows = rows % kRows;
  size_t work = linear4_work_bytes(a, ctx->num_cus);
  if (rest.rows) work = std::max(work, linear4_work_bytes(rest, ctx->num_cus));
  if (work) {
    nva_status st = reserve_for(ctx, ctx->d_lin4, work, stream_capturing(ctx->stream),
                                "4-bit linear work area");
    if (st != NVA_OK) return st;
    a.work = ctx->d_lin4.ptr;
  }
  Timed tm(ctx, "linear4");
  for (int r = 0; r < rows; r += a.rows) {
    a.rows = std::min(rows - r, kRows);
    a.x = x + (size_t)r * l->in;
    a.y = y + (size_t)r * l->out;
    HIP_TRY(ctx, launch_linear4(a, ctx->num_cus, ctx->stream), "4-bit linear kernel launch");
  }
  tm.done();
  return NVA_OK;
} catch (const std::exception &) {
  return no_memory(ctx);
}

}  // extern "C"
