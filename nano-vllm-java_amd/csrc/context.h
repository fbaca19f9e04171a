// The context behind the C ABI and what its entry points share: grow-only buffers, work plans, error
// reporting, the device guard and kernel timing.  Included by the host sources that implement
// include/nva.h.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <chrono>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <map>
#include <string>
#include <vector>

#include "../../include/nva.h"
#include "nva_internal.h"

namespace nva {

inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }


// Grow-only device buffer.  One that a captured graph may hold (`captured`) is kept when it is
// replaced by a larger one, as the graph's replays go on using it.
struct DevBuf {
  void *ptr = nullptr;
  size_t cap = 0;
  bool captured = false;
  std::vector<void *> kept;
  hipError_t reserve(size_t bytes) {
    if (bytes <= cap) return hipSuccess;
    if (ptr && captured) {
      kept.push_back(ptr);  // (throws std::bad_alloc before anything changes)
    } else if (ptr) {
      hipError_t e = hipFree(ptr);
      if (e != hipSuccess) return e;
    }
    ptr = nullptr;
    cap = 0;
    captured = false;
    size_t want = std::max<size_t>(bytes, 4096);
    hipError_t e = hipMalloc(&ptr, want);
    if (e == hipSuccess) cap = want;
    return e;
  }
  void release() {
    if (ptr) (void)hipFree(ptr);
    for (void *p : kept) (void)hipFree(p);
    kept.clear();
    ptr = nullptr;
    cap = 0;
    captured = false;
  }
};

// Grow-only pinned host buffer whose last upload is tracked by an event, so it is only
// overwritten once the device has consumed it.
struct Staging {
  void *ptr = nullptr;
  size_t cap = 0;
  hipEvent_t done = nullptr;
  bool pending = false;
  hipError_t wait() {
    if (pending) {
      pending = false;
      return hipEventSynchronize(done);
    }
    return hipSuccess;
  }
  hipError_t reserve(size_t bytes) {
    hipError_t e = wait();
    if (e != hipSuccess) return e;
    if (!done) {
      e = hipEventCreateWithFlags(&done, hipEventDisableTiming);
      if (e != hipSuccess) return e;
    }
    if (bytes <= cap) return hipSuccess;
    if (ptr) (void)hipHostFree(ptr);
    ptr = nullptr;
    cap = 0;
    size_t want = std::max<size_t>(bytes, 4096);
    e = hipHostMalloc(&ptr, want, hipHostMallocDefault);
    if (e == hipSuccess) cap = want;
    return e;
  }
  hipError_t upload(DevBuf &dst, size_t bytes, hipStream_t s) {
    hipError_t e = hipMemcpyAsync(dst.ptr, ptr, bytes, hipMemcpyHostToDevice, s);
    if (e != hipSuccess) return e;
    e = hipEventRecord(done, s);
    if (e == hipSuccess) pending = true;
    return e;
  }
  void release() {
    if (pending) (void)hipEventSynchronize(done);
    pending = false;
    if (ptr) (void)hipHostFree(ptr);
    if (done) (void)hipEventDestroy(done);
    ptr = nullptr;
    done = nullptr;
    cap = 0;
  }
};

// A work plan: the flattened row / merge / tile lists for one attention configuration of the
// current step, built on the host and uploaded once, then reused by every layer with the same
// configuration.
struct PlanKey {
  int window, mfma, fp32_tiles, tile_q, wg_per_item, blocks_per_cu;
  int tile_groups;             // prefill grid height: KV heads x query-head groups
  int tokens;                  // rows of q / out in the forward call
  int paged;                   // keys through block tables (else dense k/v rows)
  int block_size, num_blocks;  // arena geometry the tables are checked against
  int head_dim, num_heads, num_kv_heads;  // size the work of a mixed plan's two kernels
  int cross = 0;               // over the encoder's rows instead of the sequence's own keys
  int64_t kv_rows = 0;         // cross: rows of the encoder pool
  int item_heads = 0;          // query heads of a column group of a span item (0: no span kernel)
  int split_tile_q = 0;        // queries of a split tile
  int tile_heads = 0;          // and of a span tile (0: no tile kernel for this head dim)
  int span_tile_cols = 0;      // columns of a span tile
  int span_blocks_per_cu = 0;
  bool operator==(const PlanKey &o) const {
    return cross == o.cross && kv_rows == o.kv_rows && item_heads == o.item_heads &&
           split_tile_q == o.split_tile_q && tile_heads == o.tile_heads &&
           span_tile_cols == o.span_tile_cols &&
           span_blocks_per_cu == o.span_blocks_per_cu && window == o.window && mfma == o.mfma &&
           fp32_tiles == o.fp32_tiles && tile_q == o.tile_q &&
           head_dim == o.head_dim && num_heads == o.num_heads && num_kv_heads == o.num_kv_heads &&
           wg_per_item == o.wg_per_item && blocks_per_cu == o.blocks_per_cu &&
           tile_groups == o.tile_groups && tokens == o.tokens && paged == o.paged &&
           block_size == o.block_size && num_blocks == o.num_blocks;
  }
};

struct Plan {
  PlanKey key{};
  bool valid = false;
  int num_rows = 0, num_merge = 0, num_tiles = 0, num_parts = 0;
  int num_slots = 0;  // prefill stream-K slots (grid x)
  int num_spans = 0, max_cols = 0;                // span items, and the most columns of one
  int num_span_tiles = 0, num_span_slots = 0;     // span tiles and their stream-K slots
  int max_parts = 0;  // most partials any merged row has
  bool beside = false;     // rows and items run on the side stream, beside the tiles
  bool covers_all = true;  // every output row is written by some kernel
  size_t off_rows = 0, off_merge = 0, off_tiles = 0, off_slots = 0;
  size_t off_spans = 0, off_span_tiles = 0, off_span_slots = 0, off_row_part = 0;
  std::vector<char> host;  // the packed lists at the offsets above
  uint64_t id = 0;         // unique per build (identifies the plan held in a scratch array)
  bool on_device = false;  // host bytes uploaded to dev
  DevBuf dev;
  Staging stage;
};

// Workspace of the no-allocation entry point: the plan, the split partials and the shared-KV
// gather rows of one call live in fixed regions of a device's static scratch array instead of
// the context's grow-only buffers.  base is that device's address of the array (from
// hipGetSymbolAddress), used == bytes already taken (gather rows, at the front).
struct Scratch {
  char *base = nullptr;
  size_t used = 0;
};

struct PendingTiming {
  const char *name, *variant;  // variant: null, or the second entry that counts it
  hipEvent_t start, stop;
};

// Which tile kernel a layer configuration's prefill runs on in the current step.
struct TileChoice {
  int head_dim, num_heads, num_kv_heads, window;
  int tile_heads;  // of its spans (0: no prefix is shared)
  bool fp32;
};

struct KernelStat {
  int64_t launches = 0;
  double ms = 0.0;
};

}  // namespace nva

using namespace nva;

struct nva_ctx {
  int device = 0;
  int num_cus = 256;
  hipStream_t own_stream = nullptr;
  hipStream_t side_stream = nullptr;  // decode rows of a mixed step run here, beside the tiles
  hipEvent_t fork_ev = nullptr, join_ev = nullptr;
  hipStream_t stream = nullptr;
  std::string err;

  // Step metadata (host copies) and its device mirror.
  bool has_step = false;
  bool is_prefill = false;
  int num_seqs = 0;
  int num_tokens = 0;
  int max_q = 0, max_k = 0;
  int bt_stride = 0;
  int num_slots = 0;
  int64_t slot_max = -1;  // largest slot of the step (negative slots are skipped)
  bool has_cu = false, has_slots = false, has_ctx_lens = false, has_tables = false,
       has_pos = false;
  std::vector<int32_t> cu_q, cu_k, slots, ctx_lens, tables, seq_ids, pos;
  // Shared prefixes of the step's sequences, and the page size their tables were compared at (0:
  // not yet).
  std::vector<nva_prefix_group> groups;
  int groups_block_size = 0;
  // The encoder rows each sequence's cross attention reads.
  bool has_encoder = false;
  std::vector<int32_t> enc_start, enc_len;
  DevBuf d_step;
  Staging step_stage;
  size_t off_cu_q = 0, off_cu_k = 0, off_slots = 0, off_ctx = 0, off_tables = 0, off_pos = 0;

  // The step's metadata built on the device, in place of the above (has_step is false then); its
  // arrays are those of the tables.
  const nva_tables *dev_step = nullptr;
  int dev_seqs = 0, dev_tokens = 0, dev_max_new = 0;
  // The arena geometry that the host step's tables were checked against for the 4-bit cache, and of how many
  // of its sequences.
  int checked_blocks = 0, checked_block_size = 0, checked_seqs = 0;

  std::vector<Plan *> plans;
  std::vector<TileChoice> tile_choices;
  DevBuf d_part;     // split partials
  DevBuf d_q_rot;    // fused path scratch for rotated q
  DevBuf d_k_rot;    // fused path scratch for rotated k
  DevBuf d_v_norm;   // fused path scratch for normalised v (dense prefill with a v norm)
  DevBuf d_lin;      // split-K partial sums of the linear kernel
  DevBuf d_gather;   // shared-KV gather [2, T, Hkv, d]
  DevBuf d_plan4;    // work lists of attention over the 4-bit cache
  DevBuf d_part4;    // and its partials
  DevBuf d_lin4;     // parts of x and partial sums of the 4-bit linear kernels

  // One word the store / RoPE kernel writes the XCD of its last workgroup to, read by the decode
  // launch that follows (null if its allocation failed: no rotation).
  int32_t *xcd_hint = nullptr;

  // This device's address of the no-allocation scratch array (null if the lookup failed).
  char *scratch = nullptr;
  hipError_t scratch_err = hipSuccess;

  // Prefill occupancy (resident workgroups per CU) by (head dim, heads per workgroup), queried
  // once on this context's device.
  std::map<int, int> occupancy;

  bool timing = false;
  std::vector<PendingTiming> pending;
  std::vector<hipEvent_t> event_pool;
  std::map<std::string, KernelStat> stats;

  const int32_t *dev_i32(size_t off) const {
    return reinterpret_cast<const int32_t *>(static_cast<char *>(d_step.ptr) + off);
  }
};

struct nva_kv {
  nva_ctx *ctx = nullptr;
  int num_layers = 0, num_blocks = 0, block_size = 0, num_kv_heads = 0;
  std::vector<int32_t> head_dims;
  std::vector<float *> k, v;
  std::vector<int64_t> bytes;
};

struct nva_rope {
  nva_ctx *ctx = nullptr;
  int max_pos = 0, head_size = 0;
  float *table = nullptr;  // [max_pos, rotary_dim]: cos, then sin
  int rotary_dim = 0;
  bool interleaved = false;
  // The layout of the reference's own table, which every kernel reads.
  bool plain() const { return rotary_dim == head_size && !interleaved; }
};

// Block tables that grow and shrink on the device.
struct nva_tables {
  nva_ctx *ctx = nullptr;
  int max_seqs = 0, max_tokens = 0, max_step_tokens = 0, num_pages = 0, block_size = 0, width = 0;
  int max_page = -1;  // largest block id it may hand out
  char *memory = nullptr;
  int32_t *table = nullptr, *lens = nullptr, *free_pages = nullptr, *slots = nullptr,
          *positions = nullptr, *cu_q = nullptr, *state = nullptr;
};

// A 4-bit weight, laid out for the matrix cores (linear4.hip).
struct nva_linear4 {
  int device = 0;  // any context of it may use the weight
  int in = 0, out = 0;
  uint8_t *weight = nullptr;
};

// The 4-bit arena: one buffer a layer (mx4.h: the form; kv4.hip: the layout).
struct nva_kv4 {
  nva_ctx *ctx = nullptr;
  int num_layers = 0, num_blocks = 0, block_size = 0, num_kv_heads = 0;
  std::vector<int32_t> head_dims;
  std::vector<uint8_t *> pages;
  std::vector<int64_t> bytes;
};

namespace nva {

inline nva_status fail(nva_ctx *ctx, nva_status st, const char *fmt, ...) {
  if (ctx) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    try {
      ctx->err = buf;
    } catch (const std::exception &) {  // no memory for the text
      ctx->err.clear();
    }
  }
  return st;
}

// Host memory ran out in an entry point (no exception may leave it).
inline nva_status no_memory(nva_ctx *ctx) {
  ctx->err = "out of memory";  // short: needs no allocation
  return NVA_E_OOM;
}

inline nva_status hip_fail(nva_ctx *ctx, hipError_t e, const char *what) {
  (void)hipGetLastError();  // reported here, it must not surface at a later launch check
  return fail(ctx, e == hipErrorOutOfMemory ? NVA_E_OOM : NVA_E_HIP, "%s: %s", what,
              hipGetErrorString(e));
}

#define HIP_TRY(ctx, expr, what)                \
  do {                                          \
    hipError_t e_ = (expr);                     \
    if (e_ != hipSuccess) return hip_fail(ctx, e_, what); \
  } while (0)

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Makes the context's device current for the scope of an entry point (its grow-only buffers
// are allocated, and its occupancy queried, on that device) and restores the caller's.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int device) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != device) (void)hipSetDevice(device);
  }
  explicit DeviceGuard(const nva_ctx *ctx) : DeviceGuard(ctx->device) {}
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
  }
};

inline int ctx_prefill_blocks_per_cu(nva_ctx *ctx, int head_dim, int hpw, bool fp32) {
  const int key = (head_dim * 16 + hpw) * 2 + (fp32 ? 1 : 0);
  auto it = ctx->occupancy.find(key);
  if (it != ctx->occupancy.end()) return it->second;
  const int n = fp32 ? prefill_fp32_blocks_per_cu(head_dim, hpw) : prefill_blocks_per_cu(head_dim, hpw);
  ctx->occupancy[key] = n;
  return n;
}

inline int ctx_span_blocks_per_cu(nva_ctx *ctx, int head_dim) {
  const int key = -head_dim;  // beside the prefill kernels' keys, which are positive
  auto it = ctx->occupancy.find(key);
  if (it == ctx->occupancy.end())
    it = ctx->occupancy.emplace(key, span_tile_blocks_per_cu(head_dim)).first;
  return it->second;
}

// Timings that find no host memory are dropped: the call they time is not to fail for them.
inline void give_event(nva_ctx *ctx, hipEvent_t e) {
  try {
    ctx->event_pool.push_back(e);
  } catch (const std::exception &) {
    (void)hipEventDestroy(e);
  }
}

inline void add_stat(nva_ctx *ctx, const char *name, double ms) {
  try {
    KernelStat &s = ctx->stats[name];
    s.launches++;
    s.ms += ms;
  } catch (const std::exception &) {
  }
}

inline hipEvent_t take_event(nva_ctx *ctx) {
  if (!ctx->event_pool.empty()) {
    hipEvent_t e = ctx->event_pool.back();
    ctx->event_pool.pop_back();
    return e;
  }
  hipEvent_t e = nullptr;
  if (hipEventCreate(&e) != hipSuccess) return nullptr;
  return e;
}

// Brackets one kernel launch with timing events when timing is on.  A launch that one of several
// kernels serves is counted under its own name (variant) too.
struct Timed {
  nva_ctx *ctx;
  const char *name, *variant;
  hipStream_t stream;
  hipEvent_t start = nullptr;
  Timed(nva_ctx *c, const char *n, hipStream_t s = nullptr, const char *v = nullptr)
      : ctx(c), name(n), variant(v), stream(s ? s : c->stream) {
    if (ctx->timing) {
      start = take_event(ctx);
      if (start) (void)hipEventRecord(start, stream);
    }
  }
  void done() {
    if (!start) return;
    hipEvent_t stop = take_event(ctx);
    if (!stop) return;
    (void)hipEventRecord(stop, stream);
    try {
      ctx->pending.push_back({name, variant, start, stop});
    } catch (const std::exception &) {
      give_event(ctx, start);
      give_event(ctx, stop);
    }
    start = nullptr;
  }
};

inline void resolve_timings(nva_ctx *ctx) {
  for (auto &p : ctx->pending) {
    float ms = 0.f;
    if (hipEventSynchronize(p.stop) == hipSuccess &&
        hipEventElapsedTime(&ms, p.start, p.stop) == hipSuccess) {
      for (const char *n : {p.name, p.variant})
        if (n) add_stat(ctx, n, ms);
    }
    give_event(ctx, p.start);
    give_event(ctx, p.stop);
  }
  ctx->pending.clear();
}

// Host time of one plan build (and its upload), kept as the "plan" entry of the kernel stats
// when timing is on: the per-step planning cost a scheduler step pays at its first layer.
struct HostTimed {
  nva_ctx *ctx;
  const char *name;
  std::chrono::steady_clock::time_point t0;
  bool on;
  HostTimed(nva_ctx *c, const char *n) : ctx(c), name(n), on(c->timing) {
    if (on) t0 = std::chrono::steady_clock::now();
  }
  ~HostTimed() {
    if (!on) return;
    const double ms =
        std::chrono::duration<double, std::milli>(std::chrono::steady_clock::now() - t0).count();
    add_stat(ctx, name, ms);
  }
};

inline nva_status check_desc(nva_ctx *ctx, const nva_attn_desc *d) {
  if (!d) return fail(ctx, NVA_E_ARG, "attention descriptor is null");
  if (d->num_heads <= 0 || d->num_kv_heads <= 0 || d->head_dim <= 0)
    return fail(ctx, NVA_E_ARG, "numHeads, numKvHeads and headDim must be > 0");
  if (d->num_heads % d->num_kv_heads)
    return fail(ctx, NVA_E_ARG, "numHeads %d is not a multiple of numKvHeads %d", d->num_heads,
                d->num_kv_heads);
  if (d->head_dim % 4) return fail(ctx, NVA_E_UNSUPPORTED, "headDim must be a multiple of 4");
  return NVA_OK;
}

inline bool stream_capturing(hipStream_t s) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(s, &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
}


// What norm_rope_attention hands to either cache's attention: the rotated q and k and the v rows.
nva_status attention4_rows(nva_ctx *ctx, nva_kv4 *kv, const nva_attn_desc &d, const float *q,
                           const float *k, const float *v, int num_tokens, float *out);
nva_status check_forward4(nva_ctx *ctx, nva_kv4 *kv, const nva_attn_desc *desc, int num_tokens);

}  // namespace nva
