// extern "C" entry points around positions and the K/V cache (declared in
// include/flexatt.h): argument checks, then the kernel launchers.
#include <math.h>
#include <stdint.h>

#include "../../include/flexatt.h"
#include "capi_checks.h"
#include "flexatt_kernels.h"

namespace {
using namespace flexatt;

// The bytes a [b, h, s, d] view spans.
struct Span {
  uintptr_t lo, hi;
};
Span span_of(const flexatt_tensor* t, int dt, int64_t n_b, int64_t n_h, int64_t n_s, int64_t n_d) {
  const int64_t last = (n_b - 1) * t->stride_b + (n_h - 1) * t->stride_h + (n_s - 1) * t->stride_s + n_d;
  return Span{(uintptr_t)t->data, (uintptr_t)t->data + (uintptr_t)(last * (int64_t)elt_size(dt))};
}
Span span_of(const void* p, size_t bytes) { return Span{(uintptr_t)p, (uintptr_t)p + bytes}; }
bool overlap(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

int check_sizes(int dtype, int64_t b, int64_t h, int64_t s, int head_dim) {
  if (elt_size(dtype) == 0) return FLEXATT_EDTYPE;
  if (b <= 0 || h <= 0 || s <= 0) return FLEXATT_EINVAL;
  if (head_index(head_dim) < 0) return FLEXATT_EHEADDIM;
  // (s: indices of up to a few tiles behind the last row fit 32 bits)
  if (s > 1 << 30 || b * h > INT32_MAX || b * h * s > INT32_MAX) return FLEXATT_ESHAPE;
  return FLEXATT_OK;
}

int check_rotary(const flexatt_rotary* r, bool append) {
  if (!r) return FLEXATT_EINVAL;
  if (r->heads_q != 0 || !append) FLEXATT_TRY(check_sizes(r->dtype, r->batch, r->heads_q, r->seqlen, r->head_dim));
  if (r->heads_kv < 0) return FLEXATT_EINVAL;
  if (r->heads_kv > 0) FLEXATT_TRY(check_sizes(r->dtype, r->batch, r->heads_kv, r->seqlen, r->head_dim));
  if (r->rotary_dim < 0 || r->rotary_dim > r->head_dim || r->rotary_dim % 2) return FLEXATT_EINVAL;
  if (r->rotary_dim > 0 && !r->inv_freq) return FLEXATT_EINVAL;
  if ((r->interleaved & ~1) || (r->inverse & ~1) || r->reserved != 0 || !isfinite(r->magnitude))
    return FLEXATT_EINVAL;
  if (r->positions ? r->position_bytes != 4 && r->position_bytes != 8 : r->position_bytes != 0) return FLEXATT_EINVAL;
  if (((uintptr_t)r->inv_freq) % 8 || (r->positions && ((uintptr_t)r->positions) % r->position_bytes))
    return FLEXATT_ELAYOUT;
  // (a thread has 16 bytes of each half of a token's pairs, or one pair of them; rotary.hip)
  const int es = (int)elt_size(r->dtype), units = r->rotary_dim * es % 32 == 0 ? r->head_dim * es / 32 : r->head_dim / 2;
  return check_launch(((int64_t)r->batch * r->seqlen * units + 255) / 256, 256);
}

RotaryArgs rotary_args(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* qo) {
  RotaryArgs a = {};
  if (r->heads_q > 0) {
    a.q = view(q);
    a.qo = mview(qo);
  }
  a.inv_freq = r->inv_freq;
  a.positions = r->positions;
  a.pos_sb = r->position_stride_b;
  a.pos_ss = r->position_stride_s;
  a.pos_bytes = r->position_bytes;
  a.B = r->batch;
  a.Hq = r->heads_q;
  a.Hkv = r->heads_kv;
  a.S = r->seqlen;
  a.D = r->head_dim;
  a.rotary = r->rotary_dim;
  a.inter = r->interleaved;
  a.mag = r->magnitude;
  a.sign = r->inverse ? -1.0f : 1.0f;
  a.heads = r->heads_q + r->heads_kv;
  return a;
}

// [dtype][head index]
const TreeLauncher kTree[3][4] = {
    {tree_attn_f32_d32, tree_attn_f32_d64, tree_attn_f32_d128, tree_attn_f32_d256},
    {tree_attn_f16_d32, tree_attn_f16_d64, tree_attn_f16_d128, tree_attn_f16_d256},
    {tree_attn_bf16_d32, tree_attn_bf16_d64, tree_attn_bf16_d128, tree_attn_bf16_d256},
};
const WeightLauncher kWeights[3][4] = {
    {weight_sums_f32_d32, weight_sums_f32_d64, weight_sums_f32_d128, weight_sums_f32_d256},
    {weight_sums_f16_d32, weight_sums_f16_d64, weight_sums_f16_d128, weight_sums_f16_d256},
    {weight_sums_bf16_d32, weight_sums_bf16_d64, weight_sums_bf16_d128, weight_sums_bf16_d256},
};

int check_scores(float scale, float cap, int window) {
  if (!(cap >= 0.f) || !isfinite(cap) || !isfinite(scale) || window < 0) return FLEXATT_EINVAL;
  return FLEXATT_OK;
}

// The score parameters of a Shape without causal, ALiBi, interval and block masks.
Shape score_shape(int B, int Hq, int Hkv, int Sq, int Skv, float scale, float cap, int window) {
  Shape s = {};
  s.B = B;
  s.Hq = Hq;
  s.Hkv = Hkv;
  s.G = Hq / Hkv;
  s.Sq = Sq;
  s.Skv = Skv;
  s.scale = scale;
  s.scale_log2 = scale * kLog2e;
  s.window = window;
  s.cap = cap;
  s.inv_cap = cap > 0.f ? 1.0f / cap : 0.f;
  s.tanh_k = cap > 0.f ? 2.0f * kLog2e * scale / cap : 0.f;
  s.cap_log2 = cap * kLog2e;
  s.blk_h = 1;
  return s;
}

int check_tree(const flexatt_tree* p) {
  if (!p) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_q, p->tokens, p->head_dim));
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim));
  if (p->heads_q % p->heads_kv != 0) return FLEXATT_ESHAPE;
  // (2^32 work-items are one launch's most)
  if ((int64_t)(p->heads_q / p->heads_kv) * p->tokens > 1 << 20) return FLEXATT_ERANGE;
  if ((int64_t)p->batch * p->heads_q * p->tokens > 1 << 23) return FLEXATT_ERANGE;
  FLEXATT_TRY(check_scores(p->scale, p->soft_cap, p->sliding_window));
  if (p->reserved != 0 || !p->lengths) return FLEXATT_EINVAL;
  if (p->tree_mask ? p->mask_batch != 1 && p->mask_batch != p->batch : p->mask_batch != 0) return FLEXATT_EINVAL;
  if (p->sliding_window > 0 && p->tree_mask && !p->depths) return FLEXATT_EINVAL;
  return FLEXATT_OK;
}

// How the key tiles are cut (tree_chunk, on the device, where the lengths are): into
// about as many chunks as workgroups run at once, of eight tiles at least (two per wave;
// of 4 or 16 changes a short cache's 15 us by less than 0.2).  Rows of 256 bytes and more
// leave room for one workgroup per CU (LDS; cut for two: bf16 D=256, window 4096, 25 ->
// 35 us), shorter ones for two (cut for one: fp16 T=64 D=64 56 -> 75 us).  Chunks end
// with their (b, hkv), which makes up to one more for each.  With a full cache a (b,
// hkv) has its even share of the chunks, and up to twice that where lengths are
// unequal.
struct TreePlan {
  int slots, nchunk, min_tiles, nsplit;
};
TreePlan tree_plan(const flexatt_tree* p) {
  TreePlan t;
  const int rowb = p->head_dim * (int)elt_size(p->dtype);
  const int64_t rt = ((int64_t)(p->heads_q / p->heads_kv) * p->tokens + 31) / 32;
  const int share = tree_share(rowb, (int)elt_size(p->dtype), rt);
  const int64_t groups = (rt + share - 1) / share;
  // a chunk's row tiles are on one of the 8 XCDs (tree_attn_kernel): whole chunks of each
  // (fp32 B=2 Hq=8 Hkv=2 T=53 caches of 22374 D=128, 7 row tiles: 36 chunks, five on some
  // XCDs for 32 CUs, 192 us, 32 chunks 117)
  const int64_t fit = (rowb >= 256 ? 1 : 2) * cus(), slots = groups <= fit / 8 ? fit / 8 / groups * 8 : fit / groups;
  const int64_t bh = (int64_t)p->batch * p->heads_kv, tiles = (p->cache_rows + 31) / 32;
  // a cache of up to 512 rows whole: what the chunks save the merge costs (bf16 B=1 Hq=32
  // Hkv=8 T=8 D=128, 500 rows 13.4 -> 11.3 us, 1000 rows 14.0 -> 14.9; fp32 D=64, 500 rows
  // 15.1 -> 16.8)
  t.min_tiles = elt_size(p->dtype) == 2 && tiles <= 16 ? 16 : 8;
  t.slots = slots < 1 ? 1 : (int)slots;
  const int64_t most = (tiles + t.min_tiles - 1) / t.min_tiles;  // chunks of one (b, hkv)
  int64_t ns = 2 * ((t.slots + bh - 1) / bh) + 1;
  if (2 * bh > t.slots && p->batch > 1) ns = 3;  // (few chunks each: unequal lengths count most)
  // A chunk is longer than all sequences' tiles times Hkv / slots (tree_chunk), so a single
  // one that has them all makes slots / Hkv chunks at most, one where Hkv alone fills the
  // slots: no partials are kept, and no merge launched, for chunks that never are.
  const int64_t even = (t.slots + p->heads_kv - 1) / p->heads_kv;
  if (ns > even) ns = even;
  if (ns > most) ns = most;
  t.nsplit = (int)ns;
  int64_t n = t.slots + bh;
  if (n > bh * ns) n = bh * ns;
  t.nchunk = (int)n;
  return t;
}
size_t tree_rows(const flexatt_tree* p) { return (size_t)p->batch * p->heads_q * p->tokens; }

// Keys of a workgroup of the weight sums (WsCfg).
int weight_keys(const flexatt_weights* p) { return p->head_dim * (int)elt_size(p->dtype) <= 512 ? 256 : 128; }

int check_weights(const flexatt_weights* p) {
  if (!p) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_q, p->seqlen_q, p->head_dim));
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_kv, p->seqlen_kv, p->head_dim));
  if (p->heads_q % p->heads_kv != 0) return FLEXATT_ESHAPE;
  if ((int64_t)(p->heads_q / p->heads_kv) * p->seqlen_q > 1 << 30) return FLEXATT_ESHAPE;
  FLEXATT_TRY(check_scores(p->scale, p->soft_cap, p->sliding_window));
  if ((p->causal & ~1) || (p->accumulate & ~1) || p->reserved != 0) return FLEXATT_EINVAL;
  // (a workgroup per block of keys; where there are that many its rows are not shared)
  const int keys = weight_keys(p);
  return check_launch((int64_t)p->batch * p->heads_kv * ((p->seqlen_kv + keys - 1) / keys), 256);
}

// Which blocks of keys a workgroup has, one or a pair (the second from the other end,
// which under a causal mask evens out the work), and how many workgroups share their
// query rows: what takes the fewest rounds of workgroups (two per CU, one with rows of
// 512 bytes) times their row tiles, a block counted as some five more to load and add up.
// (In one run, bf16 B=2 Hq=32 Hkv=8 S=4096 D=128 causal, 128 pairs: 4 parts 162 us, 6 and
// 8 167, 12 175, 16 177.  Blocks alone where they leave CUs idle: bf16 Hq=32 Hkv=8 D=128, 1 row over
// 700 keys 11.7 -> 7.4 us, fp32 Hq=8 Hkv=1 D=256, 5 over 2803 30 -> 16; pairs where they
// do not: bf16 B=3, 32 heads, 1 row over 19106 keys 122 -> 115 us.)
struct WeightPlan {
  int pair, parts;
};
WeightPlan weight_plan(const flexatt_weights* p) {
  const int rowb = p->head_dim * (int)elt_size(p->dtype);
  const int keys = weight_keys(p);
  const int64_t nkb = (p->seqlen_kv + keys - 1) / keys;
  const int64_t bh = (int64_t)p->batch * p->heads_kv, slots = (rowb >= 512 ? 1 : 2) * cus();
  // the row tiles that see block x (starts on the device: as if the rows were the last)
  const int64_t start = p->query_starts ? (int64_t)p->seqlen_kv - p->seqlen_q : p->query_start;
  const auto tiles_of = [&](int64_t x) {
    int64_t lo = p->causal ? x * keys - start : 0, hi = p->seqlen_q;
    if (p->sliding_window > 0 && (x + 1) * keys + p->sliding_window - start < hi)
      hi = (x + 1) * keys + p->sliding_window - start;
    if (lo < 0) lo = 0;
    return hi > lo ? ((hi - lo) * (p->heads_q / p->heads_kv) + 31) / 32 : 0;
  };
  // the most of a block and of a pair: of the ends', the quarters' and the middle's
  int64_t tiles = 0, both = 0;
  for (int64_t x : {(int64_t)0, nkb / 4, (nkb - 1) / 2}) {
    const int64_t a = tiles_of(x), b = nkb - 1 - x != x ? tiles_of(nkb - 1 - x) : 0;
    tiles = a > tiles ? a : tiles;
    tiles = b > tiles ? b : tiles;
    both = a + b > both ? a + b : both;
  }
  // row tiles of a part, at least: the second launch adds parts up (bf16 Hq=28 Hkv=4 D=128,
  // 49 rows over 2123 keys, 11 tiles: of four 14.8 us, two 12.0, one 14.5; fp32, whose
  // tiles take four times as long, 32 heads, 200 rows, D=128: 40, 24 and 16)
  const int64_t least = elt_size(p->dtype) == 2 ? 2 : 1;
  WeightPlan best = {0, 1};
  int64_t best_cost = INT64_MAX;
  for (int pair = nkb > 1 ? 1 : 0; pair >= 0; --pair) {
    const int64_t groups = (pair ? (nkb + 1) / 2 : nkb) * bh, work = pair ? both : tiles;
    for (int64_t n = 1; n <= 64 && (n == 1 || tiles / n >= least); ++n) {
      const int64_t cost = (groups * n + slots - 1) / slots * ((work + n - 1) / n + (pair ? 9 : 5));
      if (cost < best_cost) best = {pair, (int)n}, best_cost = cost;
    }
  }
  return best;
}
}  // namespace

extern "C" {

int flexatt_rotary_apply(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* k,
                         const flexatt_tensor* q_out, const flexatt_tensor* k_out, void* stream) {
  FLEXATT_TRY(check_rotary(r, false));
  FLEXATT_TRY(check_tensor(q, r->dtype));
  FLEXATT_TRY(check_out_tensor(q_out, r->dtype, r->batch, r->heads_q, r->seqlen, r->head_dim));
  if (r->heads_kv == 0 && (k || k_out)) return FLEXATT_EINVAL;
  RotaryArgs a = rotary_args(r, q, q_out);
  if (r->heads_kv > 0) {
    FLEXATT_TRY(check_tensor(k, r->dtype));
    FLEXATT_TRY(check_out_tensor(k_out, r->dtype, r->batch, r->heads_kv, r->seqlen, r->head_dim));
    a.k = view(k);
    a.ko = mview(k_out);
  }
  return (int)rotary_run(r->dtype, a, (hipStream_t)stream);
}

int flexatt_rotary_append(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* k,
                          const flexatt_tensor* v, const flexatt_tensor* q_out, const flexatt_tensor* k_cache,
                          const flexatt_tensor* v_cache, int32_t cache_rows, const int32_t* lengths, void* stream) {
  FLEXATT_TRY(check_rotary(r, true));
  if (r->heads_kv == 0 || cache_rows <= 0 || !lengths) return FLEXATT_EINVAL;
  if ((int64_t)r->batch * r->heads_kv * cache_rows > INT32_MAX) return FLEXATT_ESHAPE;
  FLEXATT_TRY(check_tensor(k, r->dtype));
  FLEXATT_TRY(check_tensor(v, r->dtype));
  if (r->heads_q > 0) {
    FLEXATT_TRY(check_tensor(q, r->dtype));
    FLEXATT_TRY(check_out_tensor(q_out, r->dtype, r->batch, r->heads_q, r->seqlen, r->head_dim));
  } else if (q || q_out) {
    return FLEXATT_EINVAL;
  }
  FLEXATT_TRY(check_out_tensor(k_cache, r->dtype, r->batch, r->heads_kv, cache_rows, r->head_dim));
  FLEXATT_TRY(check_out_tensor(v_cache, r->dtype, r->batch, r->heads_kv, cache_rows, r->head_dim));
  FLEXATT_TRY(check_out_pair(k_cache, v_cache, r->dtype, r->batch, r->heads_kv, cache_rows, r->head_dim));
  const auto span = [&](const flexatt_tensor* t, int heads, int rows) {
    return t ? span_of(t, r->dtype, r->batch, heads, rows, r->head_dim) : Span{};
  };
  for (const Span& x : {span(q, r->heads_q, r->seqlen), span(q_out, r->heads_q, r->seqlen),
                        span(k, r->heads_kv, r->seqlen), span(v, r->heads_kv, r->seqlen),
                        span_of(lengths, (size_t)r->batch * 4)})
    for (const flexatt_tensor* y : {k_cache, v_cache})
      if (overlap(x, span(y, r->heads_kv, cache_rows))) return FLEXATT_ELAYOUT;
  RotaryArgs a = rotary_args(r, q, q_out);
  a.k = view(k);
  a.v = view(v);
  a.ko = mview(k_cache);
  a.vo = mview(v_cache);
  a.cache_rows = cache_rows;
  a.lengths = lengths;
  a.heads += r->heads_kv;
  return (int)rotary_run(r->dtype, a, (hipStream_t)stream);
}

size_t flexatt_tree_fwd_workspace(const flexatt_tree* p) {
  if (check_tree(p) != FLEXATT_OK) return SIZE_MAX;
  const int ns = tree_plan(p).nsplit;
  if (ns == 1) return 0;
  return tree_rows(p) * ns * (p->head_dim + 1) * sizeof(float) + (size_t)p->batch * p->heads_kv * sizeof(int);
}

int flexatt_tree_fwd(const flexatt_tree* p, const flexatt_tensor* q, const flexatt_tensor* k_cache,
                     const flexatt_tensor* v_cache, const flexatt_tensor* o, float* lse, void* workspace,
                     size_t workspace_bytes, void* stream) {
  FLEXATT_TRY(check_tree(p));
  FLEXATT_TRY(check_tensor(q, p->dtype));
  FLEXATT_TRY(check_tensor(k_cache, p->dtype));
  FLEXATT_TRY(check_tensor(v_cache, p->dtype));
  for (const flexatt_tensor* x : {k_cache, v_cache})  // offsets within a tile of 32 rows are 32 bits
    if (p->cache_rows > 1 && x->stride_s >= (1 << 26) / (int64_t)elt_size(p->dtype)) return FLEXATT_ERANGE;
  FLEXATT_TRY(check_out_tensor(o, p->dtype, p->batch, p->heads_q, p->tokens, p->head_dim));
  if (!lse) return FLEXATT_EINVAL;
  const size_t need = flexatt_tree_fwd_workspace(p);
  if (need > 0) {
    if (!workspace || workspace_bytes < need) return FLEXATT_EINVAL;
    if (((uintptr_t)workspace) % 16 != 0) return FLEXATT_ELAYOUT;
  }
  TreeArgs a = {};
  a.q = view(q);
  a.k = view(k_cache);
  a.v = view(v_cache);
  a.o = mview(o);
  a.lse = lse;
  const TreePlan plan = tree_plan(p);
  a.slots = plan.slots;
  a.nchunk = plan.nchunk;
  a.min_tiles = plan.min_tiles;
  a.nsplit = plan.nsplit;
  if (a.nsplit > 1) {
    a.part_o = (float*)workspace;
    a.part_lse = a.part_o + tree_rows(p) * a.nsplit * p->head_dim;
    a.counts = (int*)(a.part_lse + tree_rows(p) * a.nsplit);
  }
  a.lengths = p->lengths;
  a.mask = p->tree_mask;
  a.mask_sb = p->mask_batch > 1 ? (int64_t)p->tokens * p->tokens : 0;
  a.depths = p->depths;
  a.p = score_shape(p->batch, p->heads_q, p->heads_kv, p->tokens, p->cache_rows, p->scale, p->soft_cap,
                    p->sliding_window);
  return (int)kTree[p->dtype][head_index(p->head_dim)](a, (hipStream_t)stream);
}

size_t flexatt_weight_sums_workspace(const flexatt_weights* p) {
  if (check_weights(p) != FLEXATT_OK) return SIZE_MAX;
  const int n = weight_plan(p).parts;
  return n == 1 ? 0 : (size_t)n * p->batch * p->heads_kv * p->seqlen_kv * sizeof(float);
}

int flexatt_weight_sums(const flexatt_weights* p, const flexatt_tensor* q, const flexatt_tensor* k, const float* lse,
                        float* sums, void* workspace, size_t workspace_bytes, void* stream) {
  FLEXATT_TRY(check_weights(p));
  FLEXATT_TRY(check_tensor(q, p->dtype));
  FLEXATT_TRY(check_tensor(k, p->dtype));
  if (!lse || !sums) return FLEXATT_EINVAL;
  // (other workgroups still read the inputs while the sums are written)
  const Span out = span_of(sums, (size_t)p->batch * p->heads_kv * p->seqlen_kv * 4);
  for (const Span& in : {span_of(q, p->dtype, p->batch, p->heads_q, p->seqlen_q, p->head_dim),
                         span_of(k, p->dtype, p->batch, p->heads_kv, p->seqlen_kv, p->head_dim),
                         span_of(lse, (size_t)p->batch * p->heads_q * p->seqlen_q * 4),
                         span_of(p->lengths, p->lengths ? (size_t)p->batch * 4 : 0),
                         span_of(p->query_starts, p->query_starts ? (size_t)p->batch * 4 : 0)})
    if (overlap(in, out)) return FLEXATT_ELAYOUT;
  const size_t need = flexatt_weight_sums_workspace(p);
  if (need > 0) {
    if (!workspace || workspace_bytes < need) return FLEXATT_EINVAL;
    if (((uintptr_t)workspace) % 16 != 0) return FLEXATT_ELAYOUT;
  }
  WeightArgs a = {};
  a.q = view(q);
  a.k = view(k);
  a.lse = lse;
  a.sums = sums;
  a.lengths = p->lengths;
  a.starts = p->query_starts;
  a.start = p->query_start;
  a.add = p->accumulate;
  a.part = (float*)workspace;
  const WeightPlan plan = weight_plan(p);
  a.nparts = plan.parts;
  a.pair = plan.pair;
  a.p = score_shape(p->batch, p->heads_q, p->heads_kv, p->seqlen_q, p->seqlen_kv, p->scale, p->soft_cap,
                    p->sliding_window);
  a.p.causal = p->causal;
  return (int)kWeights[p->dtype][head_index(p->head_dim)](a, (hipStream_t)stream);
}

int flexatt_evict_rows(const flexatt_evict* p, const flexatt_tensor* k_cache, const flexatt_tensor* v_cache,
                       const float* scores, const flexatt_tensor* k_out, const flexatt_tensor* v_out,
                       float* scores_out, int32_t* slots, int32_t* lengths_out, void* stream) {
  if (!p) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim));
  if (p->keep < 1 || p->recent < 0 || p->sinks < 0 || p->out_rows < p->keep || (p->fill & ~1)) return FLEXATT_EINVAL;
  if ((int64_t)p->recent + p->sinks > p->keep) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_kv, p->out_rows, p->head_dim));
  FLEXATT_TRY(check_launch((int64_t)p->batch * p->heads_kv, p->cache_rows <= 2048 ? 256 : 1024));  // (evict_run)
  if (!p->lengths || !scores || !scores_out || !slots || !lengths_out) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_tensor(k_cache, p->dtype));
  FLEXATT_TRY(check_tensor(v_cache, p->dtype));
  FLEXATT_TRY(check_out_tensor(k_out, p->dtype, p->batch, p->heads_kv, p->out_rows, p->head_dim));
  FLEXATT_TRY(check_out_tensor(v_out, p->dtype, p->batch, p->heads_kv, p->out_rows, p->head_dim));
  FLEXATT_TRY(check_out_pair(k_out, v_out, p->dtype, p->batch, p->heads_kv, p->out_rows, p->head_dim));
  const int64_t bh = (int64_t)p->batch * p->heads_kv;
  const Span in[] = {span_of(k_cache, p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim),
                     span_of(v_cache, p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim),
                     span_of(scores, bh * p->cache_rows * 4), span_of(p->lengths, p->batch * 4)};
  const Span out[] = {span_of(k_out, p->dtype, p->batch, p->heads_kv, p->out_rows, p->head_dim),
                      span_of(v_out, p->dtype, p->batch, p->heads_kv, p->out_rows, p->head_dim),
                      span_of(scores_out, bh * p->out_rows * 4), span_of(slots, bh * p->keep * 4),
                      span_of(lengths_out, p->batch * 4)};
  for (const Span& x : in)
    for (const Span& y : out)
      if (overlap(x, y)) return FLEXATT_ELAYOUT;
  for (int i = 2; i < 5; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return FLEXATT_ELAYOUT;
  EvictArgs a = {};
  a.k = view(k_cache);
  a.v = view(v_cache);
  a.ko = mview(k_out);
  a.vo = mview(v_out);
  a.scores = scores;
  a.scores_out = scores_out;
  a.slots = slots;
  a.lengths = p->lengths;
  a.lengths_out = lengths_out;
  a.B = p->batch;
  a.H = p->heads_kv;
  a.C = p->cache_rows;
  a.D = p->head_dim;
  a.keep = p->keep;
  a.recent = p->recent;
  a.sinks = p->sinks;
  a.out_rows = p->out_rows;
  a.fill = p->fill;
  a.es = (int)elt_size(p->dtype);
  return (int)evict_run(a, cus(), (hipStream_t)stream);
}

}  // extern "C"
