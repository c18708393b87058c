// extern "C" entry points around positions and the K/V cache (declared in
// include/flexatt.h): argument checks, then the kernel launchers.
#include <float.h>
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
Span span_bytes(const flexatt_tensor* t, int64_t es, int64_t n_b, int64_t n_h, int64_t n_s, int64_t n_d) {
  const int64_t last = (n_b - 1) * t->stride_b + (n_h - 1) * t->stride_h + (n_s - 1) * t->stride_s + n_d;
  return Span{(uintptr_t)t->data, (uintptr_t)t->data + (uintptr_t)(last * es)};
}
Span span_of(const flexatt_tensor* t, int dt, int64_t n_b, int64_t n_h, int64_t n_s, int64_t n_d) {
  return span_bytes(t, (int64_t)elt_size(dt), n_b, n_h, n_s, n_d);
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

int check_norm(const flexatt_rotary* r, const flexatt_norm* n) {
  if (!n) return FLEXATT_EINVAL;
  if (n->weight_dtype != FLEXATT_F32 && n->weight_dtype != r->dtype) return FLEXATT_EDTYPE;
  if (!(n->eps >= FLT_MIN) || !isfinite(n->eps) || r->inverse) return FLEXATT_EINVAL;
  if ((r->heads_q > 0) != (n->q_weight != nullptr) || (r->heads_kv > 0) != (n->k_weight != nullptr)) return FLEXATT_EINVAL;
  for (const void* w : {n->q_weight, n->k_weight})
    if ((uintptr_t)w % elt_size(n->weight_dtype)) return FLEXATT_ELAYOUT;
  return FLEXATT_OK;
}

// (numbers of heads with a group's added to them fit 32 bits)
int check_norm_heads(const flexatt_rotary* r) {
  return (int64_t)r->heads_q + r->heads_kv > 1 << 30 ? FLEXATT_ERANGE : FLEXATT_OK;
}

// The launch of norm_rotary.hip: a workgroup has 256 / (D / (32 / size)) tokens, and of many
// tokens all heads of q, k or v; few tokens make some thousand workgroups at most.
int check_norm_launch(const flexatt_rotary* r, bool append) {
  FLEXATT_TRY(check_norm_heads(r));
  const int64_t per = 256 / (r->head_dim * (int)elt_size(r->dtype) / 32), kinds = (r->heads_q > 0) + (r->heads_kv > 0) * (append ? 2 : 1);
  return check_launch(((int64_t)r->batch * r->seqlen + per - 1) / per * kinds, 256);
}

// What a call reads besides its tensors, within `out`.
bool within(const flexatt_rotary* r, const flexatt_norm* n, Span out) {
  if (r->rotary_dim > 0 && overlap(span_of(r->inv_freq, (size_t)r->rotary_dim / 2 * 8), out)) return true;
  if (r->positions) {
    const int64_t x = (r->batch - 1) * r->position_stride_b, y = (r->seqlen - 1) * r->position_stride_s, es = r->position_bytes;
    const uintptr_t at = (uintptr_t)r->positions;
    const Span all = {at + (uintptr_t)(((x < 0 ? x : 0) + (y < 0 ? y : 0)) * es),
                      at + (uintptr_t)(((x > 0 ? x : 0) + (y > 0 ? y : 0) + 1) * es)};
    if (overlap(all, out)) return true;
  }
  if (!n) return false;
  const size_t bytes = r->head_dim * elt_size(n->weight_dtype);
  return (n->q_weight && overlap(span_of(n->q_weight, bytes), out)) || (n->k_weight && overlap(span_of(n->k_weight, bytes), out));
}

NormRotaryArgs norm_args(const RotaryArgs& r, const flexatt_norm* n) {
  NormRotaryArgs a = {};
  a.r = r;
  if (n) {
    a.norm = 1;
    a.wq = n->q_weight;
    a.wk = n->k_weight;
    a.w_wide = n->weight_dtype == FLEXATT_F32;
    a.eps = n->eps;
  }
  return a;
}

// [head index]
const NormRotaryLauncher kNorm[4] = {norm_rotary_d32, norm_rotary_d64, norm_rotary_d128, norm_rotary_d256};
const NormRotaryLauncher kNormGrad[4] = {norm_rotary_grad_d32, norm_rotary_grad_d64, norm_rotary_grad_d128,
                                         norm_rotary_grad_d256};

bool is_code(int32_t code) { return code == FLEXATT_E4M3 || code == FLEXATT_INT8; }

// The new tokens' tensors of an append, apart from the cache: `row`: bytes of an element
// of the cache's.
int check_append(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* k, const flexatt_tensor* v,
                 const flexatt_tensor* q_out, const flexatt_tensor* k_cache, const flexatt_tensor* v_cache, int64_t row,
                 int32_t cache_rows, const int32_t* lengths) {
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
  FLEXATT_TRY(check_out_view(k_cache, row, r->batch, r->heads_kv, cache_rows, r->head_dim));
  FLEXATT_TRY(check_out_view(v_cache, row, r->batch, r->heads_kv, cache_rows, r->head_dim));
  FLEXATT_TRY(check_out_views(k_cache, v_cache, row, r->batch, r->heads_kv, cache_rows, r->head_dim));
  const auto span = [&](const flexatt_tensor* t, int heads) {
    return t ? span_of(t, r->dtype, r->batch, heads, r->seqlen, r->head_dim) : Span{};
  };
  for (const Span& x : {span(q, r->heads_q), span(q_out, r->heads_q), span(k, r->heads_kv), span(v, r->heads_kv),
                        span_of(lengths, (size_t)r->batch * 4)})
    for (const flexatt_tensor* y : {k_cache, v_cache})
      if (overlap(x, span_bytes(y, row, r->batch, r->heads_kv, cache_rows, r->head_dim))) return FLEXATT_ELAYOUT;
  return FLEXATT_OK;
}

RotaryArgs append_args(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* k, const flexatt_tensor* v,
                       const flexatt_tensor* q_out, const flexatt_tensor* k_cache, const flexatt_tensor* v_cache,
                       int32_t cache_rows, const int32_t* lengths) {
  RotaryArgs a = rotary_args(r, q, q_out);
  a.k = view(k);
  a.v = view(v);
  a.ko = mview(k_cache);
  a.vo = mview(v_cache);
  a.cache_rows = cache_rows;
  a.lengths = lengths;
  a.heads += r->heads_kv;
  return a;
}

// [dtype][head index]
const TreeLauncher kTree[3][4] = {
    {tree_attn_f32_d32, tree_attn_f32_d64, tree_attn_f32_d128, tree_attn_f32_d256},
    {tree_attn_f16_d32, tree_attn_f16_d64, tree_attn_f16_d128, tree_attn_f16_d256},
    {tree_attn_bf16_d32, tree_attn_bf16_d64, tree_attn_bf16_d128, tree_attn_bf16_d256},
};
const PrefixLauncher kPrefix[3][4] = {
    {prefix_attn_f32_d32, prefix_attn_f32_d64, prefix_attn_f32_d128, prefix_attn_f32_d256},
    {prefix_attn_f16_d32, prefix_attn_f16_d64, prefix_attn_f16_d128, prefix_attn_f16_d256},
    {prefix_attn_bf16_d32, prefix_attn_bf16_d64, prefix_attn_bf16_d128, prefix_attn_bf16_d256},
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

// [fp16, bf16][head index]
const QuantTreeLauncher kQuantTree[2][4] = {
    {quant_attn_f16_d32, quant_attn_f16_d64, quant_attn_f16_d128, quant_attn_f16_d256},
    {quant_attn_bf16_d32, quant_attn_bf16_d64, quant_attn_bf16_d128, quant_attn_bf16_d256},
};

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
int64_t row_tiles(const flexatt_tree* p) { return ((int64_t)(p->heads_q / p->heads_kv) * p->tokens + 31) / 32; }
// `share`: row tiles of a workgroup; `fit`: workgroups that run at once.
TreePlan plan_of(const flexatt_tree* p, int share, int64_t fit) {
  TreePlan t;
  const int64_t groups = (row_tiles(p) + share - 1) / share;
  // a chunk's row tiles are on one of the 8 XCDs (tree_attn_kernel): whole chunks of each
  // (fp32 B=2 Hq=8 Hkv=2 T=53 caches of 22374 D=128, 7 row tiles: 36 chunks, five on some
  // XCDs for 32 CUs, 192 us, 32 chunks 117)
  const int64_t slots = groups <= fit / 8 ? fit / 8 / groups * 8 : fit / groups;
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
TreePlan tree_plan(const flexatt_tree* p) {
  const int rowb = p->head_dim * (int)elt_size(p->dtype);
  return plan_of(p, tree_share(rowb, (int)elt_size(p->dtype), row_tiles(p)), (rowb >= 256 ? 1 : 2) * (int64_t)cus());
}
TreePlan quant_plan(const flexatt_tree* p) {
  return plan_of(p, 1, (p->head_dim >= 128 ? 1 : 2) * (int64_t)cus());
}
// A launch's workgroups: whole eights of chunks for each group of row tiles.
int64_t workgroups(int64_t chunks, int64_t groups) { return (chunks + 7) / 8 * 8 * groups; }

int check_quant_tree(const flexatt_tree* p) {
  FLEXATT_TRY(check_tree(p));
  if (p->tree_mask && p->tokens > 1 << 15) return FLEXATT_ERANGE;  // (offsets in a mask are 32 bits)
  if (p->dtype == FLEXATT_F32) return FLEXATT_EDTYPE;
  return check_launch(workgroups(quant_plan(p).nchunk, row_tiles(p)), quant_threads(p->head_dim));
}
// The launch behind a shared prefix, whose rows are those of all sequences: `np` chunks of
// the prefix, and of each sequence's own cache as TreePlan has them.  Where one round of
// workgroups can have it all, the two that make the longest chunk shortest, in steps of the
// waves (bf16 B=4 Hq=32 Hkv=8 T=1 D=128, a prefix of 16000 rows, caches of 1000: 27 us with
// eight workgroups in a second round, 22 without); else the prefix gets its share of a
// round, by key tiles times row tiles or, with eight row tiles a workgroup, by their times
// (64 sequences of one token behind 4000 rows, caches of 600: 44 -> 40 us).
struct PrefixPlan {
  TreePlan own;
  int np;
  bool wide;
  int64_t workgroups;
  int threads;  // of one
};
PrefixPlan prefix_plan(const flexatt_tree* p, int prefix_rows) {
  const int rowb = p->head_dim * (int)elt_size(p->dtype);
  const int64_t rows = (int64_t)(p->heads_q / p->heads_kv) * p->tokens, all = (rows * p->batch + 31) / 32;
  const bool wide = prefix_wide(rowb, (int)elt_size(p->dtype), all, row_tiles(p));
  const int share = wide ? 8 : tree_share(rowb, (int)elt_size(p->dtype), all), own_share = wide ? 1 : share;
  const int64_t groups = (all + share - 1) / share, own_groups = (row_tiles(p) + own_share - 1) / own_share;
  const int64_t tiles = (prefix_rows + 31) / 32, own_tiles = (p->cache_rows + 31) / 32;
  const int64_t slots = (rowb >= 256 || wide ? 1 : 2) * (int64_t)cus();
  const int64_t waves = wide ? 1 : rowb > 512 ? 2 : share == 4 ? 2 : 4, own_waves = wide ? 8 : waves;
  const int64_t least = 8, most = (tiles + least - 1) / least < 64 ? (tiles + least - 1) / least : 64;
  const int64_t per = groups * p->heads_kv, own_per = own_groups * p->heads_kv * p->batch;
  PrefixPlan t;
  t.own = plan_of(p, own_share, slots);
  t.wide = wide;
  int64_t np = 0, best = INT64_MAX;
  for (int64_t ns = 1; ns <= (own_tiles + least - 1) / least && ns * own_per + per <= slots; ++ns) {
    int64_t n = (slots - ns * own_per) / per;
    if (n > most) n = most;
    const int64_t x = (tiles + n * waves - 1) / (n * waves), y = (own_tiles + ns * own_waves - 1) / (ns * own_waves);
    const int64_t cost = x > y ? x : y;
    if (cost >= best) continue;
    best = cost;
    np = n;
    t.own.nsplit = (int)ns;
    t.own.slots = t.own.nchunk = (int)(ns * p->heads_kv * p->batch);
  }
  if (np == 0 && wide) {
    // in times of a prefix tile: a chunk of it costs five more, a sequence's own workgroup
    // eight and a quarter of each tile; as many chunks as make one no longer than all work's
    // share of a CU
    const int64_t own = own_per * (32 + own_tiles);  // (quarters)
    for (np = 1; np < most && (tiles / np + 5) * slots * 4 > np * per * (tiles / np + 5) * 4 + own;) ++np;
  } else if (np == 0) {
    const int64_t mine = groups * tiles, others = own_groups * p->batch * own_tiles;
    np = (slots * mine / (mine + others) + per / 2) / per;
    np = np < 1 ? 1 : np > most ? most : np;
  }
  t.np = (int)np;
  t.workgroups = workgroups(p->heads_kv * np, groups) + workgroups(t.own.nchunk, own_groups);
  t.threads = wide || share > 1 ? 512 : rowb > 512 ? 128 : 256;
  return t;
}
size_t tree_rows(const flexatt_tree* p) { return (size_t)p->batch * p->heads_q * p->tokens; }

size_t plan_bytes(const flexatt_tree* p, const TreePlan& plan) {
  const int ns = plan.nsplit;
  if (ns == 1) return 0;
  return tree_rows(p) * ns * (p->head_dim + 1) * sizeof(float) + (size_t)p->batch * p->heads_kv * sizeof(int);
}

// The workspace and score parameters of a call whose tensors are set.
TreeArgs tree_args(const flexatt_tree* p, const TreePlan& plan, const flexatt_tensor* q, const flexatt_tensor* k_cache,
                   const flexatt_tensor* v_cache, const flexatt_tensor* o, float* lse, void* workspace) {
  TreeArgs a = {};
  a.q = view(q);
  a.k = view(k_cache);
  a.v = view(v_cache);
  a.o = mview(o);
  a.lse = lse;
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
  return a;
}

size_t prefix_bytes(const flexatt_tree* p, const PrefixPlan& plan) {
  return tree_rows(p) * (plan.np + plan.own.nsplit) * (p->head_dim + 1) * sizeof(float) +
         (size_t)p->batch * p->heads_kv * sizeof(int);
}
int check_prefix(const flexatt_tree* p, int32_t prefix_rows) {
  FLEXATT_TRY(check_tree(p));
  if (prefix_rows < 1) return FLEXATT_EINVAL;
  if ((int64_t)prefix_rows + p->cache_rows > 1 << 30) return FLEXATT_ESHAPE;
  const PrefixPlan plan = prefix_plan(p, prefix_rows);
  return check_launch(plan.workgroups, plan.threads);
}

int check_workspace(size_t need, const void* workspace, size_t bytes) {
  if (need == 0) return FLEXATT_OK;
  if (!workspace || bytes < need) return FLEXATT_EINVAL;
  return (uintptr_t)workspace % 16 != 0 ? FLEXATT_ELAYOUT : FLEXATT_OK;
}

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
  FLEXATT_TRY(check_append(r, q, k, v, q_out, k_cache, v_cache, (int64_t)elt_size(r->dtype), cache_rows, lengths));
  return (int)rotary_run(r->dtype, append_args(r, q, k, v, q_out, k_cache, v_cache, cache_rows, lengths),
                         (hipStream_t)stream);
}

int flexatt_norm_rotary_apply(const flexatt_rotary* r, const flexatt_norm* n, const flexatt_tensor* q,
                              const flexatt_tensor* k, const flexatt_tensor* q_out, const flexatt_tensor* k_out,
                              void* stream) {
  FLEXATT_TRY(check_rotary(r, false));
  FLEXATT_TRY(check_norm(r, n));
  FLEXATT_TRY(check_norm_launch(r, false));
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
  return (int)kNorm[head_index(r->head_dim)](r->dtype, norm_args(a, n), (hipStream_t)stream);
}

size_t flexatt_norm_rotary_grad_workspace(const flexatt_rotary* r) {
  if (check_rotary(r, false) != FLEXATT_OK || check_norm_heads(r) != FLEXATT_OK) return SIZE_MAX;
  const NormGradPlan p = norm_grad_plan(r->batch, r->seqlen, r->heads_q, r->heads_kv, r->head_dim, (int)elt_size(r->dtype));
  return (size_t)p.columns * (p.q_groups + p.k_groups) * r->head_dim * sizeof(float);
}

int flexatt_norm_rotary_grad(const flexatt_rotary* r, const flexatt_norm* n, const flexatt_tensor* q,
                             const flexatt_tensor* k, const flexatt_tensor* q_grad, const flexatt_tensor* k_grad,
                             const flexatt_tensor* dq, const flexatt_tensor* dk, void* dq_weight, void* dk_weight,
                             void* workspace, size_t workspace_bytes, void* stream) {
  FLEXATT_TRY(check_rotary(r, false));
  FLEXATT_TRY(check_norm(r, n));
  FLEXATT_TRY(check_norm_heads(r));
  FLEXATT_TRY(check_tensor(q, r->dtype));
  FLEXATT_TRY(check_tensor(q_grad, r->dtype));
  FLEXATT_TRY(check_out_tensor(dq, r->dtype, r->batch, r->heads_q, r->seqlen, r->head_dim));
  if (r->heads_kv == 0 && (k || k_grad || dk || dk_weight)) return FLEXATT_EINVAL;
  RotaryArgs a = rotary_args(r, q, dq);
  if (r->heads_kv > 0) {
    FLEXATT_TRY(check_tensor(k, r->dtype));
    FLEXATT_TRY(check_tensor(k_grad, r->dtype));
    FLEXATT_TRY(check_out_tensor(dk, r->dtype, r->batch, r->heads_kv, r->seqlen, r->head_dim));
    if (!dk_weight) return FLEXATT_EINVAL;
    a.k = view(k);
    a.ko = mview(dk);
  }
  if (!dq_weight || !workspace || workspace_bytes < flexatt_norm_rotary_grad_workspace(r)) return FLEXATT_EINVAL;
  if ((uintptr_t)workspace % 16) return FLEXATT_ELAYOUT;
  for (const void* w : {dq_weight, dk_weight})
    if ((uintptr_t)w % elt_size(n->weight_dtype)) return FLEXATT_ELAYOUT;
  // (workgroups still read the inputs while others write the outputs)
  const auto span = [&](const flexatt_tensor* t, int heads) {
    return t ? span_of(t, r->dtype, r->batch, heads, r->seqlen, r->head_dim) : Span{};
  };
  const size_t weight = r->head_dim * elt_size(n->weight_dtype);
  const Span outs[] = {span(dq, r->heads_q), span(dk, r->heads_kv), span_of(dq_weight, weight),
                       span_of(dk_weight, dk_weight ? weight : 0), span_of(workspace, flexatt_norm_rotary_grad_workspace(r))};
  const Span ins[] = {span(q, r->heads_q), span(k, r->heads_kv), span(q_grad, r->heads_q), span(k_grad, r->heads_kv)};
  for (const Span& y : outs) {
    if (within(r, n, y)) return FLEXATT_ELAYOUT;
    for (const Span& x : ins)
      if (overlap(x, y)) return FLEXATT_ELAYOUT;
    for (const Span& x : outs)
      if (&x != &y && overlap(x, y)) return FLEXATT_ELAYOUT;
  }
  NormRotaryArgs g = norm_args(a, n);
  g.gq = view(q_grad);
  if (r->heads_kv > 0) g.gk = view(k_grad);
  g.dwq = dq_weight;
  g.dwk = dk_weight;
  g.part = (float*)workspace;
  return (int)kNormGrad[head_index(r->head_dim)](r->dtype, g, (hipStream_t)stream);
}

int flexatt_norm_rotary_append(const flexatt_rotary* r, const flexatt_norm* n, const flexatt_tensor* q,
                               const flexatt_tensor* k, const flexatt_tensor* v, const flexatt_tensor* q_out,
                               const flexatt_tensor* k_cache, const flexatt_tensor* v_cache, int32_t cache_rows,
                               const int32_t* lengths, void* stream) {
  FLEXATT_TRY(check_rotary(r, true));
  FLEXATT_TRY(check_norm(r, n));
  FLEXATT_TRY(check_norm_launch(r, true));
  FLEXATT_TRY(check_append(r, q, k, v, q_out, k_cache, v_cache, (int64_t)elt_size(r->dtype), cache_rows, lengths));
  for (const flexatt_tensor* y : {k_cache, v_cache})
    if (within(r, n, span_of(y, r->dtype, r->batch, r->heads_kv, cache_rows, r->head_dim))) return FLEXATT_ELAYOUT;
  const RotaryArgs a = append_args(r, q, k, v, q_out, k_cache, v_cache, cache_rows, lengths);
  return (int)kNorm[head_index(r->head_dim)](r->dtype, norm_args(a, n), (hipStream_t)stream);
}

int flexatt_quant_append(const flexatt_rotary* r, const flexatt_norm* n, int32_t code, const flexatt_tensor* q,
                         const flexatt_tensor* k, const flexatt_tensor* v, const flexatt_tensor* q_out,
                         const flexatt_tensor* k_cache, const flexatt_tensor* v_cache, float* k_scales,
                         float* v_scales, int32_t cache_rows, const int32_t* lengths, void* stream) {
  FLEXATT_TRY(check_rotary(r, true));
  if (!is_code(code) || r->inverse) return FLEXATT_EINVAL;
  if (n) FLEXATT_TRY(check_norm(r, n));
  FLEXATT_TRY(check_norm_launch(r, true));
  FLEXATT_TRY(check_append(r, q, k, v, q_out, k_cache, v_cache, 1, cache_rows, lengths));
  if (!k_scales || !v_scales) return FLEXATT_EINVAL;
  if ((uintptr_t)k_scales % 4 || (uintptr_t)v_scales % 4) return FLEXATT_ELAYOUT;
  const size_t bytes = (size_t)r->batch * r->heads_kv * cache_rows * 4;
  const Span ks = span_of(k_scales, bytes), vs = span_of(v_scales, bytes);
  if (overlap(ks, vs)) return FLEXATT_ELAYOUT;
  const auto span = [&](const flexatt_tensor* t, int heads) {
    return t ? span_of(t, r->dtype, r->batch, heads, r->seqlen, r->head_dim) : Span{};
  };
  for (const Span& x : {span(q, r->heads_q), span(q_out, r->heads_q), span(k, r->heads_kv), span(v, r->heads_kv),
                        span_of(lengths, (size_t)r->batch * 4),
                        span_bytes(k_cache, 1, r->batch, r->heads_kv, cache_rows, r->head_dim),
                        span_bytes(v_cache, 1, r->batch, r->heads_kv, cache_rows, r->head_dim)})
    if (overlap(x, ks) || overlap(x, vs)) return FLEXATT_ELAYOUT;
  for (const Span& y : {ks, vs, span_bytes(k_cache, 1, r->batch, r->heads_kv, cache_rows, r->head_dim),
                        span_bytes(v_cache, 1, r->batch, r->heads_kv, cache_rows, r->head_dim)})
    if (within(r, n, y)) return FLEXATT_ELAYOUT;
  NormRotaryArgs a = norm_args(append_args(r, q, k, v, q_out, k_cache, v_cache, cache_rows, lengths), n);
  a.kind = code;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  return (int)kNorm[head_index(r->head_dim)](r->dtype, a, (hipStream_t)stream);
}

int flexatt_dequant_rows(const flexatt_dequant* p, const flexatt_tensor* k_cache, const flexatt_tensor* v_cache,
                         const float* k_scales, const float* v_scales, const flexatt_tensor* k_out,
                         const flexatt_tensor* v_out, void* stream) {
  if (!p) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_sizes(p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim));
  if (!is_code(p->code) || (p->fill & ~1) || p->reserved != 0 || !p->lengths) return FLEXATT_EINVAL;
  const int64_t bh = (int64_t)p->batch * p->heads_kv, rows = dequant_rows(p->head_dim * (int)elt_size(p->dtype), bh, p->cache_rows);
  FLEXATT_TRY(check_launch(bh * ((p->cache_rows + rows - 1) / rows), 256));
  FLEXATT_TRY(check_view(k_cache, 1));
  FLEXATT_TRY(check_view(v_cache, 1));
  FLEXATT_TRY(check_out_tensor(k_out, p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim));
  FLEXATT_TRY(check_out_tensor(v_out, p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim));
  FLEXATT_TRY(check_out_pair(k_out, v_out, p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim));
  if (!k_scales || !v_scales) return FLEXATT_EINVAL;
  if ((uintptr_t)k_scales % 4 || (uintptr_t)v_scales % 4) return FLEXATT_ELAYOUT;
  const size_t bytes = (size_t)p->batch * p->heads_kv * p->cache_rows * 4;
  for (const Span& x : {span_bytes(k_cache, 1, p->batch, p->heads_kv, p->cache_rows, p->head_dim),
                        span_bytes(v_cache, 1, p->batch, p->heads_kv, p->cache_rows, p->head_dim),
                        span_of(k_scales, bytes), span_of(v_scales, bytes), span_of(p->lengths, (size_t)p->batch * 4)})
    for (const flexatt_tensor* y : {k_out, v_out})
      if (overlap(x, span_of(y, p->dtype, p->batch, p->heads_kv, p->cache_rows, p->head_dim))) return FLEXATT_ELAYOUT;
  DequantArgs a = {};
  a.k = view(k_cache);
  a.v = view(v_cache);
  a.ko = mview(k_out);
  a.vo = mview(v_out);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.lengths = p->lengths;
  a.B = p->batch;
  a.H = p->heads_kv;
  a.C = p->cache_rows;
  a.D = p->head_dim;
  a.kind = p->code;
  a.fill = p->fill;
  return (int)dequant_run(p->dtype, a, (hipStream_t)stream);
}

size_t flexatt_tree_fwd_workspace(const flexatt_tree* p) {
  return check_tree(p) != FLEXATT_OK ? SIZE_MAX : plan_bytes(p, tree_plan(p));
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
  const TreePlan plan = tree_plan(p);
  FLEXATT_TRY(check_workspace(plan_bytes(p, plan), workspace, workspace_bytes));
  return (int)kTree[p->dtype][head_index(p->head_dim)](tree_args(p, plan, q, k_cache, v_cache, o, lse, workspace),
                                                       (hipStream_t)stream);
}

size_t flexatt_quant_tree_fwd_workspace(const flexatt_tree* p) {
  return check_quant_tree(p) != FLEXATT_OK ? SIZE_MAX : plan_bytes(p, quant_plan(p));
}

int flexatt_quant_tree_fwd(const flexatt_tree* p, int32_t code, const flexatt_tensor* q, const flexatt_tensor* k_cache,
                           const flexatt_tensor* v_cache, const float* k_scales, const float* v_scales,
                           const flexatt_tensor* o, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  FLEXATT_TRY(check_quant_tree(p));
  if (!is_code(code)) return FLEXATT_EINVAL;
  FLEXATT_TRY(check_tensor(q, p->dtype));
  for (const flexatt_tensor* x : {k_cache, v_cache}) {
    FLEXATT_TRY(check_view(x, 1));
    if (p->cache_rows > 1 && x->stride_s >= 1 << 26) return FLEXATT_ERANGE;  // (as flexatt_tree_fwd)
  }
  FLEXATT_TRY(check_out_tensor(o, p->dtype, p->batch, p->heads_q, p->tokens, p->head_dim));
  if (!lse || !k_scales || !v_scales) return FLEXATT_EINVAL;
  if ((uintptr_t)k_scales % 4 || (uintptr_t)v_scales % 4) return FLEXATT_ELAYOUT;
  const TreePlan plan = quant_plan(p);
  FLEXATT_TRY(check_workspace(plan_bytes(p, plan), workspace, workspace_bytes));
  QuantTreeArgs a = {};
  a.t = tree_args(p, plan, q, k_cache, v_cache, o, lse, workspace);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.kind = code;
  return (int)kQuantTree[p->dtype == FLEXATT_BF16][head_index(p->head_dim)](a, (hipStream_t)stream);
}

size_t flexatt_prefix_fwd_workspace(const flexatt_tree* p, int32_t prefix_rows) {
  return check_prefix(p, prefix_rows) != FLEXATT_OK ? SIZE_MAX : prefix_bytes(p, prefix_plan(p, prefix_rows));
}

int flexatt_prefix_fwd(const flexatt_tree* p, int32_t prefix_rows, const flexatt_tensor* q,
                       const flexatt_tensor* prefix_k, const flexatt_tensor* prefix_v, const flexatt_tensor* k_cache,
                       const flexatt_tensor* v_cache, const flexatt_tensor* o, float* lse, void* workspace,
                       size_t workspace_bytes, void* stream) {
  FLEXATT_TRY(check_prefix(p, prefix_rows));
  FLEXATT_TRY(check_tensor(q, p->dtype));
  if (!prefix_k || !prefix_v) return FLEXATT_EINVAL;
  flexatt_tensor pk = *prefix_k, pv = *prefix_v;
  pk.stride_b = pv.stride_b = 0;  // (no batch)
  prefix_k = &pk, prefix_v = &pv;
  for (const flexatt_tensor* x : {prefix_k, prefix_v, k_cache, v_cache}) {
    FLEXATT_TRY(check_tensor(x, p->dtype));
    const int rows = x == prefix_k || x == prefix_v ? prefix_rows : p->cache_rows;  // (as flexatt_tree_fwd)
    if (rows > 1 && x->stride_s >= (1 << 26) / (int64_t)elt_size(p->dtype)) return FLEXATT_ERANGE;
  }
  FLEXATT_TRY(check_out_tensor(o, p->dtype, p->batch, p->heads_q, p->tokens, p->head_dim));
  if (!lse) return FLEXATT_EINVAL;
  const PrefixPlan plan = prefix_plan(p, prefix_rows);
  FLEXATT_TRY(check_workspace(prefix_bytes(p, plan), workspace, workspace_bytes));
  PrefixArgs a = {};
  a.t = tree_args(p, plan.own, q, k_cache, v_cache, o, lse, nullptr);
  a.np = plan.np;
  a.wide = plan.wide;
  a.pitch = plan.np + plan.own.nsplit;
  a.t.part_o = (float*)workspace;
  a.t.part_lse = a.t.part_o + tree_rows(p) * a.pitch * p->head_dim;
  a.t.counts = (int*)(a.t.part_lse + tree_rows(p) * a.pitch);
  a.k = view(prefix_k);
  a.v = view(prefix_v);
  a.P = prefix_rows;
  return (int)kPrefix[p->dtype][head_index(p->head_dim)](a, (hipStream_t)stream);
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
