// Kernel argument blocks and launcher declarations (internal to libflexatt).
#pragma once
#include <hip/hip_runtime.h>

#include "flexatt_device.h"

namespace flexatt {

struct FwdArgs {
  View q, k, v;
  MutView o;
  float* lse;
  Shape p;
  int nqt;    // number of query tiles (set by the launcher)
  int gpack;  // query heads per workgroup (set by the launcher)
  int bstride;  // block-sparse maps: bytes per wave's block-map row in dynamic LDS (set by the launcher)
};

struct DeltaArgs {
  View o, dout;
  float* delta;
  int B, H, S, D;
  int* zero;  // when set: 4 queue counters the pass clears for the kernels after it
};

struct BwdArgs {
  View q, k, v, dout;
  const float* lse;
  const float* delta;
  MutView dq, dk, dv;
  Shape p;
  int ntiles;  // number of row tiles of the kernel's grid (set by the launcher)
  // dQ with Delta computed in the kernel (bwd_q only): O, and where Delta is
  // written for the dK/dV kernel; delta_out == nullptr: Delta is read from delta.
  View o;
  float* delta_out;
  // Staged dS (D = 128 fp16/bf16): the workspace the dK/dV kernel writes and
  // the dQ kernel reads, and the units stored per query head (the layout is
  // described with ds_tile_offset); ds == nullptr: not staged.
  char* ds;
  int64_t ds_head;
  // Work queue (staged path): queue == nullptr keeps the static work order;
  // otherwise workgroups from nstatic on take their slot from the counter.
  int* queue;
  int nstatic;
  // Staged dK/dV with each KV block's query tiles shared by nparts workgroups:
  // their fp32 sums [part][dK, dV][B * Hkv * Skv][D] (nparts == 1: none)
  float* part;
  int nparts;
};

// Split-KV forward (fwd_split.hip): partials in the caller's workspace, none
// with one split per row tile.
struct DecodeArgs {
  View q, k, v;
  MutView o;
  float* lse;
  float* part_o;    // [B * Hq * Sq][nsplit][D], O of each partial / its row sums
  float* part_lse;  // [B * Hq * Sq][nsplit], LSE of each partial in log2 units
  Shape p;
  int nsplit;  // workgroups per row tile
  int chunk;   // 32-row KV tiles per workgroup (nsplit > 1)
  int nw;      // waves per workgroup with one split (4 or 8; D = 256: 4)
  int nrt;     // 32-row tiles of packed query rows per (b, hkv) (set by the launcher)
  int plain;   // workgroups in plain order instead of by XCD (set by the launcher)
};

// Backward in one launch with the streams split over waves (bwd_split.hip).
struct BwdSplitArgs {
  View q, k, v, dout;
  const float* lse;
  const float* delta;
  MutView dq, dk, dv;
  Shape p;
  float* part;  // nsplit > 1: [split][dK, dV][B * Hkv * Skv][D] fp32
  int nsplit;   // workgroups per KV item
  int nw;       // waves per workgroup (4 or 8; D = 128: 4)
  int nkt;      // 32-row KV tiles (set by the launcher)
  int nrt;      // 32-row tiles of packed query rows per (b, hkv) (set by the launcher)
};

// Rotary positions, out of place or into a cache (rotary.hip).
struct RotaryArgs {
  View q, k, v;        // k with Hkv > 0, v with the append
  MutView qo, ko, vo;  // ko, vo: the cache with cache_rows > 0
  const double* inv_freq;
  const void* positions;  // int32 or int64 (pos_bytes), or pos_bytes 0: the token's slot
  int64_t pos_sb, pos_ss;
  const int* lengths;     // [B], the append
  int B, Hq, Hkv, S, D, rotary, inter, pos_bytes, cache_rows;
  int heads;  // q, k and v heads walked in all
  int hpt;    // heads per thread (set by the launcher)
  float mag, sign;
};

// The same with a norm of each head before the rotation, and into a cache of 8 bits
// (norm_rotary.hip).
struct NormRotaryArgs {
  RotaryArgs r;  // the gradient: q, k what went in, qo, ko their gradients
  View gq, gk;   // the gradient: of what came out
  const void *wq, *wk;  // [D], 4 bytes each with w_wide, else of the call's type
  void *dwq, *dwk;
  float* part;   // the gradient: [groups of heads][columns][D]
  float *k_scales, *v_scales;  // [B][Hkv][cache_rows] with kind
  float eps;
  int norm, w_wide;
  int kind;      // 0, or enum flexatt_code: the cache's rows are bytes
  int q_groups, k_groups;  // groups of q heads and of k heads (set by the launcher)
};

// The gradient's workgroups: `columns` of tokens times the groups of hpt heads, q's and
// k's apart, as many as three a CU, which run at once (registers; bf16 B=2 S=4096 Hq=32
// Hkv=8 D=128: 768 of them, 16 heads each, 50 us, 1280 56).
struct NormGradPlan {
  int columns, hpt, q_groups, k_groups;
};
inline NormGradPlan norm_grad_plan(int B, int S, int Hq, int Hkv, int D, int es) {
  constexpr int64_t kMost = 768;
  NormGradPlan p;
  const int64_t per = 256 / (D * es / 32), nb = ((int64_t)B * S + per - 1) / per;
  for (p.hpt = 1;; p.hpt *= 2) {
    p.q_groups = (Hq + p.hpt - 1) / p.hpt;
    p.k_groups = (Hkv + p.hpt - 1) / p.hpt;
    if (nb * (p.q_groups + p.k_groups) <= kMost || (p.q_groups <= 1 && p.k_groups <= 1) || p.hpt >= 1 << 20) break;
  }
  const int64_t groups = p.q_groups + p.k_groups, most = kMost > groups ? kMost / groups : 1;
  p.columns = (int)(nb < most ? nb : most);
  return p;
}

// A cache of 8 bits read back (dequant.hip).
struct DequantArgs {
  View k, v;  // bytes
  MutView ko, vo;
  const float *k_scales, *v_scales;  // [B][H][C]
  const int* lengths;
  int B, H, C, D, kind;
  int fill;  // 1: rows behind the length are zeroed
};
// Rows of one of its workgroups, of rowb output bytes: four rounds of its threads where
// that leaves four workgroups a CU, else one.
inline int dequant_rows(int rowb, int64_t bh, int64_t cache_rows) {
  const int once = 256 / (rowb / 16);
  return bh * ((cache_rows + 4 * once - 1) / (4 * once)) >= 1024 ? 4 * once : once;
}

// Attention of a tree of drafted tokens over a cache (tree_attn.hip).
struct TreeArgs {
  View q, k, v;
  MutView o;
  float* lse;
  float* part_o;    // [B * Hq * T][nsplit][D], O of each partial / its row sums
  float* part_lse;  // [B * Hq * T][nsplit], LSE of each partial in log2 units
  const int* lengths;          // [B]
  const unsigned char* mask;   // [1 or B][T][T], or nullptr: a chain
  int64_t mask_sb;
  const int* depths;           // [B][T] with a window, or nullptr: t
  Shape p;  // Sq: T, Skv: rows of the cache
  int* counts;    // [B * Hkv], chunks of each (b, hkv), for the merge; nullptr with nsplit 1
  int slots;      // workgroups per row tile that run at once
  int nchunk;     // most chunks of all (b, hkv) together
  int min_tiles;  // least 32-key tiles of a chunk
  int nsplit;     // most chunks of one (b, hkv)
  int nrt;        // groups of packed query row tiles per (b, hkv) (set by the launcher)
};

// The same behind a prefix that all sequences share (tree_attn.hip): t.nsplit is the most
// chunks of a sequence's own cache.
struct PrefixArgs {
  TreeArgs t;
  View k, v;  // [Hkv, P, D]: sh, ss
  int P;
  int np;     // chunks of the prefix, the first partials of every row
  int pitch;  // partials of a row, np + t.nsplit
  int npre;   // workgroups of the prefix, the first of the launch (set by the launcher)
  int nrtp;   // groups of the prefix's row tiles, B * G * T rows (set by the launcher)
  int wide;   // eight row tiles of the prefix a workgroup
};

// The same over a cache of 8 bits (quant_attn.hip): t.k and t.v are bytes.
struct QuantTreeArgs {
  TreeArgs t;
  const float *k_scales, *v_scales;  // [B][Hkv][Skv]
  int kind;
};

// Attention weight received by each key (weight_sums.hip).
struct WeightArgs {
  View q, k;
  const float* lse;   // [B][Hq][Sq]
  float* sums;        // [B][Hkv][Skv]
  const int* lengths;  // [B] or nullptr: Skv
  const int* starts;   // [B] or nullptr: start
  Shape p;
  int start;  // position of the first query row
  int add;    // 1: added to what sums holds
  float* part;  // nparts > 1: [nparts][B][Hkv][Skv]
  int nparts;   // workgroups that share the query rows of a block of keys
  int pair;     // 1: a workgroup has block x and the x-th from the end
};

// Eviction (evict.hip).
struct EvictArgs {
  View k, v;
  MutView ko, vo;
  const float* scores;  // [B][H][C]
  float* scores_out;    // [B][H][out_rows]
  int* slots;           // [B][H][keep]
  const int* lengths;
  int* lengths_out;
  int B, H, C, D, keep, recent, sinks, out_rows;
  int fill;  // 1: rows of ko and vo behind the last kept one, up to keep, are zeroed
  int es;    // bytes per element
  int lanes_log2, nparts;  // lanes that copy a row, workgroups per (sequence, head) (set by the launcher)
};

// Row tiles of 32 that the waves of one tree attention workgroup share a key tile for, of
// `tiles` in all: four of 256-byte rows, or two where four would pad by more than a sixth
// (tree_attn.hip).
inline int tree_share(int row_bytes, int elt_bytes, int64_t tiles) {
  if (elt_bytes != 2 || row_bytes > 256 || tiles < 2) return 1;
  return row_bytes > 128 && (tiles + 3) / 4 * 4 * 6 <= (tiles + 1) / 2 * 2 * 7 ? 4 : 2;
}

// Whether a workgroup has eight row tiles of a shared prefix, of `all`, and a sequence's own
// rows are `own` (tree_attn.hip): 16-bit rows of 256 bytes, where eight pad by a sixth at
// most (bf16 Hq=32 Hkv=8 D=128, 128 sequences of 2 tokens behind 8000 rows 82 -> 68 us, 64
// of 1 behind 4000 46 -> 40; D=64, 28 row tiles behind 8000 rows 26 -> 31).
inline bool prefix_wide(int row_bytes, int elt_bytes, int64_t all, int64_t own) {
  return elt_bytes == 2 && row_bytes == 256 && own <= 2 && (all + 7) / 8 * 8 * 6 <= all * 7;
}

// Threads of a workgroup over a cache of 8 bits (quant_attn.hip).
constexpr int quant_threads(int head_dim) { return head_dim == 128 ? 512 : 256; }

typedef hipError_t (*TreeLauncher)(const TreeArgs&, hipStream_t);

typedef hipError_t (*PrefixLauncher)(const PrefixArgs&, hipStream_t);
typedef hipError_t (*QuantTreeLauncher)(const QuantTreeArgs&, hipStream_t);
typedef hipError_t (*NormRotaryLauncher)(int dtype, const NormRotaryArgs&, hipStream_t);
typedef hipError_t (*WeightLauncher)(const WeightArgs&, hipStream_t);
typedef hipError_t (*FwdLauncher)(const FwdArgs&, hipStream_t);
typedef hipError_t (*DecodeLauncher)(const DecodeArgs&, hipStream_t);
typedef hipError_t (*BwdLauncher)(const BwdArgs&, hipStream_t);
typedef hipError_t (*BwdSplitLauncher)(const BwdSplitArgs&, hipStream_t);

#define FLEXATT_DECL_D(D)                                                     \
  hipError_t fwd_mfma_bf16_d##D(const FwdArgs&, hipStream_t);                 \
  hipError_t fwd_mfma_f16_d##D(const FwdArgs&, hipStream_t);                  \
  hipError_t bwd_dq_mfma_bf16_d##D(const BwdArgs&, hipStream_t);              \
  hipError_t bwd_dq_mfma_f16_d##D(const BwdArgs&, hipStream_t);               \
  hipError_t bwd_dkdv_mfma_bf16_d##D(const BwdArgs&, hipStream_t);            \
  hipError_t bwd_dkdv_mfma_f16_d##D(const BwdArgs&, hipStream_t);

FLEXATT_DECL_D(32)
FLEXATT_DECL_D(64)
FLEXATT_DECL_D(128)
FLEXATT_DECL_D(256)
#undef FLEXATT_DECL_D
// D = 256 forward with wave-specialised pairs (fwd_ws.hip), called by the
// D = 256 forward launcher
hipError_t fwd_ws_bf16_d256(const FwdArgs&, hipStream_t);
hipError_t fwd_ws_f16_d256(const FwdArgs&, hipStream_t);
bool fwd_ws_fits(const Shape& p);  // its LDS (with a block map's lists) fits one CU

// [lo, hi) of every position's document (doc_bounds.hip): ids [B][S] integers
// of ids_bytes bytes, bounds int32 [B][S][2].
hipError_t doc_bounds_run(const void* ids, int ids_bytes, int B, int S, int* bounds, hipStream_t);

hipError_t bwd_delta(int dtype, const DeltaArgs&, hipStream_t);

hipError_t rotary_run(int dtype, const RotaryArgs&, hipStream_t);
hipError_t evict_run(const EvictArgs&, int cus, hipStream_t);
hipError_t dequant_run(int dtype, const DequantArgs&, hipStream_t);

// Tree attention (tree_attn.hip, quant_attn.hip), weight sums (weight_sums.hip), norm and
// rotation (norm_rotary.hip), every D.
#define FLEXATT_DECL_CACHE(D)                              \
  hipError_t tree_attn_bf16_d##D(const TreeArgs&, hipStream_t); \
  hipError_t tree_attn_f16_d##D(const TreeArgs&, hipStream_t);  \
  hipError_t tree_attn_f32_d##D(const TreeArgs&, hipStream_t);  \
  hipError_t prefix_attn_bf16_d##D(const PrefixArgs&, hipStream_t); \
  hipError_t prefix_attn_f16_d##D(const PrefixArgs&, hipStream_t);  \
  hipError_t prefix_attn_f32_d##D(const PrefixArgs&, hipStream_t);  \
  hipError_t weight_sums_bf16_d##D(const WeightArgs&, hipStream_t); \
  hipError_t weight_sums_f16_d##D(const WeightArgs&, hipStream_t);  \
  hipError_t weight_sums_f32_d##D(const WeightArgs&, hipStream_t);  \
  hipError_t quant_attn_bf16_d##D(const QuantTreeArgs&, hipStream_t); \
  hipError_t quant_attn_f16_d##D(const QuantTreeArgs&, hipStream_t);  \
  hipError_t norm_rotary_d##D(int, const NormRotaryArgs&, hipStream_t); \
  hipError_t norm_rotary_grad_d##D(int, const NormRotaryArgs&, hipStream_t);

FLEXATT_DECL_CACHE(32)
FLEXATT_DECL_CACHE(64)
FLEXATT_DECL_CACHE(128)
FLEXATT_DECL_CACHE(256)
#undef FLEXATT_DECL_CACHE

// Split-KV forward (fwd_split.hip).
hipError_t fwd_split_bf16_d32(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_f16_d32(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_bf16_d64(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_f16_d64(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_bf16_d128(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_f16_d128(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_bf16_d256(const DecodeArgs&, hipStream_t);
hipError_t fwd_split_f16_d256(const DecodeArgs&, hipStream_t);

// Backward in one launch (bwd_split.hip), D <= 128.
hipError_t bwd_split_bf16_d32(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_f16_d32(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_bf16_d64(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_f16_d64(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_bf16_d128(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_f16_d128(const BwdSplitArgs&, hipStream_t);

// dK and dV from the splits' sums (a.part, a.nsplit), every D.
hipError_t bwd_split_sum_bf16_d32(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_f16_d32(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_bf16_d64(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_f16_d64(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_bf16_d128(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_f16_d128(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_bf16_d256(const BwdSplitArgs&, hipStream_t);
hipError_t bwd_split_sum_f16_d256(const BwdSplitArgs&, hipStream_t);

// The same two for fp32 inputs (f32_split.hip; the forward with one split), D <= 128.
hipError_t fwd_split_f32_d32(const DecodeArgs&, hipStream_t);
hipError_t bwd_split_f32_d32(const BwdSplitArgs&, hipStream_t);
hipError_t fwd_split_f32_d64(const DecodeArgs&, hipStream_t);
hipError_t bwd_split_f32_d64(const BwdSplitArgs&, hipStream_t);
hipError_t fwd_split_f32_d128(const DecodeArgs&, hipStream_t);
hipError_t bwd_split_f32_d128(const BwdSplitArgs&, hipStream_t);

// dK/dV as a KV-stationary tile stream (bwd_kv.hip), D = 64, 128 and 256.
hipError_t bwd_kv_bf16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_f16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_bf16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_f16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_bf16_d256(const BwdArgs&, hipStream_t);  // dV and dK passes as items of one launch
hipError_t bwd_kv_f16_d256(const BwdArgs&, hipStream_t);

// dK/dV that also writes its dS to a.ds (bwd_kv.hip), and dQ = scale * dS K
// from it (bwd_dq_ds.hip), D = 64, 128 and 256.
hipError_t bwd_kv_ds_bf16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_bf16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_bf16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_bf16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_bf16_d256(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f16_d256(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_bf16_d256(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f16_d256(const BwdArgs&, hipStream_t);

// fp32 inputs on the fp32 matrix cores (f32_mfma.hip): forward, dK/dV (with
// or without writing dS), dQ from the staged dS and dQ recomputing S and dP,
// every D.
hipError_t fwd_f32_d32(const FwdArgs&, hipStream_t);
hipError_t fwd_f32_d64(const FwdArgs&, hipStream_t);
hipError_t fwd_f32_d128(const FwdArgs&, hipStream_t);
hipError_t fwd_f32_d256(const FwdArgs&, hipStream_t);
hipError_t bwd_dq_f32_d32(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_f32_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_f32_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_f32_d256(const BwdArgs&, hipStream_t);
hipError_t bwd_dkdv_f32_d32(const BwdArgs&, hipStream_t);
hipError_t bwd_dkdv_f32_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_dkdv_f32_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_dkdv_f32_d256(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f32_d32(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f32_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f32_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_kv_ds_f32_d256(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f32_d32(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f32_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f32_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_dq_ds_f32_d256(const BwdArgs&, hipStream_t);

// dQ as a query-stationary tile stream (bwd_q.hip), D = 64 and 128; with
// a.delta_out set it also computes Delta (written there) from O and dO.
hipError_t bwd_q_bf16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_q_f16_d128(const BwdArgs&, hipStream_t);
hipError_t bwd_q_bf16_d64(const BwdArgs&, hipStream_t);
hipError_t bwd_q_f16_d64(const BwdArgs&, hipStream_t);

}  // namespace flexatt
