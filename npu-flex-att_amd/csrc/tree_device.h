// What the attention kernels over a K/V cache share (tree_attn.hip, quant_attn.hip): a
// sequence's key tiles and how they are cut into chunks, tile copies to LDS, and the merge of
// the chunks' partials.
#pragma once
#include "flexatt_device.h"
#include "flexatt_kernels.h"

namespace flexatt {
namespace {  // (each source that includes it has kernels of its own)

constexpr float kTreeRescale = 8.0f;  // lazy rescale threshold, log2 units (as the forward)

// Sequence b: its length, and its key tiles [t0, t1).  `bad`: the tree does not fit.
struct TreeSeq {
  int n, t0, t1;
  bool bad;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
  TreeSeq x;
  x.n = a.lengths[b];
  x.bad = x.n < 0 || x.n > a.p.Skv - a.p.Sq;
  if (x.bad) x.n = 0;
  x.t0 = a.p.window > 0 ? max(x.n - a.p.window, 0) / 32 : 0;
  x.t1 = (x.n + a.p.Sq + 31) / 32;
  return x;
}
// The chunk of workgroup x: which (b, hkv) (b < 0: none, x is past the last chunk),
// which chunk of how many, its first tile and how many.  Every lane of a wave calls
// it and gets the same; lane l looks at sequences l, l + 64, ....
struct TreeChunk {
  int b, hk, s, ns, first, count;
};
__device__ __forceinline__ TreeChunk tree_chunk(const TreeArgs& a, int x, int nw) {
  const int lane = threadIdx.x & 63;
  const int B = a.p.B, H = a.p.Hkv;
  auto tiles_of = [&](int b) {
    const TreeSeq q = tree_seq(a, min(b, B - 1));
    return b < B ? q.t1 - q.t0 : 0;
  };
  const int mine = tiles_of(lane);
  int total = 0, most = 0;
  for (int b0 = 0, v = mine; b0 < B; b0 += 64, v = tiles_of(b0 + lane)) {
    total += __builtin_amdgcn_readlane(wave_scan(v), 63);
    most = max(most, (int)wave_max((unsigned)v));
  }
  // The shortest chunks, whole rounds of the waves, with which one round of workgroups
  // has them all; not looked for where there are many sequences anyway.  Quotients by
  // reciprocals (a division of integers is some forty instructions): `len` only has to
  // be as long as the two bounds, and a sequence's chunks at most nsplit and at most
  // one more than its tiles over len.
  int len = max((int)((float)total * (float)H * fast_rcp((float)a.slots) * 1.00001f),
                (int)((float)most * fast_rcp((float)a.nsplit) * 1.00001f)) + 1;
  len = (max(len, a.min_tiles) + nw - 1) / nw * nw;
  auto chunks_of = [&](int v) {
    const int c = (int)((float)(v + len - 1) * fast_rcp((float)len));
    return v > 0 ? min(max(c, 1), a.nsplit) : 0;
  };
  if (2 * B * H <= a.slots && B <= 64) {
    for (int tries = 0; tries < 8; ++tries) {
      if (__builtin_amdgcn_readlane(wave_scan(chunks_of(mine)), 63) * H <= a.slots) break;
      len += nw;
    }
  }
  TreeChunk r;
  r.b = -1;
  for (int b0 = 0, v = mine; b0 < B; b0 += 64, v = tiles_of(b0 + lane)) {
    const int c = chunks_of(v), upto = wave_scan(c);
    const unsigned long long in = __builtin_amdgcn_ballot_w64(upto * H > x);
    if (in) {
      const int l = __builtin_ctzll(in);
      const int tiles = __builtin_amdgcn_readlane(v, l), n = __builtin_amdgcn_readlane(c, l);
      x -= (__builtin_amdgcn_readlane(upto, l) - n) * H;
      r.b = b0 + l;
      const float inv = fast_rcp((float)n);
      r.hk = (int)((float)x * inv);
      r.s = x - r.hk * n;
      while (r.s < 0) r.s += n, r.hk -= 1;
      while (r.s >= n) r.s -= n, r.hk += 1;
      r.ns = n;
      int each = (int)((float)tiles * inv) + 1;
      while ((each - 1) * n >= tiles) each -= 1;
      while (each * n < tiles) each += 1;
      r.first = r.s * each;
      r.count = max(min(each, tiles - r.first), 0);
      return r;
    }
    x -= __builtin_amdgcn_readlane(upto, 63) * H;
  }
  return r;
}

// The chunk x < Hkv np of a shared prefix.  A window leaves its last rows only: as many as
// the sequence with the fewest cached tokens reaches.  Chunks are whole multiples of UNIT tiles.
template <int UNIT>
__device__ __forceinline__ TreeChunk prefix_chunk(const PrefixArgs& a, int x) {
  const int t1 = (a.P + 31) / 32;
  int t0 = 0;
  if (a.t.p.window > 0) {
    const int lane = threadIdx.x & 63, B = a.t.p.B;
    unsigned need = 0;
    for (int b = lane; b < B; b += 64) need = max(need, (unsigned)max(a.t.p.window - tree_seq(a.t, b).n, 0));
    t0 = (a.P - (int)min(wave_max(need), (unsigned)a.P)) / (32 * UNIT) * UNIT;
  }
  TreeChunk r;
  r.b = 0;
  r.hk = x / a.np;
  r.s = x - r.hk * a.np;
  r.ns = a.np;
  const int each = (t1 - t0 + a.np * UNIT - 1) / (a.np * UNIT) * UNIT;
  r.first = t0 + r.s * each;
  r.count = max(min(each, t1 - r.first), 0);
  return r;
}

// Direct-to-LDS copies of a tile of rows: lane offsets from the tile's first row (the
// swizzle repeats after PERIOD copies, so there are as many of them) and a scalar
// base, a copy being RPC rows.
__device__ __forceinline__ void load_lds16_base(unsigned voff, uint64_t base, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds_addr) : "memory");
}
// Merge of a row's partials, one wave per row, four columns per lane and D / 4 lanes
// for every NG-th partial: M = max LSE_s, O = sum 2^(LSE_s - M) O_s /
// sum 2^(LSE_s - M).  A partial without keys has LSE -inf and is left out; one with a
// NaN score makes the row NaN.  Latency-bound: all LSEs at once, one per lane.
template <class T, int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  constexpr int TPR = D / 4, NG = TPR < 64 ? 64 / TPR : 1;
  const Shape& p = a.p;
  const int lane = threadIdx.x & 63;
  const int row32 = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row32 >= p.B * p.Hq * p.Sq) return;
  const int64_t row = row32;
  const int bh = row32 / p.Sq, i = row32 - bh * p.Sq;
  const int b = bh / p.Hq, hq = bh - b * p.Hq;
  const int most = a.nsplit;
  const float* pl = a.part_lse + row * most;
  const int c = lane % TPR, g = lane / TPR;
  const f32x4* po = (const f32x4*)(a.part_o + row * most * D) + c;
  // The first partials are read before it is known how many the row has: what is
  // there instead of the others is read (nsplit of them are the row's) and not used.
  constexpr int U = 4;
  f32x4 v[U];
  float lw[U], ll;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = min(g + NG * u, most - 1);
    v[u] = po[(int64_t)t * TPR];
    lw[u] = pl[t];
  }
  ll = pl[min(lane, most - 1)];
  const int ns = a.counts[b * p.Hkv + hq / p.G];
  if (ns == 1) return;  // (and a sequence that does not fit) written by its workgroup
  float mx = lane < ns ? ll : kNegInf;
  for (int s0 = 64; s0 < ns; s0 += 64) mx = fmaxf(mx, s0 + lane < ns ? pl[s0 + lane] : kNegInf);
#pragma unroll
  for (int x = 32; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
  const float m0 = mx == kNegInf ? 0.f : mx;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  float ws = 0.f;
  for (int s0 = g;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool keys = s0 + NG * u < ns && lw[u] != kNegInf;  // without keys the values do not count, not even an inf
      const float w = keys ? fast_exp2(lw[u] - m0) : 0.f;
      ws += w;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = keys ? __builtin_fmaf(w, v[u][j], acc[j]) : acc[j];
    }
    s0 += NG * U;
    if (s0 - g >= ns) break;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(s0 + NG * u, most - 1);
      v[u] = po[(int64_t)t * TPR];
      lw[u] = pl[t];
    }
  }
#pragma unroll
  for (int x = TPR; x < 64; x *= 2) {
    ws += __shfl_xor(ws, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor(acc[j], x);
  }
  const bool none = ws == 0.f;  // no key for this row
  if (g == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = none ? 0.f : acc[j] / ws;
    T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)i * a.o.ss + 4 * c;
    if constexpr (sizeof(T) == 4) *(f32x4*)out = acc;
    else st_global8(out, pack4<T>(acc[0], acc[1], acc[2], acc[3]));
  }
  if (lane == 0) a.lse[row] = none ? kNegInf : (mx + log2f(ws)) * kLn2;
}

}  // namespace
}  // namespace flexatt
