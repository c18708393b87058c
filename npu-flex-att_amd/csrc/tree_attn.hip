// Attention of a tree of drafted tokens over a K/V cache (speculative decoding;
// with one token, ordinary decoding over a batch of caches of unequal lengths).
// No counterpart in the reference, which has no cache.
//
// Semantics: those of the forward (npu_flash_attention.py:17-166: scale, soft-cap,
// mask, online softmax in the log2 domain, LSE in natural log) with, for drafted
// token t of a sequence of n cached tokens, the keys j < n (with a window,
// n + depth[t] - j <= W) and those slots n + u, u < T, whose mask[t][u] is set
// (no mask: u <= t).  A row without keys is 0 with LSE -inf; a sequence whose
// n + T rows do not fit the cache (or n < 0) is NaN.
//
// Decomposition
//  * the G * T query rows of one KV head are packed with the heads innermost into
//    tiles of 32, the columns of an MFMA tile, so heads and tokens share K and V; a wave
//    has one such tile, and of several tiles of 16-bit rows up to 256 bytes two or four
//    waves share the key tiles in LDS (tree_share);
//  * the 32-key tiles of a (b, hkv), as many as the sequence's own length has, are cut
//    into equal chunks of about `len` tiles, one per workgroup; `len` is found on the
//    device from all lengths, so that a cache of large capacity that holds little, or a
//    batch of unequal lengths, fills the chip once; the workgroups of one chunk for
//    different row tiles share an XCD and with it L2;
//  * within a chunk, wave (or group of waves) w takes tiles w, w + NW, ... with its own
//    LDS stages and online softmax, a wave alone without barriers; the states of a row
//    tile's waves are combined through LDS, and the chunks' partials (O over its row sum,
//    LSE) by a second kernel in a fixed order;
//  * rows behind n + T are never read: the copies repeat the last row instead, so
//    what a cache holds there (NaN too) does not matter.
// Precision: scores, maxima, row sums, accumulators, partials and LSE are fp32.  P
// alone is rounded to the type, as in the forward: it is an operand of the 16-bit MFMAs
// of P V (a second one for what the rounding leaves out would double them).  A weight
// is off by half a step at most (2^-8 of it in bf16, 2^-11 in fp16; the row sum has the
// unrounded ones), which over many keys averages out to about what O's own rounding is:
// the rms error of bf16 outputs is 1.8e-3 to 2.3e-3 of their rms, 1.7e-3 the output's
// rounding alone, of fp16 ones 2.9e-4 and 2.1e-4; the same rounding in a plain fp32
// computation gives the same errors to three digits.
// What bounds it: K and V from HBM for long caches and few rows; from some hundred
// rows per KV head on the softmax's VALU work and the MFMAs; latency for short caches.
// Of that the instructions are the larger part: a launch finds the instruction cache
// cold and runs most of this code once, at about one cycle a byte, so what is outside
// the tile loop is kept short (16-byte LDS accesses in the combine, rolled loops).
//   bf16 B=8 Hq=32 Hkv=8 T=16, caches of 24576 to 32768, D=128: 181 us, 5.2 TB/s
//   bf16 B=2 Hq=16 Hkv=8 T=16, window 4096, soft-cap 50, D=256: 25 us (the merge 4.8), 2.7 TB/s
//   fp16 B=4 Hq=28 Hkv=4 T=64, caches up to 16384, D=64: 52 us, 0.52 PFLOP/s
//   fp16 B=3 Hq=28 Hkv=4 T=64, caches of 20000, D=128: 87 us, 0.63 PFLOP/s
//   bf16 B=1 Hq=32 Hkv=8 T=8, a cache of 4097, D=128: 14 us (9.5 and the merge 4.6)
// Shared key tiles halve or quarter the copies from L2, which many rows wait for.  The
// alternative, two row tiles per wave of its own key tiles, reads LDS as little but has a
// SIMD to itself (register file) and copies as much: the D=128 cases above 186 and 193 us.
// Pairs instead of fours: 147 us for the latter, D=64 55 (fours 56).
#include "flexatt_device.h"
#include "flexatt_kernels.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
constexpr float kTreeRescale = 8.0f;  // lazy rescale threshold, log2 units (as the forward)

// LDS stages by the bytes of a row: two of a K and a V tile per wave, so that the
// next tile is in flight during the whole of this one, where four waves' fit
// 160 KB (rows up to 256 bytes); one above, K refilled after the scores and V
// after P V; two waves of 1 KB rows.
template <class T, int D>
struct TreeCfg {
  static constexpr int BN = 32;                       // keys per tile
  static constexpr int ROWB = D * (int)sizeof(T);     // bytes per row
  static constexpr int KC = ROWB / 32;                // 32-byte steps of S^T = K Q^T
  static constexpr int DB = D / 32;                   // 32-row blocks of O^T
  static constexpr int CPR = ROWB / 16;               // 16-byte chunks per row
  static constexpr int RPC = 64 / CPR;                // rows per 1 KB copy
  static constexpr int TB = BN * ROWB;                // bytes of one K or V tile
  static constexpr int E = TB / 1024;                 // copies per tile
  static constexpr int PK = RPC >= 16 ? 1 : 16 / RPC;  // copies after which K's swizzle repeats (16 rows)
  static constexpr int VROWS = sizeof(T) == 4 ? (CPR >= 16 ? 8 : 1) : CPR == 4 ? 1 : CPR == 32 ? 8 : 4;
  static constexpr int PV = RPC >= VROWS ? 1 : VROWS / RPC;  // and V's
  static constexpr int NW = ROWB <= 512 ? 4 : 2;      // waves per workgroup
  static constexpr int ST = ROWB <= 256 ? 2 : 1;      // stages
  static constexpr int WAVEB = ST * 2 * TB;
  static_assert(E * 1024 == TB && NW * WAVEB <= 160 * 1024 && E % PK == 0 && E % PV == 0, "tiles");
};

// V tiles of 32-bit elements are read one element per lane, 32 of a row by each
// half wave from rows 4 apart: the second one's chunks sit in the other half of
// a 256-byte bank row.
template <int CPR>
__device__ __forceinline__ int swz_v32(int r, int c) {
  if constexpr (CPR >= 16) return c ^ (((r >> 2) & 1) << 3);
  else return c;
}
template <class T, int CPR>
__device__ __forceinline__ int swz_v(int r, int p) {  // logical chunk at physical chunk p
  if constexpr (sizeof(T) == 4) return swz_v32<CPR>(r, p);
  else return swz_tr_inv<CPR>(r, p);
}

// One 32-byte step of the scores: A rows are keys, B columns query rows; lane half
// h has the bytes 16 h .. 16 h + 15 of the step of its row.
template <class T>
__device__ __forceinline__ f32x16 mma_step(i32x4 k, i32x4 q, f32x16 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__int_as_float(k[e]), __int_as_float(q[e]), c, 0, 0, 0);
    return c;
  } else {
    typedef typename Mfma<T>::v8 V8;
    return Mfma<T>::mma(as_v8<V8>(k), as_v8<V8>(q), c);
  }
}

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

// Direct-to-LDS copies of a tile of rows: lane offsets from the tile's first row (the
// swizzle repeats after PERIOD copies, so there are as many of them) and a scalar
// base, a copy being RPC rows.
__device__ __forceinline__ void load_lds16_base(unsigned voff, uint64_t base, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds_addr) : "memory");
}
}  // namespace

// WPT neighbouring waves, a row tile each, share their key tiles: each copies its share of
// a tile, and a barrier a tile keeps them in step.
template <class T, int D, int NW, int WPT, bool CAP>
__global__ __launch_bounds__(NW * WPT * 64)
__attribute__((amdgpu_waves_per_eu(D * sizeof(T) >= 256 ? (WPT == 1 ? 1 : 2) : WPT == 1 ? 2 : 4)))
void tree_attn_kernel(TreeArgs a) {
  using C = TreeCfg<T, D>;
  constexpr int ST = C::ST, EC = C::E / WPT;  // copies a wave makes of a tile
  constexpr int PK = C::PK > WPT ? C::PK / WPT : 1, PV = C::PV > WPT ? C::PV / WPT : 1, CROWS = WPT * C::RPC;
  static_assert(WPT == 1 || (ST == 2 && C::E % WPT == 0), "shared tiles");
  constexpr int kCombine = NW * WPT * 64 * 4 * (2 + 16 * C::DB);
  __shared__ __attribute__((aligned(1024))) char smem[NW * C::WAVEB > kCombine ? NW * C::WAVEB : kCombine];

  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid / (WPT * 64));  // its key tiles
  const int sub = WPT > 1 ? __builtin_amdgcn_readfirstlane((tid >> 6) % WPT) : 0;
  const int h = lane >> 5, l32 = lane & 31;

  // (chunk, row tiles): the row tiles of one chunk are 8 workgroups apart, on one XCD
  // and started together (as rows of a two-dimensional grid, started one after the
  // other, they find the chunk gone from L2: fp16 B=4 Hq=28 Hkv=4 T=64, caches of
  // 16384 D=64, 58 -> 74 us)
  int rt0 = 0, x = blockIdx.x;
  if (a.nrt > 1) {
    rt0 = blockIdx.x / 8 % a.nrt * WPT;
    x = blockIdx.x / (8 * a.nrt) * 8 + blockIdx.x % 8;
  }
  rt0 += sub;
  const TreeChunk ck = tree_chunk(a, x, NW);
  if (ck.b < 0) return;
  const int b = ck.b, hk = ck.hk, s = ck.s, ns = ck.ns;
  TreeSeq sq = tree_seq(a, b);
  sq.n = __builtin_amdgcn_readfirstlane(sq.n);
  sq.t0 = __builtin_amdgcn_readfirstlane(sq.t0);
  if (rt0 == 0 && s == 0 && tid == 0 && a.counts) a.counts[b * p.Hkv + hk] = sq.bad ? 1 : ns;

  float c2 = p.scale_log2;
  bool flip = false;
  if constexpr (!CAP) {  // as in the forward: a negative scale moves into Q
    flip = c2 < 0.f;
    c2 = c2 == 0.f ? 1e-30f : fabsf(c2);
  }
  int koff[C::KC], voff[C::DB];
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) koff[kc] = l32 * C::ROWB + swz_col<C::CPR>(l32, 2 * kc + h) * 16;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int db = 0; db < C::DB; ++db)  // row 4 h (rows 8 i + 4 h + j have its swizzle)
      voff[db] = 4 * h * C::ROWB + swz_v32<C::CPR>(4 * h, 8 * db + (l32 >> 2)) * 16 + (l32 & 3) * 4;
  } else {
    const int tr_row = 4 * h + ((lane & 15) >> 2);
    const int tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
      voff[db] = tr_row * C::ROWB + swz_tr<C::CPR>(tr_row, 4 * db + (tr_col >> 3)) * 16 + (tr_col & 7) * 2;
  }
  // this lane's offsets in a tile's copies
  const unsigned kss = (unsigned)(a.k.ss * (int)sizeof(T)), vss = (unsigned)(a.v.ss * (int)sizeof(T));
  const int crow = lane / C::CPR + sub * C::RPC, cchunk = lane % C::CPR;
  unsigned kvo[PK], vvo[PV];
#pragma unroll
  for (int e = 0; e < PK; ++e) kvo[e] = (e * CROWS + crow) * kss + swz_col<C::CPR>(e * CROWS + crow, cchunk) * 16;
#pragma unroll
  for (int e = 0; e < PV; ++e) vvo[e] = (e * CROWS + crow) * vss + swz_v<T, C::CPR>(e * CROWS + crow, cchunk) * 16;
  const unsigned wbase = lds_addr_of(smem) + wave * C::WAVEB;
  // this wave's LDS reads have returned: the buffer they read may be refilled
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

  // packed query rows of this lane
  const int R = p.G * p.Sq;
  const int r = min(32 * rt0 + l32, R - 1);
  const int hq = hk * p.G + r % p.G, qi = r / p.G;  // head, drafted token

  if (sq.bad) {
    if (s == 0 && 32 * rt0 + l32 < R) {
      T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss;
      for (int d = wave * 2 + h; d < D; d += NW * 2) out[d] = from_f32<T>(__builtin_nanf(""));
      if (wave == 0 && h == 0) a.lse[((int64_t)b * p.Hq + hq) * p.Sq + qi] = __builtin_nanf("");
    }
    return;
  }

  i32x4 qf[C::KC];
  const char* src = (const char*)((const T*)a.q.data + b * a.q.sb + hq * a.q.sh + (int64_t)qi * a.q.ss) + 16 * h;
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) qf[kc] = ld_global16(src + 32 * kc);

  // this wave's tiles: first + NW * j, j < nt
  const int n = sq.n, last = n + p.Sq - 1;
  const int first = sq.t0 + ck.first + wave;
  const int nt = __builtin_amdgcn_readfirstlane(max((ck.count - wave + NW - 1) / NW, 0));
  const uint64_t kp = (uint64_t)((const T*)a.k.data + b * a.k.sb + hk * a.k.sh);
  const uint64_t vp = (uint64_t)((const T*)a.v.data + b * a.v.sb + hk * a.v.sh);
  auto issue_k = [&](int t, int st) {
    const unsigned dst = wbase + st * 2 * C::TB + sub * 1024;
    const uint64_t base = kp + (uint64_t)(t * C::BN) * kss;
    if (t * C::BN + C::BN - 1 <= last) {
#pragma unroll
      for (int e = 0; e < EC; ++e)
        load_lds16_base(kvo[e % PK], base + (uint64_t)(e / PK * PK * CROWS) * kss, dst + e * WPT * 1024);
    } else {  // rows behind the last one repeat it
#pragma unroll 1
      for (int e = 0; e < EC; ++e) {
        const int kr = e * CROWS + crow;
        load_lds16_base(min(kr, last - t * C::BN) * kss + swz_col<C::CPR>(kr, cchunk) * 16, base, dst + e * WPT * 1024);
      }
    }
  };
  auto issue_v = [&](int t, int st) {
    const unsigned dst = wbase + st * 2 * C::TB + C::TB + sub * 1024;
    const uint64_t base = vp + (uint64_t)(t * C::BN) * vss;
    if (t * C::BN + C::BN - 1 <= last) {
#pragma unroll
      for (int e = 0; e < EC; ++e)
        load_lds16_base(vvo[e % PV], base + (uint64_t)(e / PV * PV * CROWS) * vss, dst + e * WPT * 1024);
    } else {
#pragma unroll 1
      for (int e = 0; e < EC; ++e) {
        const int kr = e * CROWS + crow;
        load_lds16_base(min(kr, last - t * C::BN) * vss + swz_v<T, C::CPR>(kr, cchunk) * 16, base, dst + e * WPT * 1024);
      }
    }
  };
  if (nt > 0) {
    issue_k(first, 0);
    issue_v(first, 0);
  }

  // Row qi sees the cached keys [row_lo, n); the tiles that hold only keys every row
  // sees need no mask.
  int row_lo = 0, full_lo = 0;
  if (p.window > 0) {
    const int depth = a.depths ? max(a.depths[(int64_t)b * p.Sq + qi], 0) : qi;
    // (n + depth - window without leaving 32 bits: depth at most the window counts)
    full_lo = row_lo = max(n - (p.window - min(depth, p.window)), 0);
#pragma unroll
    for (int y = 32; y; y >>= 1) full_lo = max(full_lo, __shfl_xor(full_lo, y));
    full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  }
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;

  // wait for Q here, once: see fwd_split.hip
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) {
    if constexpr (!CAP) {
      constexpr int kSign = sizeof(T) == 4 ? (int)0x80000000 : (int)0x80008000;
      const int f = flip ? kSign : 0;
      qf[kc] ^= i32x4{f, f, f, f};
    }
    pin(qf[kc]);
  }

  f32x16 acc[C::DB];
  float m_run = kNegInf, l_run = 0.f;
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x16{};

  const int steps = WPT == 1 ? nt : __builtin_amdgcn_readfirstlane((ck.count + NW - 1) / NW);
  for (int j = 0; j < steps; ++j) {
    const int t = first + NW * j;
    const bool more = j + 1 < nt;
    if constexpr (WPT > 1) {
      // this wave's copies of tile j have landed and its reads of tile j - 1 have returned ...
      wait_vmcnt<0>();
      reads_done();
      __builtin_amdgcn_s_barrier();  // ... and every wave's
      asm volatile("" ::: "memory");
      if (more) {
        issue_k(t + NW, (j + 1) & 1);
        issue_v(t + NW, (j + 1) & 1);
      }
      if (j >= nt) continue;  // (the last step of waves with one tile less)
    } else if constexpr (ST == 2) {
      if (more) {  // into the stage of tile j - 1, read in the previous iteration
        reads_done();
        issue_k(t + NW, (j + 1) & 1);
        issue_v(t + NW, (j + 1) & 1);
        wait_vmcnt<2 * EC>();  // tile j landed, the next in flight
      } else {
        wait_vmcnt<0>();
      }
    } else {
      wait_vmcnt<EC>();  // K of tile j landed (its V, issued later, may be in flight)
    }
    const char* sK = smem + wave * C::WAVEB + (ST == 2 ? (j & 1) * 2 * C::TB : 0);
    const char* sV = sK + C::TB;
    const int n0 = t * C::BN;

    f32x16 sc = f32x16{};
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      const i32x4 kf = lds_read16(sK + koff[kc]);
      sc = mma_step<T>(kf, qf[kc], sc);
    }
    if constexpr (ST == 1) {
      reads_done();
      if (more) issue_k(t + NW, 0);
    }

    // element e is key n0 + 8(e/4) + 4h + e%4
    if constexpr (CAP) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = tanhf(sc[e] * p.scale * p.inv_cap);
      } else {
        soft_cap(sc, p);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] *= p.cap_log2;
    }
    if (n0 < full_lo || n0 + C::BN > n) {
      // this lane's keys, relative to its first: e, and hidden before lo or from hi on
      const int lo = row_lo - n0 - 4 * h, hi = n + (mask ? p.Sq : qi + 1) - n0 - 4 * h;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if ((unsigned)(8 * (e >> 2) + (e & 3) - lo) >= (unsigned)max(hi - lo, 0)) sc[e] = kNegInf;
      if (mask && n0 + C::BN > n) {  // all of the tile's mask bytes at once
        const unsigned char* mrow = mask + (int64_t)qi * p.Sq;
        const int u0 = n0 + 4 * h - n;
        unsigned char m[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) m[e] = mrow[min(max(u0 + 8 * (e >> 2) + (e & 3), 0), p.Sq - 1)];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (u0 + 8 * (e >> 2) + (e & 3) >= 0 && m[e] == 0) sc[e] = kNegInf;
      }
    }
    f32x16 pe;
    if constexpr (!CAP) settle(sc);  // (an unmasked tile's scores come straight from the MFMAs)
    float mx, mx2;
    max16_partial(sc, mx, mx2);
    mx = max2(mx, mx2);
    if constexpr (!CAP) mx *= c2;
    mx = fmaxf(mx, swap_halves(mx));
    if (mx != mx) mx = kNegInf;
    const bool grow = mx > m_run + kTreeRescale;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float m_new = grow ? mx : m_run;
      const float alpha = grow ? fast_exp2(m_run - m_new) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < C::DB; ++db) scale_inplace(acc[db], alpha);
      m_run = m_new;
    }
    const float m_use = (m_run == kNegInf) ? 0.f : m_run;
    float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if constexpr (!CAP) pe[e] = fast_exp2(__builtin_fmaf(sc[e], c2, -m_use));
      else pe[e] = fast_exp2(sc[e] - m_use);
      rs[e & 3] += pe[e];
    }
    l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    if constexpr (ST == 1) {  // V of tile j landed (the next K may be in flight)
      if (more) wait_vmcnt<EC>();
      else wait_vmcnt<0>();
    }
    if constexpr (sizeof(T) == 4) {
      // key 8 i + 4 h + j of lane half h is accumulator element 4 i + j: P is its own B operand
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const char* vr = sV + (8 * (i >> 2) + (i & 3)) * C::ROWB;
#pragma unroll
        for (int db = 0; db < C::DB; ++db) {
          const float v = *(const float*)(vr + voff[db]);
          acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, pe[i], acc[db], 0, 0, 0);
        }
      }
    } else {
      typedef typename Mfma<T>::v8 V8;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const V8 pb = pack8<T>(pe, 8 * c);
        const char* vr = sV + 16 * c * C::ROWB;
#pragma unroll
        for (int db = 0; db < C::DB; ++db) {
          const i16x4 lo = lds_read_tr4(vr + voff[db]);
          const i16x4 hi = lds_read_tr4(vr + 8 * C::ROWB + voff[db]);
          acc[db] = Mfma<T>::mma(cat_tr<V8>(lo, hi), pb, acc[db]);
        }
      }
    }
    if constexpr (ST == 1) {
      reads_done();
      if (more) issue_v(t + NW, 0);
    }
  }

  // The (m, l, acc) of a row tile's NW waves combined in wave order through LDS (every
  // wave's copies have landed: its last tile waited for vmcnt 0), then O / l and LSE.
  float* xm = (float*)smem + sub * NW * 64 * (2 + 16 * C::DB);  // [NW][64]
  float* xl = xm + NW * 64;                                     // [NW][64]
  f32x4* xa = (f32x4*)(xl + NW * 64);  // [NW][4 DB][64]: columns 8 y + 4 h .. + 3 of row l32
  const float l_tot = l_run + swap_halves(l_run);
  __syncthreads();
  xm[wave * 64 + lane] = m_run;
  xl[wave * 64 + lane] = l_tot;
#pragma unroll
  for (int y = 0; y < 4 * C::DB; ++y) {
    const f32x16& v = acc[y / 4];
    const int e = y % 4 * 4;
    xa[(wave * 4 * C::DB + y) * 64 + lane] = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
  }
  __syncthreads();
  float mw[NW], mall = kNegInf;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    mw[w] = xm[w * 64 + lane];
    mall = fmaxf(mall, mw[w]);
  }
  float al[NW], L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    // a wave whose maximum stayed -inf has weights of 0, or NaN scores
    const float lw = xl[w * 64 + lane];
    al[w] = mw[w] == kNegInf ? (lw == 0.f ? 0.f : 1.f) : fast_exp2(mw[w] - mall);
    L = __builtin_fmaf(al[w], lw, L);
  }
  const bool empty = L == 0.f;  // no key; NaN (a NaN query row or key) is not
  const float inv = empty ? 0.f : 1.0f / L;
  if (32 * rt0 + l32 < R) {
    const int64_t row = ((int64_t)b * p.Hq + hq) * p.Sq + qi;
    float* po = a.part_o + (row * a.nsplit + s) * D + 4 * h;
    T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss + 4 * h;
#pragma unroll 2
    for (int y = wave; y < 4 * C::DB; y += NW) {
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const f32x4 v = xa[(w * 4 * C::DB + y) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(al[w], v[e], o[e]);
      }
      o *= inv;
      if (ns > 1) *(f32x4*)(po + 8 * y) = o;
      else if constexpr (sizeof(T) == 4) *(f32x4*)(out + 8 * y) = o;
      else st_global8(out + 8 * y, pack4<T>(o[0], o[1], o[2], o[3]));
    }
    if (wave == 0 && h == 0) {
      const float lse = empty ? kNegInf : mall + log2f(L);
      if (ns > 1) a.part_lse[row * a.nsplit + s] = lse;
      else a.lse[row] = lse * kLn2;
    }
  }
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

template <class T, int D, int WPT>
void launch_tree_share(TreeArgs a, hipStream_t st) {
  constexpr int NW = WPT == 4 ? TreeCfg<T, D>::NW / 2 : TreeCfg<T, D>::NW;
  a.nrt = (int)((((int64_t)a.p.G * a.p.Sq + 31) / 32 + WPT - 1) / WPT);
  const dim3 grid((unsigned)((a.nchunk + 7) / 8 * 8 * a.nrt)), block(NW * WPT * 64);
  if (a.p.cap > 0.f) hipLaunchKernelGGL((tree_attn_kernel<T, D, NW, WPT, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((tree_attn_kernel<T, D, NW, WPT, false>), grid, block, 0, st, a);
}

template <class T, int D>
hipError_t launch_tree(const TreeArgs& a, hipStream_t st) {
  using C = TreeCfg<T, D>;
  const int share = tree_share(C::ROWB, sizeof(T), ((int64_t)a.p.G * a.p.Sq + 31) / 32);
  if constexpr (sizeof(T) == 2 && C::ROWB <= 256) {
    if constexpr (C::ROWB == 256) {
      if (share == 4) launch_tree_share<T, D, 4>(a, st);
    }
    if (share == 2) launch_tree_share<T, D, 2>(a, st);
  }
  if (share == 1) launch_tree_share<T, D, 1>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nsplit == 1) return e;
  const int64_t rows = (int64_t)a.p.B * a.p.Hq * a.p.Sq;
  hipLaunchKernelGGL((tree_merge_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError();
}

#define FLEXATT_CAT2(a, b) a##b
#define FLEXATT_CAT(a, b) FLEXATT_CAT2(a, b)
hipError_t FLEXATT_CAT(tree_attn_bf16_d, FLEXATT_D)(const TreeArgs& a, hipStream_t st) {
  return launch_tree<__bf16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(tree_attn_f16_d, FLEXATT_D)(const TreeArgs& a, hipStream_t st) {
  return launch_tree<_Float16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(tree_attn_f32_d, FLEXATT_D)(const TreeArgs& a, hipStream_t st) {
  return launch_tree<float, FLEXATT_D>(a, st);
}

}  // namespace flexatt
