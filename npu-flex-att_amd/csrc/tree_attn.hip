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
// computation gives the same errors to three digits.  Behind a shared prefix, where a wave
// has a row tile alone (few sequences) and waits for memory, what the rounding leaves is an
// operand of MFMAs of its own: errors of 1.3 to 1.4 times the output's rounding become 1.00,
// at 2% (B=4 T=1 behind 16000 rows 21.9 -> 22.3 us, 2048 rows of B=8 14.8 -> 14.9).  Where
// waves share key tiles it costs 5 to 13% (D=128 12 sequences behind 8000 rows 18.4 -> 19.9
// us, D=64 16 of 8 tokens 25.8 -> 29.3) and eight row tiles a workgroup are bound by their
// MFMAs, so there P is rounded as above.
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
#include <type_traits>

#include "flexatt_device.h"
#include "flexatt_kernels.h"
#include "tree_device.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
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
  static_assert(E * 1024 == TB && NW * ST * 2 * TB <= 160 * 1024 && E % PK == 0 && E % PV == 0, "tiles");
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

}  // namespace

namespace {
template <bool PRE>
using ArgsOf = std::conditional_t<PRE, PrefixArgs, TreeArgs>;
__device__ __forceinline__ const TreeArgs& tree_of(const TreeArgs& a) { return a; }
__device__ __forceinline__ const TreeArgs& tree_of(const PrefixArgs& a) { return a.t; }
}  // namespace

// WPT neighbouring waves, a row tile each, share their key tiles: each copies its share of
// a tile, and a barrier a tile keeps them in step.
//
// Behind a shared prefix the launch's first workgroups have its chunks, whose rows are
// those of all sequences (b, token, head, the head innermost), so that a key of it is read
// once for all of them; the others have the sequences' own caches.  Every row has partials of
// the prefix's chunks and of its own, joined as above.  Bound by latency for few rows, by the
// products for many, whose workgroups stand beside those of the own caches, which wait for
// memory (bf16 Hq=32 Hkv=8 D=128: B=8 T=1 behind 2048 rows, caches of 60 to 300: 14.2 us, the
// merge 4; fp16 B=32 T=4 behind 16383, caches of 300 to 1024: 66 to 74 us, the merge 7).
enum { kTree, kBoth, kOwn };  // no prefix; a workgroup of either kind; of the second alone
template <class T, int D, int NW, int WPT, int ST>
constexpr int tree_lds() {
  constexpr int combine = NW * WPT * 64 * 4 * (2 + 16 * TreeCfg<T, D>::DB), tiles = NW * ST * 2 * TreeCfg<T, D>::TB;
  return tiles > combine ? tiles : combine;
}
template <class T, int D, int NW, int WPT, int ST, bool CAP, int KIND>
__device__ __forceinline__ void tree_work(const ArgsOf<KIND != kTree>& args, char* smem, int block) {
  constexpr bool PRE = KIND != kTree;
  constexpr bool REST = KIND == kBoth && WPT == 1 && sizeof(T) == 2;  // (what P's rounding leaves is a second operand)
  const TreeArgs& a = tree_of(args);
  using C = TreeCfg<T, D>;
  constexpr int EC = C::E / WPT;  // copies a wave makes of a tile
  constexpr int WAVEB = ST * 2 * C::TB;
  constexpr int PK = C::PK > WPT ? C::PK / WPT : 1, PV = C::PV > WPT ? C::PV / WPT : 1, CROWS = WPT * C::RPC;
  static_assert(WPT == 1 || (ST == 2 && C::E % WPT == 0), "shared tiles");

  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid / (WPT * 64));  // its key tiles
  const int sub = WPT > 1 ? __builtin_amdgcn_readfirstlane((tid >> 6) % WPT) : 0;
  const int h = lane >> 5, l32 = lane & 31;

  // (chunk, row tiles): the row tiles of one chunk are 8 workgroups apart, on one XCD
  // and started together (as rows of a two-dimensional grid, started one after the
  // other, they find the chunk gone from L2: fp16 B=4 Hq=28 Hkv=4 T=64, caches of
  // 16384 D=64, 58 -> 74 us)
  int rt0 = 0, x = block;
  bool shared = false;  // a chunk of the prefix
  if constexpr (PRE) {
    if constexpr (KIND == kBoth) {
      shared = x < args.npre;
      if (!shared) x -= args.npre;
    }
    const int nrt = shared ? args.nrtp : a.nrt, i = x;
    rt0 = i / 8 % nrt * WPT;
    x = i / (8 * nrt) * 8 + i % 8;
  } else if (a.nrt > 1) {
    rt0 = block / 8 % a.nrt * WPT;
    x = block / (8 * a.nrt) * 8 + block % 8;
  }
  rt0 += sub;
  TreeChunk ck;
  TreeSeq sq;
  if (PRE && shared) {
    if constexpr (PRE) {
      if (x >= p.Hkv * args.np) return;
      ck = prefix_chunk<1>(args, x);
      sq = TreeSeq{args.P, 0, 0, false};
    }
  } else {
    ck = tree_chunk(a, x, NW);
    if (ck.b < 0) return;
    sq = tree_seq(a, ck.b);
    sq.n = __builtin_amdgcn_readfirstlane(sq.n);
    sq.t0 = __builtin_amdgcn_readfirstlane(sq.t0);
  }
  const int b = ck.b, hk = ck.hk, s = ck.s, ns = ck.ns;
  if constexpr (PRE) {
    if (!shared && rt0 == 0 && s == 0 && tid == 0) a.counts[b * p.Hkv + hk] = sq.bad ? 1 : args.np + ns;
  } else {
    if (rt0 == 0 && s == 0 && tid == 0 && a.counts) a.counts[b * p.Hkv + hk] = sq.bad ? 1 : ns;
  }

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
  View vk = a.k, vv = a.v;
  if constexpr (PRE) {
    if (shared) vk = args.k, vv = args.v;
  }
  const unsigned kss = (unsigned)(vk.ss * (int)sizeof(T)), vss = (unsigned)(vv.ss * (int)sizeof(T));
  const int crow = lane / C::CPR + sub * C::RPC, cchunk = lane % C::CPR;
  unsigned kvo[PK], vvo[PV];
#pragma unroll
  for (int e = 0; e < PK; ++e) kvo[e] = (e * CROWS + crow) * kss + swz_col<C::CPR>(e * CROWS + crow, cchunk) * 16;
#pragma unroll
  for (int e = 0; e < PV; ++e) vvo[e] = (e * CROWS + crow) * vss + swz_v<T, C::CPR>(e * CROWS + crow, cchunk) * 16;
  const unsigned wbase = lds_addr_of(smem) + wave * WAVEB;
  // this wave's LDS reads have returned: the buffer they read may be refilled
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

  // packed query rows of this lane
  const int R = PRE && shared ? p.B * p.G * p.Sq : p.G * p.Sq;
  const int r = min(32 * rt0 + l32, R - 1);
  const int hq = hk * p.G + r % p.G;  // head, drafted token, sequence
  int qi = r / p.G, qb = b;
  if constexpr (PRE) {
    if (shared) {
      qb = qi / p.Sq;
      qi -= qb * p.Sq;
    }
  }

  if (sq.bad) {
    if (s == 0 && 32 * rt0 + l32 < R) {
      T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss;
      for (int d = wave * 2 + h; d < D; d += NW * 2) out[d] = from_f32<T>(__builtin_nanf(""));
      if (wave == 0 && h == 0) a.lse[((int64_t)b * p.Hq + hq) * p.Sq + qi] = __builtin_nanf("");
    }
    return;
  }

  i32x4 qf[C::KC];
  const char* src = (const char*)((const T*)a.q.data + qb * a.q.sb + hq * a.q.sh + (int64_t)qi * a.q.ss) + 16 * h;
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) qf[kc] = ld_global16(src + 32 * kc);

  // this wave's tiles: first + NW * j, j < nt
  const int n = sq.n, last = PRE && shared ? n - 1 : n + p.Sq - 1;
  const int first = sq.t0 + ck.first + wave;
  const int nt = __builtin_amdgcn_readfirstlane(max((ck.count - wave + NW - 1) / NW, 0));
  const uint64_t kp = (uint64_t)((const T*)vk.data + b * vk.sb + hk * vk.sh);
  const uint64_t vp = (uint64_t)((const T*)vv.data + b * vv.sb + hk * vv.sh);
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
    const int depth = a.depths ? max(a.depths[(int64_t)qb * p.Sq + qi], 0) : qi;
    // (n + depth - window without leaving 32 bits: depth at most the window counts)
    int past = n;
    if constexpr (PRE) {
      if (shared) past += min(max(a.lengths[qb], 0), p.Skv);  // (of a sequence that does not fit: not used)
    }
    full_lo = row_lo = max(past - (p.window - min(depth, p.window)), 0);
#pragma unroll
    for (int y = 32; y; y >>= 1) full_lo = max(full_lo, __shfl_xor(full_lo, y));
    full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  }
  const unsigned char* mask = a.mask && !(PRE && shared) ? a.mask + b * a.mask_sb : nullptr;
  const int reach = PRE && shared ? n : n + (mask ? p.Sq : qi + 1);

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
      if constexpr (PRE) {
        if (32 * rt0 >= R) continue;  // (a wave without rows copies only)
      }
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
    const char* sK = smem + wave * WAVEB + (ST == 2 ? (j & 1) * 2 * C::TB : 0);
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
      const int lo = row_lo - n0 - 4 * h, hi = reach - n0 - 4 * h;
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
        V8 pl;
        if constexpr (REST) {
#pragma unroll
          for (int t = 0; t < 8; ++t) pl[t] = from_f32<T>(pe[8 * c + t] - to_f32(pb[t]));
        }
        const char* vr = sV + 16 * c * C::ROWB;
#pragma unroll
        for (int db = 0; db < C::DB; ++db) {
          const i16x4 lo = lds_read_tr4(vr + voff[db]);
          const i16x4 hi = lds_read_tr4(vr + 8 * C::ROWB + voff[db]);
          const V8 v = cat_tr<V8>(lo, hi);
          acc[db] = Mfma<T>::mma(v, pb, acc[db]);
          if constexpr (REST) acc[db] = Mfma<T>::mma(v, pl, acc[db]);
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
    const int64_t row = ((int64_t)qb * p.Hq + hq) * p.Sq + qi;
    int64_t place = row * a.nsplit + s;
    if constexpr (PRE) place = row * args.pitch + (shared ? s : args.np + s);
    float* po = a.part_o + place * D + 4 * h;
    T* out = (T*)a.o.data + qb * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss + 4 * h;
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
      if (PRE || ns > 1) *(f32x4*)(po + 8 * y) = o;
      else if constexpr (sizeof(T) == 4) *(f32x4*)(out + 8 * y) = o;
      else st_global8(out + 8 * y, pack4<T>(o[0], o[1], o[2], o[3]));
    }
    if (wave == 0 && h == 0) {
      const float lse = empty ? kNegInf : mall + log2f(L);
      if (PRE || ns > 1) a.part_lse[place] = lse;
      else a.lse[row] = lse * kLn2;
    }
  }
}

template <class T, int D, int NW, int WPT, bool CAP, bool PRE>
__global__ __launch_bounds__(NW * WPT * 64)
__attribute__((amdgpu_waves_per_eu(D * sizeof(T) >= 256 ? (WPT == 1 ? 1 : 2) : WPT == 1 ? 2 : 4)))
void tree_attn_kernel(ArgsOf<PRE> args) {
  constexpr int ST = TreeCfg<T, D>::ST;
  __shared__ __attribute__((aligned(1024))) char smem[tree_lds<T, D, NW, WPT, ST>()];
  tree_work<T, D, NW, WPT, ST, CAP, PRE ? kBoth : kTree>(args, smem, blockIdx.x);
}

// The prefix with eight row tiles a workgroup, a wave each, where there are as many: 64-key
// tiles copied by all eight waves into four stages, three ahead, and the two waves of a SIMD
// a phase apart, one in its products (O += P V of a tile and the scores of the next) while
// the other has its softmax, with a barrier after each phase.  16384 prefix rows more for 128
// tokens of Hq=32 Hkv=8 D=128 are 45 us with four waves that share 32-key tiles, 37 here
// (0.92 PFLOP/s; the regular forward reaches 1.07 at fp16).
template <class T, int D, bool CAP>
__device__ __forceinline__ void prefix_rows(const PrefixArgs& args, char* smem) {
  using C = TreeCfg<T, D>;
  typedef typename Mfma<T>::v8 V8;
  constexpr int BN = 64, NB = 2, TILEB = BN * C::ROWB, E = TILEB / 8192, CROWS = 8 * E * C::RPC, AHEAD = 2;
  static_assert(CROWS == BN && NB * C::KC == 4 * C::DB, "tiles");
  const TreeArgs& a = args.t;
  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rt = (int)blockIdx.x / 8 % args.nrtp * 8 + wave, x = (int)blockIdx.x / (8 * args.nrtp) * 8 + (int)blockIdx.x % 8;
  if (x >= p.Hkv * args.np) return;
  const TreeChunk ck = prefix_chunk<2>(args, x);
  const int hk = ck.hk, first = ck.first / 2, nv = (ck.count + 1) / 2;

  // packed query row of this lane: head, drafted token, sequence
  const int R = p.B * p.G * p.Sq, r = min(32 * rt + l32, R - 1);
  const int hq = hk * p.G + r % p.G, qb = r / p.G / p.Sq, qi = r / p.G - qb * p.Sq;
  i32x4 qf[C::KC];
  const char* src = (const char*)((const T*)a.q.data + qb * a.q.sb + hq * a.q.sh + (int64_t)qi * a.q.ss) + 16 * h;
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) qf[kc] = ld_global16(src + 32 * kc);

  int koff[C::KC], voff[C::DB];
  const int tr_row = 4 * h + ((lane & 15) >> 2), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) koff[kc] = l32 * C::ROWB + swz_col<C::CPR>(l32, 2 * kc + h) * 16;
#pragma unroll
  for (int db = 0; db < C::DB; ++db)
    voff[db] = tr_row * C::ROWB + swz_tr<C::CPR>(tr_row, 4 * db + (tr_col >> 3)) * 16 + (tr_col & 7) * 2;
  const unsigned kss = (unsigned)(args.k.ss * (int)sizeof(T)), vss = (unsigned)(args.v.ss * (int)sizeof(T));
  const int crow = wave * E * C::RPC + lane / C::CPR, cchunk = lane % C::CPR;
  unsigned kvo[E], vvo[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int row = crow + e * C::RPC;
    kvo[e] = row * kss + swz_col<C::CPR>(row, cchunk) * 16;
    vvo[e] = row * vss + swz_v<T, C::CPR>(row, cchunk) * 16;
  }
  const unsigned lds0 = lds_addr_of(smem) + wave * E * 1024;
  const uint64_t kp = (uint64_t)((const T*)args.k.data + hk * args.k.sh), vp = (uint64_t)((const T*)args.v.data + hk * args.v.sh);
  // Tile v of the chunk into stage v % 4; behind the last one that again, so that every wait
  // is for the same number of copies.
  auto issue = [&](int v) {
    const unsigned dst = lds0 + (v & 3) * 2 * TILEB;
    const int n0 = (first + min(v, nv - 1)) * BN;
    const uint64_t kb = kp + (uint64_t)n0 * kss, vb = vp + (uint64_t)n0 * vss;
    if (n0 + BN <= args.P) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        load_lds16_base(kvo[e], kb, dst + e * 1024);
        load_lds16_base(vvo[e], vb, dst + e * 1024 + TILEB);
      }
    } else {  // rows behind the last one repeat it
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const int row = crow + e * C::RPC, at = min(row, args.P - 1 - n0);
        load_lds16_base(at * kss + swz_col<C::CPR>(row, cchunk) * 16, kb, dst + e * 1024);
        load_lds16_base(at * vss + swz_v<T, C::CPR>(row, cchunk) * 16, vb, dst + e * 1024 + TILEB);
      }
    }
  };
  auto landed = [] { wait_vmcnt<2 * E>(); };

  if (nv > 0) {
    issue(0);
    issue(1);
  }

  // rows of the prefix this lane's row sees: from row_lo on (tree_work)
  int row_lo = 0, full_lo = 0;
  if (p.window > 0) {
    const int depth = a.depths ? max(a.depths[(int64_t)qb * p.Sq + qi], 0) : qi;
    const int past = args.P + min(max(a.lengths[qb], 0), p.Skv);
    full_lo = row_lo = max(past - (p.window - min(depth, p.window)), 0);
#pragma unroll
    for (int y = 32; y; y >>= 1) full_lo = max(full_lo, __shfl_xor(full_lo, y));
    full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  }
  float c2 = p.scale_log2;
  int flip = 0;
  if constexpr (!CAP) {
    if (c2 < 0.f) flip = (int)0x80008000;
    c2 = c2 == 0.f ? 1e-30f : fabsf(c2);
  }
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) {
    qf[kc] ^= i32x4{flip, flip, flip, flip};
    pin(qf[kc]);
  }

  f32x16 acc[C::DB], sc[NB];
  V8 P[2 * NB];
  float m_run = kNegInf, l_run = 0.f;
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x16{};
  auto softmax = [&](int n0) {
    if constexpr (CAP) {
#pragma unroll
      for (int bb = 0; bb < NB; ++bb) {
        soft_cap(sc[bb], p);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[bb][e] *= p.cap_log2;
      }
    }
    if (n0 < full_lo || n0 + BN > args.P) {
      const int lo = row_lo - n0 - 4 * h, hi = args.P - n0 - 4 * h;
#pragma unroll
      for (int bb = 0; bb < NB; ++bb) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((unsigned)(32 * bb + 8 * (e >> 2) + (e & 3) - lo) >= (unsigned)max(hi - lo, 0)) sc[bb][e] = kNegInf;
        pin(sc[bb]);  // finished inside the branch (no selects after it)
      }
    }
    if constexpr (!CAP) settle(sc[0], sc[1]);  // (as in tree_work)
    float mp[4];
#pragma unroll
    for (int bb = 0; bb < NB; ++bb) max16_partial(sc[bb], mp[2 * bb], mp[2 * bb + 1]);
    float mx = max2(max3(mp[0], mp[1], mp[2]), mp[3]);
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
    for (int bb = 0; bb < NB; ++bb) {
      f32x16 pe;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if constexpr (!CAP) pe[e] = fast_exp2(__builtin_fmaf(sc[bb][e], c2, -m_use));
        else pe[e] = fast_exp2(sc[bb][e] - m_use);
        rs[e & 3] += pe[e];
      }
      P[2 * bb] = pack8<T>(pe, 0);
      P[2 * bb + 1] = pack8<T>(pe, 8);
    }
    l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    // done before the barrier
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) pin(P[i]);
    pin(l_run);
  };
  // what a phase reads is read after the barrier that ends its producer
  auto pin_s = [&] {
#pragma unroll
    for (int bb = 0; bb < NB; ++bb) pin(sc[bb]);
  };
  auto pin_p = [&] {
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) pin(P[i]);
  };
  // O += P V of tile v and the scores of tile w (either < 0: not), their MFMAs in turn so
  // that neither waits for its own, LDS reads AHEAD pairs before them
  auto products = [&](int v, int w, auto both) {
    const char* sV = smem + (v & 3) * 2 * TILEB + TILEB;
    const char* sK = smem + (w & 3) * 2 * TILEB;
    if (both || w >= 0) {
#pragma unroll
      for (int bb = 0; bb < NB; ++bb) sc[bb] = f32x16{};
    }
#pragma unroll
    for (int i = 0; i < NB * C::KC; ++i) {
      if (both || v >= 0) {
        const int db = i % C::DB, c = i / C::DB;
        const char* vr = sV + 16 * c * C::ROWB + voff[db];
        const i16x4 lo = lds_read_tr4(vr), hi = lds_read_tr4(vr + 8 * C::ROWB);
        acc[db] = Mfma<T>::mma(cat_tr<V8>(lo, hi), P[c], acc[db]);
      }
      if (both || w >= 0) {
        const int bb = i % NB, kc = i / NB;
        sc[bb] = Mfma<T>::mma(as_v8<V8>(lds_read16(sK + bb * 32 * C::ROWB + koff[kc])), as_v8<V8>(qf[kc]), sc[bb]);
      }
    }
    if constexpr (both) {
      __builtin_amdgcn_sched_group_barrier(0x100, 3 * AHEAD, 2);
#pragma unroll
      for (int i = 0; i < NB * C::KC - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 2);
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 2);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2 * AHEAD, 2);
    }
  };

  // Stage v % 4 has tile v from its copy, issued when the products of tiles v - 4 and v - 3
  // begin, which is after the barrier behind every wave's last read of tile v - 4.
  if (nv > 0) {
    const bool late = wave >= 4;
    landed();
    __syncthreads();
    if (late) __syncthreads();  // the second half starts a phase later
    issue(2);
    products(-1, 0, std::false_type{});
    landed();
    __syncthreads();
    pin_s();
    for (int v = 0; v + 1 < nv; ++v) {
      softmax((first + v) * BN);
      landed();
      __syncthreads();
      pin_p();
      __builtin_amdgcn_s_setprio(1);
      issue(v + 3);
      products(v, v + 1, std::true_type{});
      __builtin_amdgcn_s_setprio(0);
      landed();
      __syncthreads();
      pin_s();
    }
    softmax((first + nv - 1) * BN);
    landed();
    __syncthreads();
    pin_p();
    products(nv - 1, -1, std::false_type{});
    wait_vmcnt<0>();  // no copy may land after the workgroup's LDS is released
    __syncthreads();
    if (!late) __syncthreads();  // the first half matches the second's count
  }

  const float L = l_run + swap_halves(l_run);
  const bool empty = L == 0.f;  // no key; NaN is not
  const float inv = empty ? 0.f : 1.0f / L;
  if (32 * rt + l32 < R) {
    const int64_t place = (((int64_t)qb * p.Hq + hq) * p.Sq + qi) * args.pitch + ck.s;
    float* po = a.part_o + place * D + 4 * h;
#pragma unroll
    for (int y = 0; y < 4 * C::DB; ++y) {
      const f32x16& v = acc[y / 4];
      const int e = y % 4 * 4;
      *(f32x4*)(po + 8 * y) = f32x4{v[e] * inv, v[e + 1] * inv, v[e + 2] * inv, v[e + 3] * inv};
    }
    if (h == 0) a.part_lse[place] = empty ? kNegInf : m_run + log2f(L);
  }
}
constexpr int kWide = 8;  // waves of its workgroup

// With it the sequences' own caches, a row tile or two each: a wave takes every eighth tile
// (a wave in four had rows where four waves share their tiles: own caches of 1000 rows alone
// 34 -> 32 us).
template <class T, int D, bool CAP>
__global__ __launch_bounds__(kWide * 64) __attribute__((amdgpu_waves_per_eu(2)))
void prefix_wide_kernel(PrefixArgs args) {
  constexpr int ST = 1, own = tree_lds<T, D, kWide, 1, ST>(), all = 4 * 2 * 64 * D * (int)sizeof(T);
  __shared__ __attribute__((aligned(1024))) char smem[own > all ? own : all];
  if ((int)blockIdx.x < args.npre) prefix_rows<T, D, CAP>(args, smem);
  else tree_work<T, D, kWide, 1, ST, CAP, kOwn>(args, smem, blockIdx.x - args.npre);
}

template <class T, int D, int WPT>
void launch_tree_share(TreeArgs a, hipStream_t st) {
  constexpr int NW = WPT == 4 ? TreeCfg<T, D>::NW / 2 : TreeCfg<T, D>::NW;
  a.nrt = (int)((((int64_t)a.p.G * a.p.Sq + 31) / 32 + WPT - 1) / WPT);
  const dim3 grid((unsigned)((a.nchunk + 7) / 8 * 8 * a.nrt)), block(NW * WPT * 64);
  if (a.p.cap > 0.f) hipLaunchKernelGGL((tree_attn_kernel<T, D, NW, WPT, true, false>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((tree_attn_kernel<T, D, NW, WPT, false, false>), grid, block, 0, st, a);
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

template <class T, int D, int WPT>
void launch_prefix_share(PrefixArgs a, hipStream_t st) {
  constexpr int NW = WPT == 4 ? TreeCfg<T, D>::NW / 2 : TreeCfg<T, D>::NW;
  const int64_t rows = (int64_t)a.t.p.G * a.t.p.Sq;
  a.t.nrt = (int)(((rows + 31) / 32 + WPT - 1) / WPT);
  a.nrtp = (int)(((rows * a.t.p.B + 31) / 32 + WPT - 1) / WPT);
  a.npre = (a.t.p.Hkv * a.np + 7) / 8 * 8 * a.nrtp;
  const dim3 grid((unsigned)(a.npre + (a.t.nchunk + 7) / 8 * 8 * a.t.nrt)), block(NW * WPT * 64);
  if (a.t.p.cap > 0.f) hipLaunchKernelGGL((tree_attn_kernel<T, D, NW, WPT, true, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((tree_attn_kernel<T, D, NW, WPT, false, true>), grid, block, 0, st, a);
}

template <class T, int D>
void launch_prefix_wide(PrefixArgs a, hipStream_t st) {
  const int64_t rows = (int64_t)a.t.p.G * a.t.p.Sq;
  a.t.nrt = (int)((rows + 31) / 32);
  a.nrtp = (int)(((rows * a.t.p.B + 31) / 32 + kWide - 1) / kWide);
  a.npre = (a.t.p.Hkv * a.np + 7) / 8 * 8 * a.nrtp;
  const dim3 grid((unsigned)(a.npre + (a.t.nchunk + 7) / 8 * 8 * a.t.nrt)), block(kWide * 64);
  if (a.t.p.cap > 0.f) hipLaunchKernelGGL((prefix_wide_kernel<T, D, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((prefix_wide_kernel<T, D, false>), grid, block, 0, st, a);
}

template <class T, int D>
hipError_t launch_prefix(const PrefixArgs& a, hipStream_t st) {
  using C = TreeCfg<T, D>;
  int share = tree_share(C::ROWB, sizeof(T), ((int64_t)a.t.p.B * a.t.p.G * a.t.p.Sq + 31) / 32);
  if constexpr (sizeof(T) == 2 && C::ROWB == 256) {
    if (a.wide) {
      launch_prefix_wide<T, D>(a, st);
      share = 0;
    }
  }
  if constexpr (sizeof(T) == 2 && C::ROWB <= 256) {
    if constexpr (C::ROWB == 256) {
      if (share == 4) launch_prefix_share<T, D, 4>(a, st);
    }
    if (share == 2) launch_prefix_share<T, D, 2>(a, st);
  }
  if (share == 1) launch_prefix_share<T, D, 1>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = (int64_t)a.t.p.B * a.t.p.Hq * a.t.p.Sq;
  TreeArgs m = a.t;
  m.nsplit = a.pitch;
  hipLaunchKernelGGL((tree_merge_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, m);
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
hipError_t FLEXATT_CAT(prefix_attn_bf16_d, FLEXATT_D)(const PrefixArgs& a, hipStream_t st) {
  return launch_prefix<__bf16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(prefix_attn_f16_d, FLEXATT_D)(const PrefixArgs& a, hipStream_t st) {
  return launch_prefix<_Float16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(prefix_attn_f32_d, FLEXATT_D)(const PrefixArgs& a, hipStream_t st) {
  return launch_prefix<float, FLEXATT_D>(a, st);
}

}  // namespace flexatt
