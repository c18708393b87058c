// Attention of a tree of drafted tokens over a K/V cache of 8 bits (norm_rotary.hip writes
// it): the semantics, the chunks of key tiles and their merge are those of tree_attn.hip.
// No counterpart in the reference, which has no cache.
//
// With codes c_j, c'_j and scales s_j, s'_j of key j's row of K and V,
//   x_ij = scale s_j (q_i . c_j),   o_i = sum_j (p_ij s'_j) c'_j / sum_j p_ij,
// so a scale meets a score and a weight, never an element.  Codes of either kind are exact
// in bf16 and fp16, the types of the MFMAs, and are converted on the way to them:
//  * K: a lane has 16 codes of its key in one LDS read, the operands of two MFMAs; which
//    k of the products they are is the same for Q's fragments, which are loaded to match;
//  * V: the transpose read of 8-bit elements gives a lane eight keys of its column, those
//    whose weights the scores' accumulators hold.
// p s' is rounded to fp16 for either type of queries, in which codes are exact: its half
// step of 2^-11 is far under that of bf16 outputs (bf16 weights: rms errors of 1.3 to 1.6
// times the output's rounding alone, fp16 ones 1.01).  For fp16 outputs, where it would be as
// much as theirs (1.3 to 1.5 times), what the rounding leaves is the operand of MFMAs of its
// own, which a wave that waits for memory has time for.  fp16's range: what is rounded is the
// weight relative to the running maximum, times 2^lift, with 2^lift times the largest scale that
// a row has met in a wave between 2^6 and 2^7, and so are the accumulators (scales that a row
// does not see are 0 for it, whatever they are); the sum of weights is relative
// to the maximum alone, since values of zeros (scales of 2^-109) beside ones of 2^75 would leave
// 32 bits with it.  2^lift is part of the weights' exponents up to 2^-32 and 2^32, of the scales
// beyond.  The running maximum is a whole number, so that sums and accumulators follow it exactly.
//
// A wave has one row tile of 32 packed query rows and every NW-th 32-key tile of its
// workgroup's chunk in LDS stages of its own, without barriers, the scales with one copy
// more.  The scores of the next tile, whose conversions and MFMAs wait for nothing, stand
// between this one's weights and in front of its second product, and a tile's LDS reads at its
// start (bf16 e4m3 B=8 Hq=32 Hkv=8 D=128, caches of 24576 to 32768: T=1 100 -> 96 us).  Row
// tiles are workgroups of their own, whose chunk comes from the XCD's L2 after the first:
// waves that share a tile's copies wait for each other (T=16, two row tiles, 122 and 125 us;
// T=24 270 -> 180, 171 now, T=16 over one cache of 4096 17.9 -> 15.2).
//
// Bound by HBM for one row tile over long caches (4.9 TB/s there), by the work on a tile from
// two on: at T=16, 117 us, VALU instructions, of which the conversions are a third, issue in
// 0.52 of the cycles and MFMAs run in 0.25, and a wave cannot issue for 0.29 of its time, for what
// is not known (copies further ahead and fewer instructions changed nothing, a raised priority
// of the products 5%); by latency for short caches, whose code is fetched once for a few tiles.
//   fp16 e4m3 the same caches, T=16: 136 us (with the rest's MFMAs; VALU 0.59, MFMAs 0.34)
//   fp16 int8 B=4 Hq=28 Hkv=4 T=64, caches of 16384: 126 us; bf16 D=64 81
//   bf16 e4m3 B=4 Hq=16 Hkv=8 T=1, caches of 16000, D=256: 57 us
//   fp16 int8 B=2 Hq=16 Hkv=8 T=16, window 4096, soft-cap 50, D=256: 26 us
//   bf16 e4m3 B=1 Hq=32 Hkv=8 T=1, a cache of 4097, D=128: 12 to 14 us (9.3 and the merge 4)
// Equal shares of all key tiles for the workgroups, in place of equal chunks of each
// sequence, shorten the longest by an eighth and change nothing (T=16 121 -> 123).
#include <type_traits>

#include "flexatt_device.h"
#include "flexatt_kernels.h"
#include "tree_device.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
template <int D>
struct QuantCfg {
  static constexpr int BN = 32;              // keys per tile
  static constexpr int KC = D / 32;          // 32-byte steps of S^T = K Q^T, two MFMAs each
  static constexpr int DB = D / 32;          // 32-row blocks of O^T
  static constexpr int CPR = D / 16;         // 16-byte chunks per row
  static constexpr int RPC = 64 / CPR;       // rows per 1 KB copy
  static constexpr int TB = BN * D;          // bytes of one K or V tile
  static constexpr int E = TB / 1024;        // copies of one
  static constexpr int PK = RPC >= 16 ? 1 : 16 / RPC;  // copies after which K's swizzle repeats
  static constexpr int PV = RPC >= 8 ? 1 : 8 / RPC;    // and V's
  static_assert(E * 1024 == TB && E % PK == 0 && E % PV == 0, "tiles");
};

// K is read 16 bytes a lane from 32 rows, V by transpose reads of 32 bytes of 16 rows
// (rows 16 c + 0..15 of a block of 32 columns); both spread evenly over the banks.
template <int CPR>
__device__ __forceinline__ int swz_k8(int r, int c) {
  if constexpr (CPR == 2) return c ^ ((r >> 3) & 1);
  else return swz_col<CPR>(r, c);
}
template <int CPR>
__device__ __forceinline__ int swz_v8(int r, int c) {
  if constexpr (CPR == 2) return c;
  else if constexpr (CPR == 4) return c ^ (((r >> 2) & 1) << 1);
  else if constexpr (CPR == 8) return c ^ (((r >> 1) & 3) << 1);
  else return c ^ ((r & 7) << 1);
}

// What 2^lift times a scale may reach: weights reach 2^8.5 before the maximum follows
// (kTreeRescale), and fp16 ends at 2^16.
constexpr float kMostScale = 0x1p7f;
// The part of a lift that the weights' exponents have.
constexpr float kMostUp = 32.f;

// Eight codes as an MFMA operand of T.
template <class T, int CODE>
__device__ __forceinline__ typename Mfma<T>::v8 operand8(int lo, int hi) {
  typedef T x2 __attribute__((ext_vector_type(2)));
  x2 p[4];
  if constexpr (CODE == FLEXATT_E4M3) {
    if constexpr (__is_same(T, __bf16)) {
      p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
      p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    } else {
      p[0] = __builtin_bit_cast(x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
      p[1] = __builtin_bit_cast(x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
      p[2] = __builtin_bit_cast(x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
      p[3] = __builtin_bit_cast(x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    }
  } else if constexpr (__is_same(T, __bf16)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int w = i < 2 ? lo : hi;
      p[i] = x2{(T)(float)(signed char)(w >> (16 * (i & 1))), (T)(float)(signed char)(w >> (16 * (i & 1) + 8))};
    }
  } else {
    // 0x6400 + u is 1024 + u in fp16, u = code + 128
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = (unsigned)(i < 2 ? lo : hi) ^ 0x80808080u;
      const unsigned w = __builtin_amdgcn_perm(0x64646464u, u, i & 1 ? 0x04030402u : 0x04010400u);
      p[i] = __builtin_bit_cast(x2, w) - x2{(T)1152.f, (T)1152.f};
    }
  }
  const i32x4 v = {__builtin_bit_cast(int, p[0]), __builtin_bit_cast(int, p[1]), __builtin_bit_cast(int, p[2]),
                   __builtin_bit_cast(int, p[3])};
  return as_v8<typename Mfma<T>::v8>(v);
}

// x 2^n, n a whole number.
__device__ __forceinline__ float ldexp(float x, float n) { return __builtin_amdgcn_ldexpf(x, (int)n); }

// acc *= s.  Accumulators of head dim 256 are kept in the other half of the register file:
// a multiply of its own would have all of them moved there and back around the branch it
// is in, in every iteration.  The caller has waited for the last MFMA's result; the wait at
// the end is that between a write and an MFMA.
template <int D>
__device__ __forceinline__ void rescale(f32x16& a, float s) {
  if constexpr (D < 256) {
    scale_inplace(a, s);
  } else {
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      float x0, x1, x2, x3, y0 = a[r], y1 = a[r + 1], y2 = a[r + 2], y3 = a[r + 3];
      asm volatile(
          "v_accvgpr_read_b32 %4, %0\n\tv_accvgpr_read_b32 %5, %1\n\t"
          "v_accvgpr_read_b32 %6, %2\n\tv_accvgpr_read_b32 %7, %3\n\ts_nop 1\n\t"
          "v_mul_f32_e32 %4, %8, %4\n\tv_mul_f32_e32 %5, %8, %5\n\t"
          "v_mul_f32_e32 %6, %8, %6\n\tv_mul_f32_e32 %7, %8, %7\n\ts_nop 1\n\t"
          "v_accvgpr_write_b32 %0, %4\n\tv_accvgpr_write_b32 %1, %5\n\t"
          "v_accvgpr_write_b32 %2, %6\n\tv_accvgpr_write_b32 %3, %7\n\ts_nop 3"
          : "+a"(y0), "+a"(y1), "+a"(y2), "+a"(y3), "=&v"(x0), "=&v"(x1), "=&v"(x2), "=&v"(x3)
          : "v"(s));
      a[r] = y0, a[r + 1] = y1, a[r + 2] = y2, a[r + 3] = y3;
    }
  }
}

// Transposed 8 x 8-bit read: lane i of 16 gets byte i % 8 at the addresses of lanes
// 2 t + i / 8, t = 0 .. 7.
__device__ __forceinline__ i32x2 lds_read_tr8(const void* p) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (__attribute__((address_space(3))) i32x2*)((__attribute__((address_space(3))) char*)p));
}

template <class T, int CODE, int D, int NW, int ST, bool CAP>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(D >= 256 ? 1 : 2)))
void quant_attn_kernel(QuantTreeArgs qa) {
  using C = QuantCfg<D>;
  typedef typename Mfma<T>::v8 V8;
  typedef _Float16 W;  // the weights' type
  constexpr bool REST = __is_same(T, _Float16);  // and what their rounding leaves
  constexpr int EC = 2 * C::E + 1;               // copies of a stage: K, V and the scales
  constexpr int SCB = 128;                       // bytes from K's scales to V's
  constexpr int STB = 2 * C::TB + 2 * SCB;       // bytes of a stage
  static_assert(ST >= 2 && NW * ST * STB <= 160 * 1024, "stages");
  constexpr int kCombine = NW * 64 * 4 * (3 + 16 * C::DB);
  __shared__ __attribute__((aligned(1024))) char smem[NW * ST * STB > kCombine ? NW * ST * STB : kCombine];

  const TreeArgs& a = qa.t;
  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // its key tiles
  const int h = lane >> 5, l32 = lane & 31;

  // (chunk, row tiles): as in tree_attn.hip
  int rt0 = 0, x = blockIdx.x;
  if (a.nrt > 1) {
    rt0 = blockIdx.x / 8 % a.nrt;
    x = blockIdx.x / (8 * a.nrt) * 8 + blockIdx.x % 8;
  }
  const TreeChunk ck = tree_chunk(a, x, NW);
  if (ck.b < 0) return;
  const int b = ck.b, hk = ck.hk, s = ck.s, ns = ck.ns;
  TreeSeq sq = tree_seq(a, b);
  sq.n = __builtin_amdgcn_readfirstlane(sq.n);
  sq.t0 = __builtin_amdgcn_readfirstlane(sq.t0);
  if (rt0 == 0 && s == 0 && tid == 0 && a.counts) a.counts[b * p.Hkv + hk] = sq.bad ? 1 : ns;

  // packed query row of this lane: head, drafted token
  const int R = p.G * p.Sq;
  const int r = min(32 * rt0 + l32, R - 1);
  const int hq = hk * p.G + r % p.G, qi = r / p.G;
  if (sq.bad) {
    if (s == 0 && 32 * rt0 + l32 < R) {
      T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss;
      for (int d = wave * 2 + h; d < D; d += NW * 2) out[d] = from_f32<T>(__builtin_nanf(""));
      if (wave == 0 && h == 0) a.lse[((int64_t)b * p.Hq + hq) * p.Sq + qi] = __builtin_nanf("");
    }
    return;
  }

  int koff[C::KC], voff[C::DB];
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) koff[kc] = l32 * D + swz_k8<C::CPR>(l32, 2 * kc + h) * 16;
  {
    const int t = (lane & 15) >> 1, row = 4 * h + (t & 3) + 2 * (t & 4);  // keys 4 h + 0..3, 8 + 4 h + 0..3
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
      voff[db] = row * D + swz_v8<C::CPR>(row, 2 * db + ((lane >> 4) & 1)) * 16 + (lane & 1) * 8;
  }
  // this lane's offsets in a tile's copies
  const unsigned kss = (unsigned)a.k.ss, vss = (unsigned)a.v.ss;
  const int crow = lane / C::CPR, cchunk = lane % C::CPR;
  unsigned kvo[C::PK], vvo[C::PV];
#pragma unroll
  for (int e = 0; e < C::PK; ++e) kvo[e] = (e * C::RPC + crow) * kss + swz_k8<C::CPR>(e * C::RPC + crow, cchunk) * 16;
#pragma unroll
  for (int e = 0; e < C::PV; ++e) vvo[e] = (e * C::RPC + crow) * vss + swz_v8<C::CPR>(e * C::RPC + crow, cchunk) * 16;
  const unsigned wbase = lds_addr_of(smem) + wave * (ST * STB);
  // this wave's LDS reads have returned: the buffer they read may be refilled
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

  // this wave's tiles: first + NW * j, j < nt
  const int n = sq.n, last = n + p.Sq - 1;
  const int first = sq.t0 + ck.first + wave;
  const int nt = __builtin_amdgcn_readfirstlane(max((ck.count - wave + NW - 1) / NW, 0));
  const uint64_t kp = (uint64_t)((const char*)a.k.data + b * a.k.sb + hk * a.k.sh);
  const uint64_t vp = (uint64_t)((const char*)a.v.data + b * a.v.sb + hk * a.v.sh);
  // (both tensors' scales in one copy, 32 lanes each)
  const float* scales = (h ? qa.v_scales : qa.k_scales) + ((int64_t)b * p.Hkv + hk) * p.Skv;
  // K, and V with the scales, of tile j of this wave into its stage
  auto issue_k = [&](int j) {
    const int t = first + NW * j;
    const unsigned dst = wbase + j % ST * STB;
    const uint64_t base = kp + (uint64_t)(t * C::BN) * kss;
    if (t * C::BN + C::BN - 1 <= last) {
#pragma unroll
      for (int e = 0; e < C::E; ++e)
        load_lds16_base(kvo[e % C::PK], base + (uint64_t)(e / C::PK * C::PK * C::RPC) * kss, dst + e * 1024);
    } else {  // rows behind the last one repeat it
#pragma unroll 1
      for (int e = 0; e < C::E; ++e) {
        const int kr = e * C::RPC + crow;
        load_lds16_base(min(kr, last - t * C::BN) * kss + swz_k8<C::CPR>(kr, cchunk) * 16, base, dst + e * 1024);
      }
    }
  };
  auto issue_v = [&](int j) {
    const int t = first + NW * j;
    const unsigned dst = wbase + j % ST * STB + C::TB;
    const uint64_t base = vp + (uint64_t)(t * C::BN) * vss;
    if (t * C::BN + C::BN - 1 <= last) {
#pragma unroll
      for (int e = 0; e < C::E; ++e)
        load_lds16_base(vvo[e % C::PV], base + (uint64_t)(e / C::PV * C::PV * C::RPC) * vss, dst + e * 1024);
    } else {
#pragma unroll 1
      for (int e = 0; e < C::E; ++e) {
        const int kr = e * C::RPC + crow;
        load_lds16_base(min(kr, last - t * C::BN) * vss + swz_v8<C::CPR>(kr, cchunk) * 16, base, dst + e * 1024);
      }
    }
    load_lds4(scales + min(t * C::BN + l32, last), wbase + j % ST * STB + 2 * C::TB);
  };
  // Q: lane half h has elements 32 kc + 16 h .. + 15 of its row, the codes' order
  i32x4 qf[2 * C::KC];
  const char* src = (const char*)((const T*)a.q.data + b * a.q.sb + hq * a.q.sh + (int64_t)qi * a.q.ss) + 32 * h;
#pragma unroll
  for (int kc = 0; kc < 2 * C::KC; ++kc) qf[kc] = ld_global16(src + 64 * (kc >> 1) + 16 * (kc & 1));
  if (nt > 0) {
    issue_k(0);
    issue_v(0);
  }
  // Row qi sees the cached keys [row_lo, n); the tiles that hold only keys every row
  // sees need no mask.
  int row_lo = 0, full_lo = 0;
  if (p.window > 0) {
    const int depth = a.depths ? max(a.depths[(int64_t)b * p.Sq + qi], 0) : qi;
    full_lo = row_lo = max(n - (p.window - min(depth, p.window)), 0);
#pragma unroll
    for (int y = 32; y; y >>= 1) full_lo = max(full_lo, __shfl_xor(full_lo, y));
    full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  }
  const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  float c2 = p.scale_log2;
  int flip = 0;
  if constexpr (!CAP) {  // as in the forward: a negative scale moves into Q
    if (c2 < 0.f) flip = (int)0x80008000;
    c2 = c2 == 0.f ? 1e-30f : fabsf(c2);
  }
  // wait for Q here, once: see fwd_split.hip
#pragma unroll
  for (int kc = 0; kc < 2 * C::KC; ++kc) {
    qf[kc] ^= i32x4{flip, flip, flip, flip};
    pin(qf[kc]);
  }
  wait_vmcnt<0>();  // (and the first tile)
#pragma unroll 1  // (a short call's time is its code's)
  for (int j = 1; j < min(nt, ST); ++j) {
    issue_k(j);
    issue_v(j);
  }

  f32x16 acc[C::DB];
  float m_run = kNegInf, l_run = 0.f;
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x16{};
  // acc is relative to 2^(m_run - lift), l_run to 2^m_run; weights are 2^(x - m_run + up), up the
  // lift as far as kMostUp, and 2^lift times a scale is at most kMostScale
  float lift = 126.f, up = kMostUp;
  bool far = true;  // up is not all of it

  // K of tile j + 1, and all that was issued before it, lands.  What may be in flight
  // behind it, as far as there are tiles: V of that tile and up to ST - 2 whole tiles.
  auto landed = [&](int j) {
    constexpr int N = ST - 2, X = C::E + 1;
    static_assert(N <= 2, "stages");
    const int more = nt - 2 - j;  // tiles behind tile j + 1
    if (more >= N) wait_vmcnt<N * EC + X>();
    else if (N > 1 && more == 1) wait_vmcnt<EC + X>();
    else if (more == 0) wait_vmcnt<X>();
    else wait_vmcnt<0>();
  };
  // K's fragments of tile j, and S^T from them: codes alone
  auto read_k = [&](int j, i32x4 (&kf)[C::KC]) {
    const char* sK = smem + wave * (ST * STB) + j % ST * STB;
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) kf[kc] = lds_read16(sK + koff[kc]);
  };
  auto scores = [&](const i32x4 (&kf)[C::KC]) {
    f32x16 sc = f32x16{};
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      sc = Mfma<T>::mma(operand8<T, CODE>(kf[kc][0], kf[kc][1]), as_v8<V8>(qf[2 * kc]), sc);
      sc = Mfma<T>::mma(operand8<T, CODE>(kf[kc][2], kf[kc][3]), as_v8<V8>(qf[2 * kc + 1]), sc);
    }
    return sc;
  };

  i32x4 kf[C::KC];
  read_k(0, kf);
  f32x16 sc = scores(kf);
  for (int j = 0; j < nt; ++j) {
    const int n0 = (first + NW * j) * C::BN;
    // K of tile j + 1 and V of tile j land; what has been read is refilled
    landed(j);
    if (j + ST < nt) {
      reads_done();
      issue_k(j + ST);
    }
    const char* sV = smem + wave * (ST * STB) + j % ST * STB + C::TB;
    const char* sS = sV + C::TB + 16 * h;
    // scales of this lane's keys: element e is key n0 + 8(e/4) + 4h + e%4
    f32x16 ks, vs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const i32x4 k4 = lds_read16(sS + 32 * i), v4 = lds_read16(sS + SCB + 32 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) ks[4 * i + e] = __int_as_float(k4[e]), vs[4 * i + e] = __int_as_float(v4[e]);
    }
    // ... and all else that the tile reads, which is there when it is used
    i32x2 vf[2][C::DB];
    auto read_v = [&] {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int db = 0; db < C::DB; ++db) vf[c][db] = lds_read_tr8(sV + 16 * c * D + voff[db]);
    };
    if constexpr (D < 256) {  // (registers)
      read_k(j + 1, kf);
      read_v();
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] *= ks[e];
    if constexpr (CAP) {
      soft_cap(sc, p);
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] *= p.cap_log2;
    }
    if (n0 < full_lo || n0 + C::BN > n) {
      // this lane's keys, relative to its first: e, and hidden before lo or from hi on
      const int lo = row_lo - n0 - 4 * h, hi = n + (mask ? p.Sq : qi + 1) - n0 - 4 * h;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if ((unsigned)(8 * (e >> 2) + (e & 3) - lo) >= (unsigned)max(hi - lo, 0)) sc[e] = kNegInf, vs[e] = 0.f;
      if (mask && n0 + C::BN > n) {  // all of the tile's mask bytes at once
        const unsigned mrow = (unsigned)qi * (unsigned)p.Sq;
        const int u0 = n0 + 4 * h - n;
        unsigned char mb[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) mb[e] = mask[mrow + (unsigned)min(max(u0 + 8 * (e >> 2) + (e & 3), 0), p.Sq - 1)];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (u0 + 8 * (e >> 2) + (e & 3) >= 0 && mb[e] == 0) sc[e] = kNegInf, vs[e] = 0.f;
      }
    }
    float mx, mx2;
    max16_partial(sc, mx, mx2);
    mx = max2(mx, mx2);
    if constexpr (!CAP) mx *= c2;
    mx = fmaxf(mx, swap_halves(mx));
    if (mx != mx) mx = kNegInf;
    float top, top2;
    max16_partial(vs, top, top2);
    top = max2(top, top2);
    top = fmaxf(top, swap_halves(top));
    const bool grow = mx > m_run + kTreeRescale, over = ldexp(top, lift) > kMostScale;
    if (__builtin_amdgcn_ballot_w64(grow || over)) {
      // (over: the largest power of two with which the largest scale is below 2^7)
      const int expo = (int)(__float_as_uint(top) >> 23) & 255;
      const float now = over ? (float)min(max(133 - expo, -126), 126) : lift;
      const float m_new = grow ? __builtin_rintf(mx) : m_run;
      const float step = grow ? fast_exp2(m_run - m_new) : 1.f;
      if (j > 0) {  // (the first tile finds zeros)
        const float alpha = ldexp(step, now - lift);
        l_run *= step;
        settle(acc[0]);
#pragma unroll
        for (int db = 0; db < C::DB; ++db) rescale<D>(acc[db], alpha);
      }
      m_run = m_new;
      lift = now;
      up = fminf(fmaxf(lift, -kMostUp), kMostUp);
      far = __builtin_amdgcn_ballot_w64(up != lift) != 0;
    }
    if (far) {
#pragma unroll
      for (int e = 0; e < 16; ++e) vs[e] = ldexp(vs[e], lift - up);
    }
    const float m_use = (m_run == kNegInf ? 0.f : m_run) - up;

    // From here on one block: the next tile's scores (behind the last one of what is
    // there, and not used) between this one's weights, whose product follows.
    if constexpr (D == 256) {
      read_k(j + 1, kf);
      read_v();
    }
    // (ahead of the SIMD's other wave: bf16 e4m3 B=8 T=16 125 -> 119 us, fp16 int8 B=4 T=64
    // D=128 143 -> 132; the part in front of it raised instead 122 and 144)
    __builtin_amdgcn_s_setprio(1);
    const f32x16 next = scores(kf);
    float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float pe;
      if constexpr (!CAP) pe = fast_exp2(__builtin_fmaf(sc[e], c2, -m_use));
      else pe = fast_exp2(sc[e] - m_use);
      rs[e & 3] += pe;
      sc[e] = pe * vs[e];
    }
    l_run += ldexp((rs[0] + rs[1]) + (rs[2] + rs[3]), -up);
    // (products are numbers of 32 bits from here on: one rounded to fp16 in a fused step and, for
    // its rest, again by way of 32 bits, is another number in 1 of 10^4)
    if constexpr (REST) pin(sc);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Mfma<W>::v8 pb = pack8<W>(sc, 8 * c);
      Mfma<W>::v8 pl;
      if constexpr (REST) {
#pragma unroll
        for (int t = 0; t < 8; ++t) pl[t] = (W)(sc[8 * c + t] - (float)pb[t]);
      }
#pragma unroll
      for (int db = 0; db < C::DB; ++db) {
        const Mfma<W>::v8 v = operand8<W, CODE>(vf[c][db][0], vf[c][db][1]);
        acc[db] = Mfma<W>::mma(v, pb, acc[db]);
        if constexpr (REST) acc[db] = Mfma<W>::mma(v, pl, acc[db]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    sc = next;
    if (j + ST < nt) {
      reads_done();
      issue_v(j + ST);
    }
  }

  // The (m, l, acc) of a row tile's NW waves combined in wave order through LDS (every
  // wave's copies have landed: its last tile waited for vmcnt 0), then O / l and LSE.
  float* xm = (float*)smem;  // [NW][64]
  float* xl = xm + NW * 64;  // [NW][64]
  float* xu = xl + NW * 64;  // [NW][64]
  f32x4* xa = (f32x4*)(xu + NW * 64);  // [NW][4 DB][64]: columns 8 y + 4 h .. + 3 of row l32
  const float l_tot = l_run + swap_halves(l_run);
  __syncthreads();
  xm[wave * 64 + lane] = m_run;
  xl[wave * 64 + lane] = l_tot;
  xu[wave * 64 + lane] = m_run - lift;
#pragma unroll
  for (int y = 0; y < 4 * C::DB; ++y) {
    const f32x16& v = acc[y / 4];
    const int e = y % 4 * 4;
    xa[(wave * 4 * C::DB + y) * 64 + lane] = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
  }
  __syncthreads();
  float mw[NW], uw[NW], mall = kNegInf, uall = kNegInf;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    mw[w] = xm[w * 64 + lane];
    uw[w] = xu[w * 64 + lane];
    mall = fmaxf(mall, mw[w]);
    uall = fmaxf(uall, uw[w]);
  }
  float al[NW], L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    // a wave whose maximum stayed -inf has weights of 0, or NaN scores
    const float lw = xl[w * 64 + lane], none = lw == 0.f ? 0.f : 1.f;
    al[w] = mw[w] == kNegInf ? none : fast_exp2(uw[w] - uall);
    L = __builtin_fmaf(mw[w] == kNegInf ? none : fast_exp2(mw[w] - mall), lw, L);
  }
  const bool empty = L == 0.f;  // no key; NaN (a NaN query row or key) is not
  const float inv = empty ? 0.f : 1.0f / L, back = empty ? 0.f : uall - mall;
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
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = ldexp(o[e] * inv, back);
      if (ns > 1) *(f32x4*)(po + 8 * y) = o;
      else st_global8(out + 8 * y, pack4<T>(o[0], o[1], o[2], o[3]));
    }
    if (wave == 0 && h == 0) {
      const float lse = empty ? kNegInf : mall + log2f(L);
      if (ns > 1) a.part_lse[row * a.nsplit + s] = lse;
      else a.lse[row] = lse * kLn2;
    }
  }
}

// Eight waves of two stages at head dim 128, where LDS leaves a CU one workgroup (four of
// four: T=1 over the long caches above 96 -> 101 us, B=16 over 2000 rows 17 -> 20); four below,
// two workgroups of them; two stages at 256, for LDS.
template <class T, int CODE, int D>
void launch_code(QuantTreeArgs a, hipStream_t st) {
  constexpr int NW = quant_threads(D) / 64, ST = D >= 128 ? 2 : 4;
  a.t.nrt = (int)(((int64_t)a.t.p.G * a.t.p.Sq + 31) / 32);
  const dim3 grid((unsigned)((a.t.nchunk + 7) / 8 * 8 * a.t.nrt)), block(NW * 64);
  if (a.t.p.cap > 0.f) hipLaunchKernelGGL((quant_attn_kernel<T, CODE, D, NW, ST, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((quant_attn_kernel<T, CODE, D, NW, ST, false>), grid, block, 0, st, a);
}

template <class T, int D>
hipError_t launch_quant(const QuantTreeArgs& a, hipStream_t st) {
  if (a.kind == FLEXATT_E4M3) launch_code<T, FLEXATT_E4M3, D>(a, st);
  else launch_code<T, FLEXATT_INT8, D>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.t.nsplit == 1) return e;
  const int64_t rows = (int64_t)a.t.p.B * a.t.p.Hq * a.t.p.Sq;
  hipLaunchKernelGGL((tree_merge_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a.t);
  return hipGetLastError();
}
}  // namespace

#define FLEXATT_CAT2(a, b) a##b
#define FLEXATT_CAT(a, b) FLEXATT_CAT2(a, b)
hipError_t FLEXATT_CAT(quant_attn_bf16_d, FLEXATT_D)(const QuantTreeArgs& a, hipStream_t st) {
  return launch_quant<__bf16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(quant_attn_f16_d, FLEXATT_D)(const QuantTreeArgs& a, hipStream_t st) {
  return launch_quant<_Float16, FLEXATT_D>(a, st);
}

}  // namespace flexatt
