// The attention weight each key of a K/V cache has received: for key j of KV head
// hk the sum over the G query heads that share it and over the query rows i of
// P_ij = exp(x_ij - LSE_i), with the scores, masks and LSE of the forward
// (npu_flash_attention.py:17-166).  No counterpart in the reference.
//
// The column sums of P need LSE, so they follow the forward as a product of their
// own: half the forward's MFMAs, and as many exponentials.
//
// Decomposition
//  * key-stationary: a wave holds NK blocks of 32 keys as A operands in registers,
//    a workgroup of four waves kWsWaves * NK * 32 keys of one (b, hkv);
//  * the query rows of the KV head's G heads, packed with the heads innermost (row
//    r: query row r / G of head r % G), are streamed in tiles of 32, the columns of
//    an MFMA tile, through a ring of LDS stages that the four waves share
//    (direct-to-LDS copies, one barrier per step of two tiles, two steps ahead), and from
//    there into registers while the MFMAs of the tile before run;
//  * a lane adds the weights of its column's rows for 16 keys of each block in fp32;
//    the 32 columns are added at the end by exchanging halves, so that lane c ends
//    up with one key's sum, in a fixed order;
//  * the tiles of a key block are shared by nparts workgroups where key blocks alone
//    would leave CUs idle; their sums go to the workspace and a second kernel adds
//    them in order.
// What bounds it: per 32 x 32 pairs and SIMD the MFMAs are 2 D cycles (16-bit types),
// one fma, one exponential (half the rate) and one add an element 256 cycles of VALU, at
// the clock that the MFMAs' power leaves (1.9 GHz; zeros instead of numbers are 15%
// faster).  bf16 B=2 Hq=32 Hkv=8 S=4096 D=128 causal: 161 us, 0.85 PFLOP/s beside 3.3e12
// exponentials a second; without the exponentials it would be 142, without masks 151,
// without the copies of new tiles 150, without the LDS reads 158.  fp16 B=4 Hq=28 Hkv=4,
// 32 rows over 16383 keys, D=64: 22 us.
#include "flexatt_device.h"
#include "flexatt_kernels.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
constexpr int kWsWaves = 4;

template <class T, int D>
struct WsCfg {
  static constexpr int ROWB = D * (int)sizeof(T);  // bytes per row
  static constexpr int KC = ROWB / 32;             // 32-byte steps of S = K Q^T
  static constexpr int TB = 32 * ROWB;             // bytes of a query tile: KC copies of 1 KB
  static constexpr int NK = ROWB <= 512 ? 2 : 1;   // 32-key blocks per wave (registers)
  static constexpr int KEYS = kWsWaves * NK * 32;  // keys per workgroup
  static constexpr int STAGEB = TB + 256;          // a tile and its 32 rows' LSE (a 64-lane copy)
  static constexpr int TPS = ROWB <= 512 ? 2 : 1;  // tiles per barrier
  static constexpr int RING = 3 * TPS;             // stages
};

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

// A query tile in LDS is a block of 2 KB for each 64 bytes of its rows, 32 rows of 64
// bytes whose 16-byte chunks are permuted by (row / 4) % 4: the 16 rows that one LDS
// cycle of a column read takes hit 16 groups of banks, and a step's reads differ from
// the one two steps on by a constant.  A copy (1 KB) is 16 rows of a block; wave w
// makes copies w, w + 4, ...
template <int KC, int X>
__device__ __forceinline__ void copy_steps(const char* row, unsigned dst) {
  if constexpr (X < KC) {
    load_lds16_at<32 * X>(row, dst + X * 1024);
    copy_steps<KC, X + kWsWaves>(row, dst);
  }
}

// Adds the 32 columns of 16 values per lane half, one step per bit of the lane:
// lanes W apart exchange the halves of the 2 W values left, so that lane c of each
// half ends up with the sum of element c % 16 (lanes c and c ^ 16 both have it).
template <int W>
__device__ __forceinline__ void exchange(float (&x)[16], int l32) {
  const bool up = l32 & W;
#pragma unroll
  for (int e = 0; e < W; ++e) {  // keep the element whose bit W is this lane's
    const float send = up ? x[e] : x[e + W], keep = up ? x[e + W] : x[e];
    x[e] = keep + __shfl_xor(send, W);
  }
}
__device__ __forceinline__ float column_sums(const f32x16& a, int l32) {
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = a[e];
  exchange<8>(x, l32);
  exchange<4>(x, l32);
  exchange<2>(x, l32);
  exchange<1>(x, l32);
  return x[0] + __shfl_xor(x[0], 16);
}
}  // namespace

template <class T, int D, int NK, bool CAP>
__global__ __launch_bounds__(kWsWaves * 64) __attribute__((amdgpu_waves_per_eu(D * sizeof(T) >= 512 ? 1 : 2)))
void weight_sums_kernel(WeightArgs a) {
  using C = WsCfg<T, D>;
  constexpr int KC = C::KC;
  __shared__ __attribute__((aligned(1024))) char smem[C::RING * C::STAGEB];
  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;

  // (part, key block or pair of them, b, hkv).  A pair is block x and block nkb - 1 - x,
  // one after the other, so that under a causal mask, too, workgroups have equal work;
  // those of one (b, hkv) share an XCD where their number is a multiple of 8
  const int nbh = p.B * p.Hkv, nkb = (p.Skv + C::KEYS - 1) / C::KEYS, nx = a.pair ? (nkb + 1) / 2 : nkb;
  const int bh = blockIdx.x % nbh, hk = bh % p.Hkv, b = bh / p.Hkv;
  const int x0 = blockIdx.x / nbh % nx, part = blockIdx.x / nbh / nx;
  int n = a.lengths ? min(max(a.lengths[b], 0), p.Skv) : p.Skv;
  n = __builtin_amdgcn_readfirstlane(n);
  const int64_t start = a.starts ? a.starts[b] : a.start;
  float* out = a.nparts > 1 ? a.part + ((int64_t)part * nbh + bh) * p.Skv : a.sums + (int64_t)bh * p.Skv;
  const bool add = a.nparts == 1 && a.add;
  const unsigned lds0 = lds_addr_of(smem);
  float c2 = p.scale_log2;
  bool flip = false;
  if constexpr (!CAP) {  // masked scores are -inf: a negative scale moves into K, and 0 becomes a tiny one
    flip = c2 < 0.f;
    c2 = c2 == 0.f ? 1e-30f : fabsf(c2);
  }
  if constexpr (CAP) c2 = p.cap_log2;
  // A weight from a score: raw, or with a soft-cap its tanh.
  auto weight = [&](float s, float l2) { return fast_exp2(__builtin_fmaf(s, c2, -l2)); };

  for (int seg = 0; seg <= a.pair; ++seg) {
    const int kb = seg == 0 ? x0 : nkb - 1 - x0;
    if (seg == 1 && kb == x0) break;
    const int j0 = kb * C::KEYS;
    if (j0 >= n) {  // no key in use
      if (a.nparts == 1 && !a.add)
        for (int j = j0 + tid; j < min(j0 + C::KEYS, p.Skv); j += kWsWaves * 64) out[j] = 0.f;
      continue;
    }

    // The query rows [i_lo, i_hi) that see a key of the workgroup, as tiles of packed
    // rows; this part's tiles.
    const int R = p.G * p.Sq;
    const int64_t jl = min(j0 + C::KEYS, n) - 1;
    int64_t i_lo = 0, i_hi = p.Sq;
    if (p.causal) i_lo = j0 - start;
    if (p.window > 0) i_hi = min(i_hi, jl + p.window - start + 1);
    i_lo = min(max(i_lo, (int64_t)0), (int64_t)p.Sq);
    i_hi = max(i_hi, i_lo);
    const int t_lo = (int)(i_lo * p.G / 32), t_hi = (int)((i_hi * p.G + 31) / 32);
    // this part's tiles: every nparts-th, so that all have their share of masked ones
    const int t0 = __builtin_amdgcn_readfirstlane(t_lo + part), dt = a.nparts;
    const int nt = __builtin_amdgcn_readfirstlane(t0 < t_hi ? (t_hi - t0 + dt - 1) / dt : 0);

    // The row of the next tile that this lane copies 16 bytes of per step, and the one
    // whose LSE it copies; a step of 32 nparts rows is dq query rows and dg heads.
    const T* qp = (const T*)a.q.data + b * a.q.sb + (int64_t)hk * p.G * a.q.sh;
    const float* lp = a.lse + ((int64_t)b * p.Hq + (int64_t)hk * p.G) * p.Sq;
    const int dq = 32 * dt / p.G, dg = 32 * dt % p.G;
    const int64_t qstep = ((int64_t)dq * a.q.ss + (int64_t)dg * a.q.sh) * (int)sizeof(T);
    const int64_t qwrap = (a.q.ss - (int64_t)p.G * a.q.sh) * (int)sizeof(T);
    const int64_t lstep = ((int64_t)dq + (int64_t)dg * p.Sq) * 4, lwrap = (1 - (int64_t)p.G * p.Sq) * 4;
    const int crow = (wave & 1) * 16 + (lane >> 2);
    const int cbyte = (wave >> 1) * 64 + ((lane & 3) ^ ((crow >> 2) & 3)) * 16;
    const int cr0 = 32 * t0 + crow, lr0 = 32 * t0 + l32;
    int cg = cr0 % p.G, lg = lr0 % p.G;
    const char* ca = (const char*)(qp + (int64_t)cg * a.q.sh + (int64_t)(cr0 / p.G) * a.q.ss) + cbyte;
    const char* la = (const char*)(lp + (int64_t)lg * p.Sq + lr0 / p.G);
    auto issue = [&](int u) {  // the part's tile u, the one after the last issued
      const int t = t0 + u * dt;
      const unsigned dst = lds0 + u % C::RING * C::STAGEB;
      if (32 * t + 31 >= R) {  // rows past the last repeat it
        asm volatile("");      // (a branch, not a selection in every tile)
        if (crow >= R - 32 * t)
          ca = (const char*)(qp + (int64_t)(p.G - 1) * a.q.sh + (int64_t)(p.Sq - 1) * a.q.ss) + cbyte;
        if (l32 >= R - 32 * t) la = (const char*)(lp + (int64_t)p.G * p.Sq - 1);
      }
      if (KC % kWsWaves == 0 || wave < KC) {
        copy_steps<KC, 0>(ca, dst + wave * 1024);
        load_lds4(la, dst + C::TB);
      }
      ca += qstep;
      la += lstep;
      if (dg) {  // G does not divide 32: the heads of the rows change
        asm volatile("");
        cg += dg;
        lg += dg;
        if (cg >= p.G) cg -= p.G, ca += qwrap;
        if (lg >= p.G) lg -= p.G, la += lwrap;
      }
    };
    // copies of one tile that a wave has issued
    constexpr int kCopies = (KC + kWsWaves - 1) / kWsWaves + 1;

    f32x16 acc[NK];
#pragma unroll
    for (int kb2 = 0; kb2 < NK; ++kb2) acc[kb2] = f32x16{};
    i32x4 kf[NK][KC];
    if (nt > 0) {
#pragma unroll
      for (int x = 0; x < NK; ++x) {
        const int64_t j = min(j0 + (wave * NK + x) * 32 + l32, n - 1);
        const char* src = (const char*)((const T*)a.k.data + b * a.k.sb + hk * a.k.sh + j * a.k.ss) + 16 * h;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) kf[x][kc] = ld_global16(src + 32 * kc);
      }
      if (seg == 1) __builtin_amdgcn_s_barrier();  // every wave has read the first block's last tiles
#pragma unroll
      for (int u = 0; u < C::RING; ++u)
        if (u < nt) issue(u);
      // wait for K here, once, with the first tiles: at its first use the compiler's
      // own wait would drain the copies of later tiles
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) pin(kf[x][kc]);
    }

    // steps 2 i and 2 i + 1 of row l32 in block i
    const int koff[2] = {l32 * 64 + (h ^ ((l32 >> 2) & 3)) * 16, l32 * 64 + ((2 + h) ^ ((l32 >> 2) & 3)) * 16};
    if constexpr (!CAP) {
      if (flip) {
        constexpr int kSign = sizeof(T) == 4 ? (int)0x80000000 : (int)0x80008000;
#pragma unroll
        for (int x = 0; x < NK; ++x)
#pragma unroll
          for (int kc = 0; kc < KC; ++kc) kf[x][kc] ^= i32x4{kSign, kSign, kSign, kSign};
      }
    }
    // The tiles that need a mask, of each block of 32 keys.
    int part_lo[NK], part_hi[NK];
#pragma unroll
    for (int x = 0; x < NK; ++x) {
      const int64_t f = j0 + (wave * NK + x) * 32, l = min(f + 31, (int64_t)n - 1);
      const int64_t lo = p.causal ? max(l - start, (int64_t)0) : 0;
      const int64_t hi = p.window > 0 ? max(f + p.window - start + 1, (int64_t)0) : p.Sq;
      part_lo[x] = __builtin_amdgcn_readfirstlane((int)((min(lo, (int64_t)p.Sq) * p.G + 31) / 32));
      part_hi[x] = __builtin_amdgcn_readfirstlane((int)(min(hi, (int64_t)p.Sq) * p.G / 32));
    }
    // The last block's scores of a tile wait for the first MFMAs of the next one, and
    // the others' for those of the block after them, so that the exponentials run
    // beside MFMAs.  (None waits: scores of 0 of a row with LSE +inf, weights of 0.)
    f32x16 sw = f32x16{};
    float lw = kPosInf;
    // A tile's rows are read from LDS while the MFMAs of the tile before last use its
    // own: as each step is done, its registers are filled again.
    i32x4 qf[KC];
    float lse = 0.f;
    if (nt > 0) {
      if (nt >= C::RING) wait_vmcnt<2 * C::TPS * kCopies>();
      else wait_vmcnt<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) qf[kc] = lds_read16(smem + koff[kc & 1] + (kc >> 1) * 2048);
      lse = *(const float*)(smem + C::TB + l32 * 4);
    }
    for (int u = 0; u < nt; ++u) {
      const int t = t0 + u * dt;
      const char* sN = smem + (u + 1) % C::RING * C::STAGEB;  // the next tile
      // a row without keys gives no weight, whatever its scores
      const bool dead = 32 * t + l32 >= R || lse == kNegInf;
      const bool any_dead = __builtin_amdgcn_ballot_w64(dead);
      const float l2 = dead ? kPosInf : lse * kLog2e;
#pragma unroll
      for (int x = 0; x < NK; ++x) {
        if (x == NK - 1) {
          if (u % C::TPS == C::TPS - 1 && u + 1 < nt) {
            // this wave's copies of the next step have landed (those of the one after may
            // be in flight), and its reads of this step's last tile have returned ...
            if (u + 1 + 2 * C::TPS <= nt) wait_vmcnt<C::TPS * kCopies>();
            else wait_vmcnt<0>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();  // ... and every wave's
            asm volatile("" ::: "memory");
#pragma unroll
            for (int y = 1; y <= C::TPS; ++y)  // into the stages of this step
              if (u + 2 * C::TPS + y < nt) issue(u + 2 * C::TPS + y);
          }
          lse = *(const float*)(sN + C::TB + l32 * 4);
        }
        // The MFMAs of this block, and between them the weights of the waiting one, added
        // a step after their exponential.  The order is held by sched_barrier: left to
        // itself the compiler puts all weights first and their registers to use again.
        f32x16 sc = f32x16{};
        f32x16& to = acc[x == 0 ? NK - 1 : x - 1];
        f32x16 pe;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          sc = mma_step<T>(kf[x][kc], qf[kc], sc);
          if (x == NK - 1) qf[kc] = lds_read16(sN + koff[kc & 1] + (kc >> 1) * 2048);
#pragma unroll
          for (int e = 16 * kc / KC; e < 16 * (kc + 1) / KC; ++e) pe[e] = weight(sw[e], x == 0 ? lw : l2);
#pragma unroll
          for (int e = kc > 0 ? 16 * (kc - 1) / KC : 16; e < 16 * kc / KC; ++e) to[e] += pe[e];
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 16 * (KC - 1) / KC; e < 16; ++e) to[e] += pe[e];
        pin(to);  // here, not behind the branch below
        if constexpr (CAP) {
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[e] = tanhf(sc[e] * p.scale * p.inv_cap);
          } else {
            soft_cap(sc, p);
          }
        }
        if (t < part_lo[x] || t >= part_hi[x] || any_dead) {
          asm volatile("");  // a branch: the compiler would compute the mask of every tile
          // keys [lo, hi) of the row, relative to the lane half's first of this block
          const int64_t pos = start + (32 * t + l32) / p.G, base = j0 + (wave * NK + x) * 32 + 4 * h;
          const int64_t hi = dead ? -1 : p.causal ? pos + 1 - base : (int64_t)1 << 30;
          const int64_t lo = p.window > 0 ? pos - p.window - base : -1;
          const int hi32 = (int)min(max(hi, (int64_t)-1), (int64_t)1 << 30);
          const int lo32 = (int)min(max(lo, (int64_t)-1), (int64_t)1 << 30);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int jj = 8 * (e >> 2) + (e & 3);
            if (jj >= hi32 || jj < lo32) sc[e] = kNegInf;
          }
        }
        sw = sc;
      }
      lw = l2;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[NK - 1][e] += weight(sw[e], lw);

#pragma unroll
    for (int x = 0; x < NK; ++x) {
      const float w = column_sums(acc[x], l32);
      const int e = l32 & 15;
      const int j = j0 + (wave * NK + x) * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
      if (l32 < 16 && j < p.Skv) {
        if (add) {
          if (j < n) out[j] += w;
        } else {
          out[j] = j < n ? w : 0.f;
        }
      }
    }
  }
}

// The parts' sums added in order.
template <int D>
__global__ __launch_bounds__(256) void weight_parts_kernel(WeightArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.p.B * a.p.Hkv * a.p.Skv;
  if (i >= rows) return;
  const int j = (int)(i % a.p.Skv), b = (int)(i / a.p.Skv / a.p.Hkv);
  const int n = a.lengths ? min(max(a.lengths[b], 0), a.p.Skv) : a.p.Skv;
  float w = 0.f;
  if (j < n)
    for (int x = 0; x < a.nparts; ++x) w += a.part[x * rows + i];
  if (!a.add) a.sums[i] = w;
  else if (j < n) a.sums[i] += w;
}

template <class T, int D>
hipError_t launch_weights(const WeightArgs& a, hipStream_t st) {
  using C = WsCfg<T, D>;
  const int64_t nkb = (a.p.Skv + C::KEYS - 1) / C::KEYS;
  const dim3 grid((unsigned)((a.pair ? (nkb + 1) / 2 : nkb) * a.nparts * a.p.B * a.p.Hkv)), block(kWsWaves * 64);
  if (a.p.cap > 0.f) hipLaunchKernelGGL((weight_sums_kernel<T, D, C::NK, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((weight_sums_kernel<T, D, C::NK, false>), grid, block, 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nparts == 1) return e;
  const int64_t rows = (int64_t)a.p.B * a.p.Hkv * a.p.Skv;
  hipLaunchKernelGGL((weight_parts_kernel<D>), dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, st, a);
  return hipGetLastError();
}

#define FLEXATT_CAT2(a, b) a##b
#define FLEXATT_CAT(a, b) FLEXATT_CAT2(a, b)
hipError_t FLEXATT_CAT(weight_sums_bf16_d, FLEXATT_D)(const WeightArgs& a, hipStream_t st) {
  return launch_weights<__bf16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(weight_sums_f16_d, FLEXATT_D)(const WeightArgs& a, hipStream_t st) {
  return launch_weights<_Float16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(weight_sums_f32_d, FLEXATT_D)(const WeightArgs& a, hipStream_t st) {
  return launch_weights<float, FLEXATT_D>(a, st);
}

}  // namespace flexatt
