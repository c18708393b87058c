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
//    an MFMA tile, through a ring of three LDS stages that the four waves share
//    (direct-to-LDS copies, one barrier per tile; a stage is refilled two tiles
//    after its last reader passed the barrier);
//  * a lane adds the weights of its column's rows for 16 keys of each block in fp32;
//    the 32 columns are added at the end by exchanging halves, so that lane c ends
//    up with one key's sum, in a fixed order;
//  * the tiles of a key block are shared by nparts workgroups where key blocks alone
//    would leave CUs idle (a causal prefill, whose first keys are seen by every row
//    and whose last by few, also balances by them: longest first); their sums go to
//    the workspace and a second kernel adds them in order.
// What bounds it: per 32 x 32 pairs and SIMD, one fma, one exponential (a quarter
// rate instruction) and one add an element are 384 cycles of VALU, the MFMAs 2 D
// cycles beside them.
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
  static constexpr int CPR = ROWB / 16;            // 16-byte chunks per row
  static constexpr int TB = 32 * ROWB;             // bytes of a query tile
  static constexpr int NK = ROWB <= 512 ? 2 : 1;   // 32-key blocks per wave (registers)
  static constexpr int KEYS = kWsWaves * NK * 32;  // keys per workgroup
  static constexpr int E = TB / 1024;              // 1 KB copies per tile
  static constexpr int EW = (E + kWsWaves - 1) / kWsWaves;  // and per wave
  static constexpr int STAGEB = TB + 256;          // a tile and its 32 rows' LSE (a 64-lane copy)
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

// Adds the 32 columns of 16 values per lane half: lane c of each half ends up with
// the sum of element c % 16 (lanes c and c ^ 16 both have it).
__device__ __forceinline__ float column_sums(const f32x16& a, int l32) {
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = a[e];
#pragma unroll
  for (int w = 8; w; w >>= 1) {
    const bool up = l32 & w;
#pragma unroll
    for (int e = 0; e < w; ++e) {  // keep the half whose bit w of the element is this lane's
      const float send = up ? x[e] : x[e + w], keep = up ? x[e + w] : x[e];
      x[e] = keep + __shfl_xor(send, w);
    }
  }
  return x[0] + __shfl_xor(x[0], 16);
}
}  // namespace

template <class T, int D, int NK, bool CAP>
__global__ __launch_bounds__(kWsWaves * 64) __attribute__((amdgpu_waves_per_eu(D * sizeof(T) >= 512 ? 1 : 2)))
void weight_sums_kernel(WeightArgs a) {
  using C = WsCfg<T, D>;
  constexpr int KC = C::KC;
  __shared__ __attribute__((aligned(1024))) char smem[3 * C::STAGEB];
  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;

  // (key block, part, b, hkv): those of one (b, hkv) share an XCD where their number
  // is a multiple of 8, and under a causal mask the longest walks go first
  const int nbh = p.B * p.Hkv;
  const int bh = blockIdx.x % nbh, hk = bh % p.Hkv, b = bh / p.Hkv;
  const int part = blockIdx.x / nbh % a.nparts, kb = blockIdx.x / nbh / a.nparts;
  const int j0 = kb * C::KEYS;
  int n = a.lengths ? min(max(a.lengths[b], 0), p.Skv) : p.Skv;
  n = __builtin_amdgcn_readfirstlane(n);
  const int64_t start = a.starts ? a.starts[b] : a.start;
  float* out = a.nparts > 1 ? a.part + ((int64_t)part * nbh + bh) * p.Skv : a.sums + (int64_t)bh * p.Skv;
  const bool add = a.nparts == 1 && a.add;
  if (j0 >= n) {  // no key in use
    if (a.nparts == 1 && !a.add)
      for (int j = j0 + tid; j < min(j0 + C::KEYS, p.Skv); j += kWsWaves * 64) out[j] = 0.f;
    return;
  }

  // The query rows [i_lo, i_hi) that see a key of the workgroup, and those that see
  // all keys of the workgroup, as tiles of packed rows; this part's tiles.
  const int R = p.G * p.Sq;
  const int64_t jl = min(j0 + C::KEYS, n) - 1;
  int64_t i_lo = 0, i_hi = p.Sq, f_lo = 0, f_hi = p.Sq;
  if (p.causal) i_lo = j0 - start, f_lo = jl - start;
  if (p.window > 0) i_hi = min(i_hi, jl + p.window - start + 1), f_hi = min(f_hi, j0 + p.window - start + 1);
  i_lo = min(max(i_lo, (int64_t)0), (int64_t)p.Sq);
  i_hi = max(i_hi, i_lo);
  f_lo = max(f_lo, (int64_t)0);
  const int t_lo = (int)(i_lo * p.G / 32), t_hi = (int)((i_hi * p.G + 31) / 32);
  const int64_t r_full_lo = f_lo * p.G, r_full_hi = f_hi * p.G;
  const int per = (t_hi - t_lo + a.nparts - 1) / a.nparts;
  const int t0 = __builtin_amdgcn_readfirstlane(t_lo + part * per);
  const int t1 = __builtin_amdgcn_readfirstlane(min(t_hi, t_lo + (part + 1) * per));

  // this lane's share of a tile's copies: packed rows 32 t + row of copy slot x, kept
  // as (query row, head) and moved on by 32 rows a tile
  const T* qp = (const T*)a.q.data + b * a.q.sb + (int64_t)hk * p.G * a.q.sh;
  const float* lp = a.lse + ((int64_t)b * p.Hq + (int64_t)hk * p.G) * p.Sq;
  const int dq = 32 / p.G, dg = 32 % p.G;
  int ci[C::EW], cg[C::EW], li, lg;
#pragma unroll
  for (int x = 0; x < C::EW; ++x) {
    const int r = 32 * t0 + ((x * kWsWaves + wave) * 64 + lane) / C::CPR;
    ci[x] = r / p.G;
    cg[x] = r % p.G;
  }
  li = (32 * t0 + l32) / p.G;
  lg = (32 * t0 + l32) % p.G;
  const unsigned lds0 = lds_addr_of(smem);
  auto issue = [&](int st) {  // the next tile into stage st; rows past the last repeat it
#pragma unroll
    for (int x = 0; x < C::EW; ++x) {
      const int e = x * kWsWaves + wave;
      if (C::E % kWsWaves == 0 || e < C::E) {
        const int row = (e * 64 + lane) / C::CPR, pc = (e * 64 + lane) % C::CPR;
        const bool in = ci[x] < p.Sq;
        const int i = in ? ci[x] : p.Sq - 1, g = in ? cg[x] : p.G - 1;
        load_lds16((const char*)(qp + (int64_t)g * a.q.sh + (int64_t)i * a.q.ss) + swz_col<C::CPR>(row, pc) * 16,
                   lds0 + st * C::STAGEB + e * 1024);
      }
      ci[x] += dq;
      cg[x] += dg;
      if (cg[x] >= p.G) cg[x] -= p.G, ci[x] += 1;
    }
    const bool in = li < p.Sq;
    load_lds4(lp + (int64_t)(in ? lg : p.G - 1) * p.Sq + (in ? li : p.Sq - 1), lds0 + st * C::STAGEB + C::TB);
    li += dq;
    lg += dg;
    if (lg >= p.G) lg -= p.G, li += 1;
  };
  // copies of one tile this wave has issued
  constexpr int kCopies = (C::E % kWsWaves == 0 ? C::EW : 0) + 1;

  f32x16 acc[NK];
#pragma unroll
  for (int kb2 = 0; kb2 < NK; ++kb2) acc[kb2] = f32x16{};
  i32x4 kf[NK][KC];
  if (t0 < t1) {
#pragma unroll
    for (int x = 0; x < NK; ++x) {
      const int64_t j = min(j0 + (wave * NK + x) * 32 + l32, n - 1);
      const char* src = (const char*)((const T*)a.k.data + b * a.k.sb + hk * a.k.sh + j * a.k.ss) + 16 * h;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) kf[x][kc] = ld_global16(src + 32 * kc);
    }
    issue(0);
    if (t0 + 1 < t1) issue(1);
    // wait for K here, once, with the first tiles: at its first use the compiler's
    // own wait would drain the copies of later tiles
#pragma unroll
    for (int x = 0; x < NK; ++x)
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) pin(kf[x][kc]);
  }

  int koff[KC];
#pragma unroll
  for (int kc = 0; kc < KC; ++kc) koff[kc] = l32 * C::ROWB + swz_col<C::CPR>(l32, 2 * kc + h) * 16;
  const float c2 = p.scale_log2;

  int st = 0;
  for (int t = t0; t < t1; ++t) {
    // this wave's copies of tile t have landed (those of t + 1 may be in flight) ...
    if (t + 1 < t1 && C::E % kWsWaves == 0) wait_vmcnt<kCopies>();
    else wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();  // ... and every wave's; all are done with tile t - 1
    asm volatile("" ::: "memory");
    if (t + 2 < t1) issue(st >= 1 ? st - 1 : 2);  // (t + 2) % 3 stages on: where tile t - 1 was
    const char* sQ = smem + st * C::STAGEB;
    const float lse = *(const float*)(sQ + C::TB + l32 * 4);

    f32x16 sc[NK];
#pragma unroll
    for (int x = 0; x < NK; ++x) sc[x] = f32x16{};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const i32x4 q = lds_read16(sQ + koff[kc]);
#pragma unroll
      for (int x = 0; x < NK; ++x) sc[x] = mma_step<T>(kf[x][kc], q, sc[x]);
    }
    const int r = 32 * t + l32;
    const bool live = r < R && lse != kNegInf;  // a row without keys gives no weight
    const float l2 = lse * kLog2e;
    const bool full = 32 * t >= r_full_lo && 32 * (int64_t)t + 31 < r_full_hi &&
                      __builtin_amdgcn_ballot_w64(!live) == 0;
    auto weight = [&](float s) {
      float y;
      if constexpr (!CAP) y = __builtin_fmaf(s, c2, -l2);
      else if constexpr (sizeof(T) == 4) y = p.cap_log2 * tanhf(s * p.scale * p.inv_cap) - l2;
      else {
        float tv;
        y = score_log2<true, false>(s, p, 0.f, 0, 0, tv) - l2;
      }
      return fast_exp2(y);
    };
    if (full) {
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[x][e] += weight(sc[x][e]);
    } else {
      const int64_t pos = start + r / p.G;
      // keys [lo, hi) of the row, relative to the lane half's first
      const int64_t base = j0 + 4 * h;
      int64_t hi = p.causal ? pos + 1 - base : (int64_t)1 << 30, lo = p.window > 0 ? pos - p.window - base : -1;
      if (!live) hi = -1;
      const int hi32 = (int)min(max(hi, (int64_t)-1), (int64_t)1 << 30), lo32 = (int)min(max(lo, (int64_t)-1), (int64_t)1 << 30);
#pragma unroll
      for (int x = 0; x < NK; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int jj = (wave * NK + x) * 32 + 8 * (e >> 2) + (e & 3);
          acc[x][e] += (jj < hi32 && jj >= lo32) ? weight(sc[x][e]) : 0.f;
        }
    }
    st = st == 2 ? 0 : st + 1;
  }

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
  const dim3 grid((unsigned)(nkb * a.nparts * a.p.B * a.p.Hkv)), block(kWsWaves * 64);
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
