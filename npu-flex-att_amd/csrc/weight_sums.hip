// The attention weight each key of a K/V cache has received: for key j of KV head
// hk the sum over the G query heads that share it and over the query rows i of
// P_ij = exp(x_ij - LSE_i), with the scores, masks and LSE of the forward
// (npu_flash_attention.py:17-166).  No counterpart in the reference.
//
// The column sums of P need LSE, so they follow the forward as a product of their
// own.  Key-stationary: a wave holds 32 keys as A operands in registers and walks
// the query rows of its KV head (heads innermost, tiles of 32, the columns of an
// MFMA tile); a lane adds the weights of its column's rows for 16 keys, and the 32
// columns are added once at the end, in a fixed order.
#include "flexatt_device.h"
#include "flexatt_kernels.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
constexpr int kWsWaves = 4;

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

template <class T, int D, bool CAP>
__global__ __launch_bounds__(kWsWaves * 64) void weight_sums_kernel(WeightArgs a) {
  constexpr int KC = D * (int)sizeof(T) / 32;  // 32-byte steps of S = K Q^T
  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;

  const int nkt = (p.Skv + 32 * kWsWaves - 1) / (32 * kWsWaves);
  const int bh = blockIdx.x / nkt, hk = bh % p.Hkv, b = bh / p.Hkv;
  const int j0 = (blockIdx.x % nkt * kWsWaves + wave) * 32;  // this wave's keys
  if (j0 >= p.Skv) return;
  int n = a.lengths ? min(max(a.lengths[b], 0), p.Skv) : p.Skv;
  n = __builtin_amdgcn_readfirstlane(n);
  const int64_t start = a.starts ? a.starts[b] : a.start;
  float* out = a.sums + (int64_t)bh * p.Skv + j0;

  f32x16 acc = f32x16{};
  if (j0 < n) {
    i32x4 kf[KC];
    {
      const int j = min(j0 + l32, n - 1);
      const char* src = (const char*)((const T*)a.k.data + b * a.k.sb + hk * a.k.sh + j * a.k.ss) + 16 * h;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) kf[kc] = ld_global16(src + 32 * kc);
    }
    // query rows i whose position start + i any key of the wave is seen from
    const int64_t j1 = min(j0 + 31, n - 1);
    int64_t i_lo = p.causal ? j0 - start : 0, i_hi = p.Sq;
    if (p.window > 0) i_hi = min(i_hi, j1 + p.window - start + 1);
    if (i_lo < 0) i_lo = 0;
    const int R = p.G * p.Sq;
    const int t_lo = (int)(min(i_lo, (int64_t)p.Sq) * p.G / 32);
    const int t_hi = i_hi <= 0 ? 0 : (int)((i_hi * p.G + 31) / 32);
    for (int t = t_lo; t < t_hi; ++t) {
      const int rr = 32 * t + l32, r = min(rr, R - 1);
      const int qi = r / p.G, hq = hk * p.G + r % p.G;
      const char* src = (const char*)((const T*)a.q.data + b * a.q.sb + hq * a.q.sh + (int64_t)qi * a.q.ss) + 16 * h;
      f32x16 sc = f32x16{};
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) sc = mma_step<T>(kf[kc], ld_global16(src + 32 * kc), sc);
      const float lse = a.lse[((int64_t)b * p.Hq + hq) * p.Sq + qi];
      const bool live = rr < R && lse != kNegInf;  // a row without keys gives no weight
      const float l2 = lse * kLog2e;
      const int64_t pos = start + qi;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = j0 + 8 * (e >> 2) + 4 * h + (e & 3);
        float y;
        if constexpr (!CAP) y = __builtin_fmaf(sc[e], p.scale_log2, -l2);
        else if constexpr (sizeof(T) == 4) y = p.cap_log2 * tanhf(sc[e] * p.scale * p.inv_cap) - l2;
        else {
          float tv;
          y = score_log2<true, false>(sc[e], p, 0.f, 0, 0, tv) - l2;
        }
        bool ok = live;
        if (p.causal) ok = ok && j <= pos;
        if (p.window > 0) ok = ok && pos - j <= p.window;
        acc[e] += ok ? fast_exp2(y) : 0.f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int x = 16; x; x >>= 1) acc[e] += __shfl_xor(acc[e], x);
    const int jj = 8 * (e >> 2) + 4 * h + (e & 3);
    if (l32 == e && j0 + jj < p.Skv) {
      const float w = j0 + jj < n ? acc[e] : 0.f;
      if (!a.add) out[jj] = w;
      else if (j0 + jj < n) out[jj] += w;
    }
  }
}

template <class T, int D>
hipError_t launch_weights(const WeightArgs& a, hipStream_t st) {
  const int nkt = (a.p.Skv + 32 * kWsWaves - 1) / (32 * kWsWaves);
  const dim3 grid((unsigned)((int64_t)nkt * a.p.B * a.p.Hkv)), block(kWsWaves * 64);
  if (a.p.cap > 0.f) hipLaunchKernelGGL((weight_sums_kernel<T, D, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((weight_sums_kernel<T, D, false>), grid, block, 0, st, a);
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
