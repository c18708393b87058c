// A K/V cache of 8 bits read back in a wider type: code * scale, the product in 32 bits,
// rounded once.  For what takes a cache of the working type: the forward over a chunk of
// a prompt, weight sums, eviction.  No counterpart in the reference, which has no cache.
//
// Bound by memory.  A thread has the codes of 16 output bytes, so that a wave's stores
// are whole lines, of four rows of K and of V, all loaded before the first is stored.
#include "flexatt_device.h"
#include "flexatt_kernels.h"

namespace flexatt {

namespace {
constexpr int kThreads = 256;

// The values of N codes in the first bytes of w (4 or 8).
template <int N>
__device__ __forceinline__ void values_of(int kind, i32x2 w, float (&x)[N]) {
#pragma unroll
  for (int g = 0; g < N / 4; ++g) {
    if (kind == FLEXATT_E4M3) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[g], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[g], true);
      x[4 * g] = lo[0], x[4 * g + 1] = lo[1], x[4 * g + 2] = hi[0], x[4 * g + 3] = hi[1];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * g + e] = (float)(signed char)(w[g] >> (8 * e));
    }
  }
}

// Workgroup x: rows of one (b, h), R times as many as its threads hold at once.
template <class T, int D, int R>
__global__ __launch_bounds__(kThreads) void dequant_kernel(DequantArgs a, int chunks) {
  constexpr int N = 16 / (int)sizeof(T), TPR = D / N, RPB = kThreads / TPR;
  typedef T vec __attribute__((ext_vector_type(N)));
  const int bh = blockIdx.x / chunks, chunk = blockIdx.x - bh * chunks;
  const int b = bh / a.H, h = bh - b * a.H;
  const int n = min(max(a.lengths[b], 0), a.C);
  const int r0 = chunk * (R * RPB) + threadIdx.x / TPR, d = threadIdx.x % TPR * N;
  if (!a.fill && chunk * (R * RPB) >= n) return;
  const char* k = (const char*)a.k.data + b * a.k.sb + h * a.k.sh + d;
  const char* v = (const char*)a.v.data + b * a.v.sb + h * a.v.sh + d;
  const int64_t s0 = (int64_t)bh * a.C;
  i32x2 ck[R], cv[R];
  float sk[R], sv[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i * RPB;
    if (r >= n) continue;
    if constexpr (N == 8) {
      ck[i] = *(const i32x2*)(k + (int64_t)r * a.k.ss);
      cv[i] = *(const i32x2*)(v + (int64_t)r * a.v.ss);
    } else {
      ck[i] = i32x2{*(const int*)(k + (int64_t)r * a.k.ss), 0};
      cv[i] = i32x2{*(const int*)(v + (int64_t)r * a.v.ss), 0};
    }
    sk[i] = a.k_scales[s0 + r];
    sv[i] = a.v_scales[s0 + r];
  }
  T* ko = (T*)a.ko.data + b * a.ko.sb + h * a.ko.sh + d;
  T* vo = (T*)a.vo.data + b * a.vo.sb + h * a.vo.sh + d;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i * RPB;
    if (r >= (a.fill ? a.C : n)) continue;
    vec x = {}, y = {};
    if (r < n) {
      float p[N], q[N];
      values_of<N>(a.kind, ck[i], p);
      values_of<N>(a.kind, cv[i], q);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = from_f32<T>(p[e] * sk[i]), y[e] = from_f32<T>(q[e] * sv[i]);
    }
    *(vec*)(ko + (int64_t)r * a.ko.ss) = x;
    *(vec*)(vo + (int64_t)r * a.vo.ss) = y;
  }
}

template <class T, int D>
hipError_t launch_d(const DequantArgs& a, hipStream_t st) {
  constexpr int RPB = kThreads / (D / (16 / (int)sizeof(T)));
  const int64_t bh = (int64_t)a.B * a.H;
  const int rows = dequant_rows(D * (int)sizeof(T), bh, a.C), chunks = (a.C + rows - 1) / rows;
  const dim3 grid((unsigned)(bh * chunks));
  if (rows == RPB) hipLaunchKernelGGL((dequant_kernel<T, D, 1>), grid, dim3(kThreads), 0, st, a, chunks);
  else hipLaunchKernelGGL((dequant_kernel<T, D, 4>), grid, dim3(kThreads), 0, st, a, chunks);
  return hipGetLastError();
}

template <class T>
hipError_t launch(const DequantArgs& a, hipStream_t st) {
  switch (a.D) {
    case 32: return launch_d<T, 32>(a, st);
    case 64: return launch_d<T, 64>(a, st);
    case 128: return launch_d<T, 128>(a, st);
    case 256: return launch_d<T, 256>(a, st);
    default: return hipErrorInvalidValue;
  }
}
}  // namespace

hipError_t dequant_run(int dtype, const DequantArgs& a, hipStream_t st) {
  switch (dtype) {
    case FLEXATT_F32: return launch<float>(a, st);
    case FLEXATT_F16: return launch<_Float16>(a, st);
    case FLEXATT_BF16: return launch<__bf16>(a, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace flexatt
