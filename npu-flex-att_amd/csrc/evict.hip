// Eviction from a K/V cache: of the n cached rows of a (sequence, KV head), the
// first `sinks`, the last `recent` and, of the others, those with the largest
// accumulated attention weight stay, `keep` in all, in slot order.  No counterpart
// in the reference, which has no cache.
//
//  * evict_select_kernel: one workgroup per (sequence, head).  A score becomes an
//    unsigned key of the same order (NaN above everything, -0 as 0), and the
//    smallest kept key is found digit by digit, 8 bits a pass: a histogram of the
//    keys that match the digits so far, and the digit at which the count from
//    above reaches the number wanted.  Keys above it stay; of those equal to it
//    the lowest slots.  A scan over the slots then gives each kept row its place.
//    Counts are integers, so the order of the atomics does not matter.
//  * evict_gather_kernel: copies the rows, 16 bytes per lane; bound by memory
//    (each kept row read and written once).
#include "flexatt_device.h"
#include "flexatt_kernels.h"

namespace flexatt {

namespace {
constexpr int kSel = 1024;  // threads of a selection
constexpr int kSelWaves = kSel / 64;

// Larger float <-> larger unsigned; NaN is the largest, and -0 equals 0.
__device__ __forceinline__ unsigned order_key(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __float_as_uint(x + 0.0f);  // -0 + 0 = 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive sum over the workgroup; `total` gets the whole sum.
__device__ __forceinline__ int scan_sum(int v, int* tot, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the previous use of tot is over
  if (lane == 63) tot[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    if (w < wave) before += tot[w];
    all += tot[w];
  }
  total = all;
  return before + x - v;
}

__global__ __launch_bounds__(kSel) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int tot[kSelWaves];
  __shared__ unsigned s_digit;
  __shared__ int s_above;
  const int tid = threadIdx.x;
  const int bh = blockIdx.x, b = bh / a.H;
  const int n = min(max(a.lengths[b], 0), a.C);
  const float* sc = a.scores + (int64_t)bh * a.C;
  float* so = a.scores_out + (int64_t)bh * a.out_rows;
  int* slots = a.slots + (int64_t)bh * a.keep;
  const int kept = min(n, a.keep);
  if (bh % a.H == 0 && tid == 0) a.lengths_out[b] = kept;
  for (int i = kept + tid; i < a.out_rows; i += kSel) so[i] = 0.f;
  for (int i = kept + tid; i < a.keep; i += kSel) slots[i] = -1;
  if (n <= a.keep) {
    for (int i = tid; i < n; i += kSel) {
      slots[i] = i;
      so[i] = sc[i];
    }
    return;
  }

  // the slots that go by their score: [lo, hi), `want` of them stay
  const int lo = a.sinks, hi = n - a.recent, want = a.keep - a.sinks - a.recent;
  unsigned prefix = 0, mask = 0;
  int need = want;  // still wanted among the keys that match the digits so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kSel) {
      const unsigned k = order_key(sc[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // the digit d with (keys above d) < need <= (keys at or above d)
    if (tid < 64) {
      int c[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = hist[255 - (4 * tid + e)];
        sum += c[e];
      }
      int x = sum;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (tid >= d) x += y;
      }
      int above = x - sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (above < need && above + c[e] >= need) {
          s_digit = 255 - (4 * tid + e);
          s_above = above;
        }
        above += c[e];
      }
      if (need <= 0 && tid == 0) {  // nothing goes by score: a threshold no key passes
        s_digit = 255;
        s_above = 0;
      }
    }
    __syncthreads();
    prefix |= s_digit << shift;
    mask |= 255u << shift;
    need -= s_above;
    __syncthreads();
  }

  // prefix: the smallest kept key; `need` of its equals stay, the lowest slots
  int ties = 0, place = 0;  // before this chunk
  for (int i0 = 0; i0 < n; i0 += kSel) {
    const int i = i0 + tid;
    const bool in = i < n, free = in && i >= lo && i < hi;
    const float x = in ? sc[i] : 0.f;
    const unsigned k = order_key(x);
    const int eq = free && k == prefix;
    int all;
    const int tie = ties + scan_sum(eq, tot, all);
    ties += all;
    const int stay = in && (!free || (want > 0 && (k > prefix || (eq && tie < need))));
    const int at = place + scan_sum(stay, tot, all);
    place += all;
    if (stay) {
      slots[at] = i;
      so[at] = x;
    }
  }
}

// Rows to their places: `nblk` workgroups for each (sequence, head), CPR lanes copy
// a row, four rows in flight.
template <int CPR>
__global__ __launch_bounds__(256) void evict_gather_kernel(EvictArgs a, int nblk) {
  constexpr int RPB = 256 / CPR, U = 4;
  const int c = threadIdx.x % CPR, r = threadIdx.x / CPR;
  const int bh = blockIdx.x / nblk, b = bh / a.H, h = bh % a.H;
  const int* slots = a.slots + (int64_t)bh * a.keep;
  const int es = a.es;
  const char* ks = (const char*)a.k.data + (b * a.k.sb + h * a.k.sh) * es + c * 16;
  const char* vs = (const char*)a.v.data + (b * a.v.sb + h * a.v.sh) * es + c * 16;
  char* kd = (char*)a.ko.data + (b * a.ko.sb + h * a.ko.sh) * es + c * 16;
  char* vd = (char*)a.vo.data + (b * a.vo.sb + h * a.vo.sh) * es + c * 16;
  const int i0 = blockIdx.x % nblk * RPB * U + r;
  int s[U];
  i32x4 x[U], y[U];
#pragma unroll
  for (int u = 0; u < U; ++u) s[u] = i0 + u * RPB < a.keep ? slots[i0 + u * RPB] : -2;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    x[u] = y[u] = i32x4{0, 0, 0, 0};
    if (s[u] >= 0) {
      x[u] = ld_global16(ks + s[u] * a.k.ss * es);
      y[u] = ld_global16(vs + s[u] * a.v.ss * es);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (s[u] >= 0 || (s[u] == -1 && a.fill)) {
      const int64_t i = i0 + u * RPB;
      *(i32x4*)(kd + i * a.ko.ss * es) = x[u];
      *(i32x4*)(vd + i * a.vo.ss * es) = y[u];
    }
  }
}

template <int CPR>
void gather(const EvictArgs& a, hipStream_t st) {
  const int rows = 256 / CPR * 4, nblk = (a.keep - 1) / rows + 1;
  hipLaunchKernelGGL((evict_gather_kernel<CPR>), dim3((unsigned)nblk * a.B * a.H), dim3(256), 0, st, a, nblk);
}
}  // namespace

hipError_t evict_run(const EvictArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(evict_select_kernel, dim3(a.B * a.H), dim3(kSel), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  switch (a.D * a.es / 16) {
    case 4: gather<4>(a, st); break;
    case 8: gather<8>(a, st); break;
    case 16: gather<16>(a, st); break;
    case 32: gather<32>(a, st); break;
    case 64: gather<64>(a, st); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace flexatt
