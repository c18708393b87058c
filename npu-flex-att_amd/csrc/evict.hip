// Eviction from a K/V cache: of the n cached rows of a (sequence, KV head), the
// first `sinks`, the last `recent` and, of the others, those with the largest
// accumulated attention weight stay, `keep` in all, in slot order.  No counterpart
// in the reference, which has no cache.
//
//  * evict_select_kernel: one workgroup per (sequence, head).  A score becomes an
//    unsigned key of the same order (NaN above everything, -0 as 0).  The keys are
//    narrowed to those that share their leading bits with the last kept one, a digit a
//    pass from the highest bit in which any two differ: a histogram, and the digit at
//    which the count from above reaches the number wanted.  Once at most 64 are left,
//    each lane of a wave counts the larger ones of one (of equal ones the lower slot is
//    the larger), and the one with the right rank is the last kept; where more than
//    that have the same key, their slots are counted in order instead.  A scan over the slots then gives each kept row its place.  Counts are
//    integers and ranks follow from keys and slots, so the order of the atomics does
//    not matter.  Latency: a chain of passes over keys that stay in registers up to
//    eight slots a thread; 256 threads up to 2048 slots, for cheaper barriers.
//  * evict_gather_kernel: copies the rows, 16 bytes per lane; bound by memory
//    (each kept row read and written once).
#include "flexatt_device.h"
#include "flexatt_kernels.h"

namespace flexatt {

namespace {
constexpr int kPer = 8;  // consecutive slots per thread and block

// Larger float <-> larger unsigned; NaN is the largest, and -0 equals 0.
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);  // -0 + 0 = 0
  const unsigned k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return x != x ? 0xffffffffu : k;
}

// Exclusive sum over a workgroup of NT threads; `total` gets the whole sum.  Every
// thread calls it.
template <int NT>
__device__ __forceinline__ int scan_sum(int v, int* tot, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();  // the previous use of tot is over
  if (lane == 63) tot[wave] = x;
  __syncthreads();
  const int mine = lane < NT / 64 ? tot[lane] : 0;
  const int upto = wave_scan(mine);
  total = __builtin_amdgcn_readlane(upto, 63);
  return __builtin_amdgcn_readlane(upto - mine, __builtin_amdgcn_readfirstlane(wave)) + x - v;
}

template <int NT>
__global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs a) {
  constexpr int kBins = 2 * NT, kDigit = NT == 1024 ? 11 : 9;
  static_assert(kBins == 1 << kDigit, "two bins per thread");
  __shared__ int hist[kBins];
  __shared__ int tot[NT / 64];
  __shared__ unsigned lows[NT / 64], highs[NT / 64];
  __shared__ unsigned ckey[64];
  __shared__ int cslot[64];
  __shared__ int s_digit, s_above, s_count, s_slot;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bh = blockIdx.x, b = bh / a.H;
  const int n = min(max(a.lengths[b], 0), a.C);
  const float* sc = a.scores + (int64_t)bh * a.C;
  float* so = a.scores_out + (int64_t)bh * a.out_rows;
  int* slots = a.slots + (int64_t)bh * a.keep;
  const int kept = min(n, a.keep);
  if (bh - b * a.H == 0 && tid == 0) a.lengths_out[b] = kept;
  for (int i = kept + tid; i < a.out_rows; i += NT) so[i] = 0.f;
  for (int i = kept + tid; i < a.keep; i += NT) slots[i] = -1;
  if (n <= a.keep) {
    for (int i = tid; i < n; i += NT) {
      slots[i] = i;
      so[i] = sc[i];
    }
    return;
  }

  // the slots that go by their score: [lo, hi), `need` of them stay
  const int lo = a.sinks, hi = n - a.recent;
  int need = a.keep - a.sinks - a.recent;
  constexpr int kBlock = NT * kPer;
  const int nb = (n - 1) / kBlock + 1;
  float x[kPer];  // this thread's slots of block `blk`: kBlock blk + kPer tid + e
  auto load = [&](int blk) {
    const int i0 = blk * kBlock + tid * kPer;
    if (i0 + kPer <= n) {
      struct __attribute__((packed, aligned(4))) Quad {
        float v[4];
      };
      const Quad* q = (const Quad*)(sc + i0);
      const Quad q0 = q[0], q1 = q[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = q0.v[e], x[4 + e] = q1.v[e];
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = sc[min(i0 + e, n - 1)];
    }
  };
  auto each = [&](auto f) {  // f(slot, key) for the slots that go by their score
    for (int blk = 0; blk < nb; ++blk) {
      if (nb > 1) load(blk);  // (a single block stays in registers)
      const int i0 = blk * kBlock + tid * kPer;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (i0 + e >= lo && i0 + e < hi) f(i0 + e, order_key(x[e]));
    }
  };
  if (nb == 1) load(0);

  // A slot stays by its score where its key is above last_key, or is last_key and the
  // slot is at most last_slot.
  unsigned last_key = 0xffffffffu;
  int last_slot = -1;
  if (need > 0) {
    hist[tid] = 0;
    hist[tid + NT] = 0;
    // the bits that all keys share
    unsigned low = 0, high = 0;  // of the complements, and of the keys, the largest
    each([&](int, unsigned k) {
      low = max(low, ~k);
      high = max(high, k);
    });
    low = wave_max(low);
    high = wave_max(high);
    if (lane == 0) lows[wave] = low, highs[wave] = high;
    __syncthreads();
    low = ~wave_max(lane < NT / 64 ? lows[lane] : 0);
    high = wave_max(lane < NT / 64 ? highs[lane] : 0);
    // keys whose bits from `top` on equal `prefix`'s are left: `count` of them
    int top = low == high ? 0 : 32 - __builtin_clz(low ^ high);
    unsigned prefix = top >= 32 ? 0 : high >> top << top;
    int count = hi - lo;
    while (count > 64 && top > 0) {
      const int shift = max(top - kDigit, 0);
      const unsigned width = (1u << (top - shift)) - 1u;
      each([&](int, unsigned k) {
        if (((uint64_t)(k ^ prefix) >> top) == 0) atomicAdd(&hist[(k >> shift) & width], 1);
      });
      __syncthreads();
      // thread t has the bins 2 t and 2 t + 1 from above
      const int h0 = hist[kBins - 1 - 2 * tid], h1 = hist[kBins - 2 - 2 * tid];
      int all;
      const int above = scan_sum<NT>(h0 + h1, tot, all);
      if (above < need && above + h0 + h1 >= need) {
        const bool first = above + h0 >= need;
        s_digit = kBins - 1 - 2 * tid - (first ? 0 : 1);
        s_above = above + (first ? 0 : h0);
        s_count = first ? h0 : h1;
      }
      hist[kBins - 1 - 2 * tid] = 0;
      hist[kBins - 2 - 2 * tid] = 0;
      __syncthreads();
      prefix |= (unsigned)s_digit << shift;
      need -= s_above;
      count = s_count;
      top = shift;
    }
    if (count > 64) {  // equal keys: the slot of the need-th of them
      last_key = prefix;
      int seen = 0;
      for (int blk = 0; blk < nb; ++blk) {
        if (nb > 1) load(blk);
        const int i0 = blk * kBlock + tid * kPer;
        int eq = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) eq += i0 + e >= lo && i0 + e < hi && order_key(x[e]) == prefix;
        int all, at = seen + scan_sum<NT>(eq, tot, all);
        seen += all;
        if (at < need && at + eq >= need) {
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (i0 + e >= lo && i0 + e < hi && order_key(x[e]) == prefix && ++at == need) s_slot = i0 + e;
        }
      }
      __syncthreads();
      last_slot = s_slot;
    } else {
      // the candidates, in any order, and the one with need - 1 larger ones
      __syncthreads();
      if (tid == 0) s_count = 0;
      __syncthreads();
      each([&](int i, unsigned k) {
        if (((uint64_t)(k ^ prefix) >> top) == 0) {
          const int c = atomicAdd(&s_count, 1);
          ckey[c] = k;
          cslot[c] = i;
        }
      });
      __syncthreads();
      const unsigned k = lane < count ? ckey[lane] : 0;
      const int i = lane < count ? cslot[lane] : 0x7fffffff;
      int larger = 0;
      for (int c = 0; c < count; ++c) {
        const unsigned kc = (unsigned)__builtin_amdgcn_readlane((int)k, c);
        larger += kc > k || (kc == k && __builtin_amdgcn_readlane(i, c) < i);
      }
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < count && larger == need - 1) | 1ull << 63);
      last_key = (unsigned)__builtin_amdgcn_readlane((int)k, l);
      last_slot = __builtin_amdgcn_readlane(i, l);
    }
  }

  // places, in slot order
  int place = 0;
  for (int blk = 0; blk < nb; ++blk) {
    if (nb > 1) load(blk);
    const int i0 = blk * kBlock + tid * kPer;
    unsigned stay = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = i0 + e;
      const unsigned k = order_key(x[e]);
      const bool by_score = k > last_key || (k == last_key && i <= last_slot);
      if (i < n && (i < lo || i >= hi || by_score)) stay |= 1u << e;
    }
    int all;
    int at = place + scan_sum<NT>(__builtin_popcount(stay), tot, all);
    place += all;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (stay & (1u << e)) {
        slots[at] = i0 + e;
        so[at] = x[e];
        at += 1;
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
  if (a.C <= 256 * kPer) hipLaunchKernelGGL(evict_select_kernel<256>, dim3(a.B * a.H), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(evict_select_kernel<1024>, dim3(a.B * a.H), dim3(1024), 0, st, a);
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
