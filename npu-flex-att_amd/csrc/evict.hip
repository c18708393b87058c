// Eviction from a K/V cache: of the n cached rows of a (sequence, KV head), the
// first `sinks`, the last `recent` and, of the others, those with the largest
// accumulated attention weight stay, `keep` in all, in slot order.  No counterpart
// in the reference, which has no cache.
//
//  * Selection.  A score becomes an unsigned key of the same order (NaN above
//    everything, -0 as 0).  The keys are narrowed to those that share their leading
//    bits with the last kept one, a digit a pass from the highest bit in which any two
//    differ: a histogram, and the digit at which the count from above reaches the number
//    wanted.  Once at most 64 are left, each lane of a wave counts the larger ones of
//    one (of equal ones the lower slot is the larger), and the one with the right rank
//    is the last kept; where more than that have the same key, their slots are counted
//    in order instead.  A scan over the slots then gives each kept row its place.
//    Counts are integers and ranks follow from keys and slots, so the order of the
//    atomics does not matter.
//  * Copies, 16 bytes per lane, of the rows of a share of the places: as many
//    workgroups as fill the chip make the same selection, each for its share.  (The
//    copies as a kernel of their own behind one selection: 64 heads of 8192 slots, bf16
//    D=128, 2048 kept, 42 -> 39 us; two heads of 2048, fp32 D=64, 1000 kept, 12 -> 9.)
// What bounds it: the copies memory (134 MB there: 26 us at the rate of a large copy),
// the selection latency: a chain of passes over keys that stay in registers up to
// sixteen slots a thread (256 threads up to 2048 slots, for cheaper barriers), and of
// that a good part the code, which a launch finds out of the instruction cache (at
// about a byte a cycle; hence one copy of each loop, and the kernel that reads the
// scores again in every pass, for more slots, apart).  Times: 64 heads of 8192 slots,
// 2048 kept, 37 us; of 16384, 4096 of D=64 kept, 38; one head of 131072 97 us.
#include "flexatt_device.h"
#include "flexatt_kernels.h"

namespace flexatt {

namespace {

// Larger float <-> larger unsigned; NaN is the largest, and -0 equals 0.  Never 0.
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

// The rows of the places [i0, i1) copied, a row by 2^lg lanes, four rows in flight.
template <int NT>
__device__ __forceinline__ void gather(const EvictArgs& a, int b, int h, const int* slots, int i0, int i1) {
  constexpr int U = 4;
  const int lg = a.lanes_log2, c = threadIdx.x & ((1 << lg) - 1), r = threadIdx.x >> lg, rows = NT >> lg;
  const int es = a.es;
  const char* ks = (const char*)a.k.data + (b * a.k.sb + h * a.k.sh) * es + c * 16;
  const char* vs = (const char*)a.v.data + (b * a.v.sb + h * a.v.sh) * es + c * 16;
  char* kd = (char*)a.ko.data + (b * a.ko.sb + h * a.ko.sh) * es + c * 16;
  char* vd = (char*)a.vo.data + (b * a.vo.sb + h * a.vo.sh) * es + c * 16;
  for (; i0 < i1; i0 += U * rows) {
    int s[U];
    i32x4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * rows + r;
      s[u] = i < i1 ? slots[i] : -2;
    }
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
        const int64_t i = i0 + u * rows + r;
        *(i32x4*)(kd + i * a.ko.ss * es) = x[u];
        *(i32x4*)(vd + i * a.vo.ss * es) = y[u];
      }
    }
  }
}

// A thread has kPer consecutive slots of a block.  MANY: more than one block of NT * kPer.  Each pass reads their scores again, the
// next block's while it works on this one's, until the candidates are few enough for a
// few registers of each thread.
template <int NT, int kPer, bool MANY>
__global__ __launch_bounds__(NT) void evict_kernel(EvictArgs a) {
  constexpr int kBins = 2 * NT, kDigit = NT == 1024 ? 11 : 9;
  static_assert(kBins == 1 << kDigit, "two bins per thread");
  __shared__ int hist[kBins];
  __shared__ int tot[NT / 64];
  __shared__ unsigned lows[NT / 64], highs[NT / 64];
  constexpr int kFew = MANY ? 4 : 0, kCand = MANY ? kFew * NT : 64;
  __shared__ unsigned ckey[kCand];
  __shared__ int cslot[kCand];
  __shared__ int s_digit, s_above, s_count, s_slot;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nbh = a.B * a.H, part = blockIdx.x / nbh, bh = blockIdx.x % nbh, b = bh / a.H;
  // this workgroup's places: what it writes of scores_out, slots, k_out and v_out
  const int p0 = (int)((int64_t)a.keep * part / a.nparts), p1 = (int)((int64_t)a.keep * (part + 1) / a.nparts);
  const int n = min(max(a.lengths[b], 0), a.C);
  const float* sc = a.scores + (int64_t)bh * a.C;
  float* so = a.scores_out + (int64_t)bh * a.out_rows;
  int* slots = a.slots + (int64_t)bh * a.keep;
  if (part == 0) {
    if (bh - b * a.H == 0 && tid == 0) a.lengths_out[b] = min(n, a.keep);
    for (int i = a.keep + tid; i < a.out_rows; i += NT) so[i] = 0.f;
  }
  if (n > a.keep) {
    // the slots that go by their score: [lo, hi), `need` of them stay
    const int lo = a.sinks, hi = n - a.recent;
    int need = a.keep - a.sinks - a.recent;
    constexpr int kBlock = NT * kPer;
    const int nb = MANY ? (n - 1) / kBlock + 1 : 1;
    // This thread's slots of block `blk`, kBlock blk + kPer tid + e: their scores, the
    // keys of those that go by them (0 for the others), and as bits e those that stay
    // anyway.
    float x[kPer], ahead[kPer];
    unsigned key[kPer], sure = 0;
    auto fetch = [&](int blk) {
      const int i0 = blk * kBlock + tid * kPer;
      if (i0 + kPer <= n) {
        struct __attribute__((packed, aligned(4))) Quad {
          float v[4];
        };
        const Quad* q = (const Quad*)(sc + i0);
#pragma unroll
        for (int y = 0; y < kPer / 4; ++y) {
          const Quad v = q[y];
#pragma unroll
          for (int e = 0; e < 4; ++e) ahead[4 * y + e] = v.v[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) ahead[e] = sc[min(i0 + e, n - 1)];
      }
    };
    auto take = [&](int blk) {
      const int i0 = blk * kBlock + tid * kPer;
      sure = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        x[e] = ahead[e];
        const bool by_score = (unsigned)(i0 + e - lo) < (unsigned)(hi - lo);
        key[e] = by_score ? order_key(x[e]) : 0;
        if (!by_score && i0 + e < n) sure |= 1u << e;
      }
    };
    auto blocks = [&](auto f) {  // f(first slot of this thread) for every block
      if (!MANY) {
        f(tid * kPer);
        return;
      }
      fetch(0);
      for (int blk = 0; blk < nb; ++blk) {
        take(blk);
        if (blk + 1 < nb) fetch(blk + 1);
        f(blk * kBlock + tid * kPer);
      }
    };
    auto each = [&](auto f) {  // f(slot, key), key 0: not one of them
      blocks([&](int i0) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) f(i0 + e, key[e]);
      });
    };
    if (!MANY) {
      fetch(0);
      take(0);
    }

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
        low = max(low, k ? ~k : 0);
        high = max(high, k);
      });
      low = wave_max(low);
      high = wave_max(high);
      if (lane == 0) lows[wave] = low, highs[wave] = high;
      __syncthreads();
      low = ~wave_max(lane < NT / 64 ? lows[lane] : 0);
      high = wave_max(lane < NT / 64 ? highs[lane] : 0);
      // keys whose bits `mask`, those from `top` on, equal prefix's are left: `count` of them
      int top = low == high ? 0 : 32 - __builtin_clz(low ^ high);
      unsigned mask = top >= 32 ? 0 : ~0u << top;
      unsigned prefix = high & mask;
      int count = hi - lo;
      auto digit = [&](auto all_of) {  // one pass: the bits [shift, top) of the last kept key
        const int shift = max(top - kDigit, 0);
        const unsigned width = (1u << (top - shift)) - 1u;
        all_of([&](int, unsigned k) {
          if (((k ^ prefix) & mask) == 0 && k) atomicAdd(&hist[(k >> shift) & width], 1);
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
        mask = ~0u << top;
      };
      auto collect = [&](auto all_of) {  // the `count` candidates to ckey and cslot, in any order
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        all_of([&](int i, unsigned k) {
          if (((k ^ prefix) & mask) == 0 && k) {
            const int c = atomicAdd(&s_count, 1);
            ckey[c] = k;
            cslot[c] = i;
          }
        });
        __syncthreads();
      };
      while (count > kCand && top > 0) digit(each);
      if constexpr (MANY) {
        if (count <= kCand && count > 64 && top > 0) {
          collect(each);
          unsigned fk[kFew];
          int fs[kFew];
#pragma unroll
          for (int e = 0; e < kFew; ++e) {
            const int c = e * NT + tid;
            fk[e] = c < count ? ckey[c] : 0;
            fs[e] = c < count ? cslot[c] : 0;
          }
          auto few = [&](auto f) {
#pragma unroll
            for (int e = 0; e < kFew; ++e) f(fs[e], fk[e]);
          };
          while (count > 64 && top > 0) digit(few);
          if (count <= 64) collect(few);
        } else if (count <= 64) {
          collect(each);
        }
      } else if (count <= 64) {
        collect(each);
      }
      if (count > 64) {  // equal keys: the slot of the need-th of them
        last_key = prefix;
        int seen = 0;
        blocks([&](int i0) {
          int eq = 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) eq += key[e] == prefix;
          int all, at = seen + scan_sum<NT>(eq, tot, all);
          seen += all;
          if (at < need && at + eq >= need) {
#pragma unroll
            for (int e = 0; e < kPer; ++e)
              if (key[e] == prefix && ++at == need) s_slot = i0 + e;
          }
        });
        __syncthreads();
        last_slot = s_slot;
      } else {  // the one with need - 1 larger ones
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
    blocks([&](int i0) {
      unsigned stay = sure;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (key[e] > last_key || (key[e] == last_key && i0 + e <= last_slot)) stay |= 1u << e;
      int all;
      int at = place + scan_sum<NT>(__builtin_popcount(stay), tot, all);
      place += all;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (stay & (1u << e)) {
          if (at >= p0 && at < p1) {
            slots[at] = i0 + e;
            so[at] = x[e];
          }
          at += 1;
        }
    });
  } else {
    for (int i = p0 + tid; i < p1; i += NT) {
      slots[i] = i < n ? i : -1;
      so[i] = i < n ? sc[i] : 0.f;
    }
  }
  __syncthreads();
  gather<NT>(a, b, bh - b * a.H, slots, p0, p1);
}

template <int NT, int kPer, bool MANY>
void launch(EvictArgs a, int cus, hipStream_t st) {
  // rows by 16-byte lanes, 64 at most (D = 256 of 4 bytes)
  a.lanes_log2 = 31 - __builtin_clz(a.D * a.es / 16);
  const int nbh = a.B * a.H, least = 4 * (NT >> a.lanes_log2);  // places of one pass of the copies
  const int64_t most = (a.keep + least - 1) / least, fill = (int64_t)cus * (NT == 1024 ? 1 : 2) / nbh;
  a.nparts = (int)(fill < 1 ? 1 : fill < most ? fill : most);
  hipLaunchKernelGGL((evict_kernel<NT, kPer, MANY>), dim3((unsigned)(nbh * a.nparts)), dim3(NT), 0, st, a);
}
}  // namespace

hipError_t evict_run(const EvictArgs& a, int cus, hipStream_t st) {
  // scores in registers as long as they fit (eight heads of 10698 slots read again in every
  // pass 34 us, in registers 23)
  if (a.C <= 256 * 8) launch<256, 8, false>(a, cus, st);
  else if (a.C <= 1024 * 8) launch<1024, 8, false>(a, cus, st);
  else if (a.C <= 1024 * 16) launch<1024, 16, false>(a, cus, st);
  else launch<1024, 8, true>(a, cus, st);
  return hipGetLastError();
}

}  // namespace flexatt
