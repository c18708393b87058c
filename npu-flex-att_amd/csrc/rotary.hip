// Rotary positions: q and k of every token turned by its position, out of place
// (training, prefill; the gradient is the same turn backwards), or on the way
// into a K/V cache together with v (serving).  No counterpart in the reference,
// whose inputs are already positioned.
//
// Pair i of the first `rotary_dim` elements of a head, (i, i + r/2) in the half
// layout and (2i, 2i+1) in the interleaved one, is a point of the plane that is
// turned by pos * inv_freq[i] and stretched by the magnitude; the other elements
// are copied.
//
// The angle is formed in 64 bits and reduced to quarter turns there: at position
// 100000 an fp32 product is off by up to 2^-24 * 100000 = 0.006 radians.  What is
// left of it, within an eighth of a turn, is rounded to 32 bits and goes through the
// Taylor series of sine and cosine there (first terms left out: x^11/11! and x^12/12!,
// under 2e-9 at pi/4, where a half step is 3e-8).
//
// Bound by memory: each element is read and written once.  A thread keeps the
// sines of its 2 x 16 bytes of one token and walks over heads, so the angles cost
// nothing beside the copies, and loads four heads at once before it stores any.
// bf16 B=2 S=4096 Hq=32 Hkv=8 D=128: 168 MB in 32 us, 5.3 TB/s, the rate of a large copy.
// Stores that pass the caches by were slower where it counts: alone as fast, and the
// attention behind them 1 to 2% longer.
// Short calls are latency: the append of one token to 8 caches 4.2 us.
#include "flexatt_device.h"
#include "flexatt_kernels.h"
#include "rotary_device.h"

namespace flexatt {

namespace {
constexpr int kThreads = 256;
constexpr int kRows = 4;  // heads loaded before the first is stored

// One head of one token in the launch's order: q heads, k heads, v heads.
struct Rows {
  const char* src;
  char* dst;   // nullptr: outside the cache, nothing written
  bool turned;
};
__device__ __forceinline__ Rows rows_of(const RotaryArgs& a, int h, int b, int s, int64_t slot, int es) {
  Rows r;
  const int which = h < a.Hq ? 0 : h < a.Hq + a.Hkv ? 1 : 2;
  const int hh = which == 0 ? h : which == 1 ? h - a.Hq : h - a.Hq - a.Hkv;
  const View& x = which == 0 ? a.q : which == 1 ? a.k : a.v;
  const MutView& y = which == 0 ? a.qo : which == 1 ? a.ko : a.vo;
  const bool cached = which != 0 && a.cache_rows > 0;
  const int64_t row = cached ? slot : s;
  r.src = (const char*)x.data + (b * x.sb + hh * x.sh + s * x.ss) * es;
  r.dst = cached && (slot < 0 || slot >= a.cache_rows)
              ? nullptr
              : (char*)y.data + (b * y.sb + hh * y.sh + row * y.ss) * es;
  r.turned = which != 2;
  return r;
}

// Rotated part a multiple of 2 E elements (E: elements of 16 bytes): a thread has
// E whole pairs of a token, two 16-byte chunks of each head.
template <class T, int D, bool INTER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int E = 16 / (int)sizeof(T), UPR = D / (2 * E), TPB = kThreads / UPR;
  typedef T vec __attribute__((ext_vector_type(E)));
  const int64_t n = (int64_t)blockIdx.x * TPB + threadIdx.x / UPR;
  const int u = threadIdx.x % UPR;
  if (n >= (int64_t)a.B * a.S) return;
  int b, s;
  int64_t slot;
  double pos;
  token_of(a, n, b, s, slot, pos);

  // unit u: pairs E u .. E u + E - 1 where they are rotated, else two chunks to copy
  const int ur = a.rotary / (2 * E);
  const bool rot = u < ur;
  int c0, c1;  // first elements of the two chunks
  if (INTER || !rot) {
    c0 = 2 * E * u;
    c1 = c0 + E;
  } else {
    c0 = E * u;
    c1 = c0 + a.rotary / 2;
  }
  float cs[E], sn[E];
#pragma unroll
  for (int e = 0; e < E; ++e) cs[e] = 1.f, sn[e] = 0.f;
  if (rot) {
#pragma unroll
    for (int e = 0; e < E; ++e) turn_of(pos, a.inv_freq[E * u + e], a.mag, a.sign, cs[e], sn[e]);
  }

  constexpr int U = kRows;
  const int h1 = min((int)(blockIdx.y + 1) * a.hpt, a.heads);
  for (int h0 = blockIdx.y * a.hpt; h0 < h1; h0 += U) {
    vec x0[U], x1[U];
    Rows r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (h0 + i >= h1) break;
      r[i] = rows_of(a, h0 + i, b, s, slot, sizeof(T));
      x0[i] = *(const vec*)(r[i].src + c0 * sizeof(T));
      x1[i] = *(const vec*)(r[i].src + c1 * sizeof(T));
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (h0 + i >= h1) break;
      vec y0 = x0[i], y1 = x1[i];
      if (rot && r[i].turned) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float p = INTER ? to_f32(2 * e < E ? x0[i][(2 * e) % E] : x1[i][(2 * e) % E]) : to_f32(x0[i][e]);
          const float q = INTER ? to_f32(2 * e < E ? x0[i][(2 * e + 1) % E] : x1[i][(2 * e + 1) % E]) : to_f32(x1[i][e]);
          const T v = from_f32<T>(__builtin_fmaf(p, cs[e], -(q * sn[e])));
          const T w = from_f32<T>(__builtin_fmaf(q, cs[e], p * sn[e]));
          if (INTER) {
            if (2 * e < E) y0[(2 * e) % E] = v, y0[(2 * e + 1) % E] = w;
            else y1[(2 * e) % E] = v, y1[(2 * e + 1) % E] = w;
          } else {
            y0[e] = v;
            y1[e] = w;
          }
        }
      }
      if (r[i].dst) {
        *(vec*)(r[i].dst + c0 * sizeof(T)) = y0;
        *(vec*)(r[i].dst + c1 * sizeof(T)) = y1;
      }
    }
  }
}

// Any even rotary_dim: a thread has one pair of a token (or two elements to copy).
template <class T>
__global__ __launch_bounds__(kThreads) void rotary_any_kernel(RotaryArgs a) {
  const int half = a.D / 2;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t n = i / half;
  const int u = (int)(i % half);
  if (n >= (int64_t)a.B * a.S) return;
  int b, s;
  int64_t slot;
  double pos;
  token_of(a, n, b, s, slot, pos);
  const bool rot = u < a.rotary / 2;
  const int c0 = rot && !a.inter ? u : 2 * u, c1 = rot && !a.inter ? u + a.rotary / 2 : 2 * u + 1;
  float cs = 1.f, sn = 0.f;
  if (rot) turn_of(pos, a.inv_freq[u], a.mag, a.sign, cs, sn);
  const int h1 = min((int)(blockIdx.y + 1) * a.hpt, a.heads);
  for (int h = blockIdx.y * a.hpt; h < h1; ++h) {
    const Rows r = rows_of(a, h, b, s, slot, sizeof(T));
    T p = ((const T*)r.src)[c0], q = ((const T*)r.src)[c1];
    if (rot && r.turned) {
      const float x = to_f32(p), y = to_f32(q);
      p = from_f32<T>(__builtin_fmaf(x, cs, -(y * sn)));
      q = from_f32<T>(__builtin_fmaf(y, cs, x * sn));
    }
    if (r.dst) {
      ((T*)r.dst)[c0] = p;
      ((T*)r.dst)[c1] = q;
    }
  }
}

template <class T, int D>
void launch_d(const RotaryArgs& a, dim3 grid, hipStream_t st) {
  if (a.inter) hipLaunchKernelGGL((rotary_kernel<T, D, true>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((rotary_kernel<T, D, false>), grid, dim3(kThreads), 0, st, a);
}

template <class T>
hipError_t launch(RotaryArgs a, hipStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool wide = a.rotary % (2 * E) == 0;
  const int per_block = wide ? kThreads / (a.D / (2 * E)) : 1;
  const int64_t tokens = (int64_t)a.B * a.S;
  const int64_t nb = wide ? (tokens + per_block - 1) / per_block : (tokens * (a.D / 2) + kThreads - 1) / kThreads;
  // heads per thread: all of them once the tokens alone make 1024 workgroups, four a CU,
  // and whole rounds of the loads (bf16 B=2 S=4096 Hq=32 Hkv=8 D=128, 256 workgroups of
  // tokens: 5 heads a thread 34.6 us, 12 31.9; with its gradients 75.8 and 73.8, and 79
  // with all 40)
  int64_t groups = (1024 + nb - 1) / nb;
  if (groups > a.heads) groups = a.heads;
  a.hpt = (int)((a.heads + groups - 1) / groups);
  if (a.hpt > kRows / 2) a.hpt = (a.hpt + kRows - 1) / kRows * kRows;
  const dim3 grid((unsigned)nb, (unsigned)((a.heads + a.hpt - 1) / a.hpt));
  if (!wide) {
    hipLaunchKernelGGL((rotary_any_kernel<T>), grid, dim3(kThreads), 0, st, a);
    return hipGetLastError();
  }
  switch (a.D) {
    case 32: launch_d<T, 32>(a, grid, st); break;
    case 64: launch_d<T, 64>(a, grid, st); break;
    case 128: launch_d<T, 128>(a, grid, st); break;
    case 256: launch_d<T, 256>(a, grid, st); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}
}  // namespace

hipError_t rotary_run(int dtype, const RotaryArgs& a, hipStream_t st) {
  switch (dtype) {
    case FLEXATT_F32: return launch<float>(a, st);
    case FLEXATT_F16: return launch<_Float16>(a, st);
    case FLEXATT_BF16: return launch<__bf16>(a, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace flexatt
