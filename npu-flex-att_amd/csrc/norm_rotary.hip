// Queries and keys normalised for each head and turned by their positions in one pass
// (training and its gradients, prefill), or on the way into a K/V cache together with v,
// which may hold 8 bits an element.  No counterpart in the reference, whose inputs are
// already normalised and positioned.
//
// A head's x becomes y = R(pos) (r x w), r = (mean x^2 + eps)^-1/2, with the rotation R of
// rotary.hip.  With g = R^T gy, the gradient turned backwards,
//   dw = sum over the rows of g x r,   dx = r (g w - x r mean(g w x r)),
// so one pass over x and gy has both sums of a row, of x^2 and of g w x, before it needs
// either.
//
// A row of 8 bits: s = max(amax, 2^-100) / top in 32 bits, top = 448 (e4m3) or 127 (int8), and
// codes round(y / s), to the nearest, of two the even one.  y, amax and y / s are in 64 bits,
// sines and norm included (for e4m3 y / s is rounded to 32 bits on its way): next to the border
// of two codes an error of y is one of a whole step, and 32 bits gave a key's code in some 10^5
// the wrong neighbour; the quotients of values of 8 or 11 bits lie on borders, where an
// approximate one decides by its own rounding.  y / s is top (1 + 2^-24) at most, which rounds
// to top: nothing is clamped.  A row with an infinity, NaN or a value beyond 32 bits, be it by a
// weight or a frequency, gets codes of 0 and a scale of NaN: it reads back as NaN.
//
// Bound by memory for long inputs.  As in rotary.hip a thread has 2 x 16 bytes of a token's
// heads and the sines of them, and walks over heads; a row's threads, 2 to 32 lanes next to
// each other, join its sums by lane shifts.  What a thread multiplies by, weights times sines,
// is formed once for all its heads.  The weights' gradients are added up in registers over
// the heads and tokens of a workgroup, in 32 bits, and over the workgroups by a second
// launch, in a fixed order.
//   bf16 B=2 S=4096 Hq=32 Hkv=8 D=128: 37 us, 4.5 TB/s, its gradient 50 us, 5.0 TB/s, and 4
//   fp16 B=4 S=777 Hq=28 Hkv=4 D=64 into a cache of int8: 11 us, 30 MB and the latency
// Short inputs are one launch and its latency, 4 to 5 us.
#include <float.h>

#include "flexatt_device.h"
#include "flexatt_kernels.h"
#include "rotary_device.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
constexpr int kThreads = 256;

// What pairs a thread has: PLAIN its elements c0 + e and c1 + e, two chunks of 16 bytes;
// INTER neighbours in 32 bytes; ANY single elements, where the turned part is no
// multiple of 32 bytes.
enum { kPlain, kInter, kAny };

template <class T, int D>
struct NormCfg {
  static constexpr int E = 16 / (int)sizeof(T);  // pairs of a thread
  static constexpr int UPR = D / (2 * E);        // threads of a row
  static constexpr int TPB = kThreads / UPR;     // tokens of a workgroup
};

// Sum and maximum over the N lanes (2 to 32, aligned) of a row, the same bits in each.
template <int CTRL>
__device__ __forceinline__ float dpp_f(float x) {
  const int i = __float_as_int(x);
  return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ float row_sum(float x) {
  x += dpp_f<0xB1>(x);                               // lane ^ 1
  if constexpr (N >= 4) x += dpp_f<0x4E>(x);         // lane ^ 2
  if constexpr (N >= 8) x += dpp_f<0x141>(x);        // 7 - lane of eight
  if constexpr (N >= 16) x += dpp_f<0x140>(x);       // 15 - lane of sixteen
  if constexpr (N >= 32) x += __shfl_xor(x, 16);
  return x;
}
template <int CTRL>
__device__ __forceinline__ double dpp_d(double x) {
  const i32x2 w = __builtin_bit_cast(i32x2, x);
  return __builtin_bit_cast(double, i32x2{__builtin_amdgcn_update_dpp(w[0], w[0], CTRL, 0xf, 0xf, false),
                                          __builtin_amdgcn_update_dpp(w[1], w[1], CTRL, 0xf, 0xf, false)});
}
// The same in 64 bits of two numbers at once, a sum and a maximum (numbers alone).
template <int N>
__device__ __forceinline__ void row_join(double& sum, double& top) {
  const auto step = [&](double a, double b) {
    sum += a;
    top = fmax(top, b);
  };
  step(dpp_d<0xB1>(sum), dpp_d<0xB1>(top));
  if constexpr (N >= 4) step(dpp_d<0x4E>(sum), dpp_d<0x4E>(top));
  if constexpr (N >= 8) step(dpp_d<0x141>(sum), dpp_d<0x141>(top));
  if constexpr (N >= 16) step(dpp_d<0x140>(sum), dpp_d<0x140>(top));
  if constexpr (N >= 32) step(__shfl_xor(sum, 16), __shfl_xor(top, 16));
}

// A row whose mean square passes 32 bits (elements of 2^64 and more, which fp16 has not) is
// normalised 2^-72 times as large: r x is the same.  Whether the wave has one: a branch that no
// other row takes, free beside the loads (bf16 B=2 S=4096 Hq=32 Hkv=8 D=128, forward and gradient:
// 91 us with it and without).
constexpr float kInf = __builtin_inff(), kLess = 0x1p-72f;
template <class T>
__device__ __forceinline__ bool passes(float m) {
  if constexpr (__is_same(T, _Float16)) return false;
  else return __builtin_amdgcn_ballot_w64(m == kInf) != 0;
}

// A thread's place in a row: its pairs' elements, whether they are turned, their sines.
template <class T, int D, int MODE>
struct Place {
  static constexpr int E = NormCfg<T, D>::E, UPR = NormCfg<T, D>::UPR;
  typedef T vec __attribute__((ext_vector_type(E)));
  int u, c0, c1, half;
  bool inter, rot;

  __device__ __forceinline__ Place(const RotaryArgs& a, int unit) : u(unit), half(a.rotary / 2), inter(a.inter) {
    rot = u < a.rotary / (2 * E);
    c0 = MODE == kPlain && rot ? E * u : 2 * E * u;
    c1 = MODE == kPlain && rot ? c0 + half : c0 + E;
  }
  __device__ __forceinline__ int pair(int e) const { return MODE == kAny ? u + e * UPR : E * u + e; }
  __device__ __forceinline__ bool turned(int e) const { return MODE == kAny ? pair(e) < half : rot; }
  __device__ __forceinline__ int first(int e) const {
    if (MODE == kPlain) return c0 + e;
    if (MODE == kInter) return c0 + 2 * e;
    return inter || !turned(e) ? 2 * pair(e) : pair(e);
  }
  __device__ __forceinline__ int second(int e) const {
    if (MODE == kPlain) return c1 + e;
    if (MODE == kInter) return c0 + 2 * e + 1;
    return inter || !turned(e) ? 2 * pair(e) + 1 : pair(e) + half;
  }
  // the two registers of a row, and element pairs of them
  __device__ __forceinline__ void load(const char* row, vec& x, vec& y) const {
    if constexpr (MODE == kAny) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = ((const T*)row)[first(e)], y[e] = ((const T*)row)[second(e)];
    } else {
      x = *(const vec*)(row + c0 * sizeof(T));
      y = *(const vec*)(row + c1 * sizeof(T));
    }
  }
  __device__ __forceinline__ void store(char* row, const vec& x, const vec& y) const {
    if constexpr (MODE == kAny) {
#pragma unroll
      for (int e = 0; e < E; ++e) ((T*)row)[first(e)] = x[e], ((T*)row)[second(e)] = y[e];
    } else {
      *(vec*)(row + c0 * sizeof(T)) = x;
      *(vec*)(row + c1 * sizeof(T)) = y;
    }
  }
  static __device__ __forceinline__ float a_of(const vec& x, const vec& y, int e) {
    if constexpr (MODE == kInter) return to_f32(2 * e < E ? x[(2 * e) % E] : y[(2 * e) % E]);
    else return to_f32(x[e]);
  }
  static __device__ __forceinline__ float b_of(const vec& x, const vec& y, int e) {
    if constexpr (MODE == kInter) return to_f32(2 * e < E ? x[(2 * e + 1) % E] : y[(2 * e + 1) % E]);
    else return to_f32(y[e]);
  }
  static __device__ __forceinline__ void put(vec& x, vec& y, int e, float a, float b) {
    if constexpr (MODE == kInter) {
      if (2 * e < E) x[(2 * e) % E] = from_f32<T>(a), x[(2 * e + 1) % E] = from_f32<T>(b);
      else y[(2 * e) % E] = from_f32<T>(a), y[(2 * e + 1) % E] = from_f32<T>(b);
    } else {
      x[e] = from_f32<T>(a), y[e] = from_f32<T>(b);
    }
  }
  // The row 2^-72 times as large, where its mean square m passes 32 bits.
  static __device__ __forceinline__ void shrink(vec& x, vec& y, float m) {
    const float s = m == kInf ? kLess : 1.f;
#pragma unroll
    for (int e = 0; e < E; ++e) put(x, y, e, a_of(x, y, e) * s, b_of(x, y, e) * s);
  }
  __device__ __forceinline__ void turns(const RotaryArgs& a, double pos, float (&cs)[E], float (&sn)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      cs[e] = 1.f, sn[e] = 0.f;
      if (turned(e)) turn_of(pos, a.inv_freq[pair(e)], a.mag, 1.f, cs[e], sn[e]);
    }
  }
  // (|x| <= pi / 4; the series' rest is under 4e-13)
  __device__ __forceinline__ void turns(const RotaryArgs& a, double pos, double (&cs)[E], double (&sn)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      cs[e] = 1.0, sn[e] = 0.0;
      if (!turned(e)) continue;
      const double q = pos * (a.inv_freq[pair(e)] * 0.63661977236758134308), n = __builtin_rint(q);
      const double x = (q - n) * 1.57079632679489661923, z = x * x;
      const int k = (int)(n - 4.0 * __builtin_floor(n * 0.25));
      double u = 1.0 / 6227020800, v = 1.0 / 479001600;
      u = __builtin_fma(u, z, -1.0 / 39916800), v = __builtin_fma(v, z, -1.0 / 3628800);
      u = __builtin_fma(u, z, 1.0 / 362880), v = __builtin_fma(v, z, 1.0 / 40320);
      u = __builtin_fma(u, z, -1.0 / 5040), v = __builtin_fma(v, z, -1.0 / 720);
      u = __builtin_fma(u, z, 1.0 / 120), v = __builtin_fma(v, z, 1.0 / 24);
      u = __builtin_fma(u, z, -1.0 / 6), v = __builtin_fma(v, z, -0.5);
      const double sp = __builtin_fma(u * z, x, x), cp = __builtin_fma(v, z, 1.0);
      const double c = (k & 1) ? sp : cp, s = (k & 1) ? cp : sp;
      cs[e] = ((k == 1 || k == 2) ? -c : c) * (double)a.mag;
      sn[e] = ((k & 2) ? -s : s) * (double)a.mag;
    }
  }
};

template <class T>
__device__ __forceinline__ float weight_at(const void* w, int wide, int i) {
  return wide ? ((const float*)w)[i] : to_f32(((const T*)w)[i]);
}

// Four codes of 8 bits, of values that round to the kind's largest in size at most.
__device__ __forceinline__ unsigned code4(int kind, double a, double b, double c, double d) {
  if (kind == FLEXATT_E4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32((float)a, (float)b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32((float)c, (float)d, w, true);
  }
  // x + 1.5 2^52 rounds x to a whole number, whose low byte is the code
  const auto whole = [](double x) { return (unsigned)__builtin_bit_cast(i32x2, x + 0x1.8p52)[0]; };
  return (whole(a) & 255) | (whole(b) & 255) << 8 | (whole(c) & 255) << 16 | whole(d) << 24;
}

// A workgroup has some heads of q, of k or of v (grid.y: the groups of a.hpt of each) for
// its tokens.  A thread's first rows are on their way before it forms its sines, and the
// next ones while it works on a pair.
template <class T, int D, int MODE, bool CODED>
__global__ __launch_bounds__(kThreads) void norm_rotary_kernel(NormRotaryArgs n) {
  using C = NormCfg<T, D>;
  using P = Place<T, D, MODE>;
  typedef typename P::vec vec;
  // rows on their way at once (codes: two take registers that a fourth wave needs, B=4 S=777
  // D=64 22.3 -> 24.2 us with the read-back)
  constexpr int E = C::E, UPR = C::UPR, U = CODED ? 1 : 2, ES = (int)sizeof(T);
  const RotaryArgs& a = n.r;
  const int64_t tok = (int64_t)blockIdx.x * C::TPB + threadIdx.x / UPR;
  if (tok >= (int64_t)a.B * a.S) return;  // (whole rows of threads)
  const int which = (int)blockIdx.y < n.q_groups ? 0 : (int)blockIdx.y < n.q_groups + n.k_groups ? 1 : 2;
  const int lo = ((int)blockIdx.y - (which == 0 ? 0 : n.q_groups + (which == 2 ? n.k_groups : 0))) * a.hpt;
  const int rows = min(a.hpt, (which ? a.Hkv : a.Hq) - lo);
  int b, s;
  int64_t slot;
  double pos;
  token_of(a, tok, b, s, slot, pos);
  const P at(a, threadIdx.x % UPR);

  const auto of = [&](auto q, auto k, auto v) { return which == 0 ? q : which == 1 ? k : v; };
  const View vx = {of(a.q.data, a.k.data, a.v.data), of(a.q.sb, a.k.sb, a.v.sb), of(a.q.sh, a.k.sh, a.v.sh),
                   of(a.q.ss, a.k.ss, a.v.ss)};
  const MutView vy = {of(a.qo.data, a.ko.data, a.vo.data), of(a.qo.sb, a.ko.sb, a.vo.sb), of(a.qo.sh, a.ko.sh, a.vo.sh),
                      of(a.qo.ss, a.ko.ss, a.vo.ss)};
  const bool cached = which != 0 && a.cache_rows > 0, coded = CODED && cached;
  const char* src = (const char*)vx.data + (b * vx.sb + lo * vx.sh + s * vx.ss) * ES;
  const bool kept = !cached || (slot >= 0 && slot < a.cache_rows);  // (a row outside the cache is not written)
  char* dst = (char*)vy.data + (b * vy.sb + lo * vy.sh + (cached ? slot : (int64_t)s) * vy.ss) * (coded ? 1 : ES);
  float* scales = nullptr;
  if (coded) scales = (which == 1 ? n.k_scales : n.v_scales) + ((int64_t)b * a.Hkv + lo) * a.cache_rows + slot;
  vec x[U], y[U], nx[U], ny[U];
  auto fetch = [&](int r0, vec (&p)[U], vec (&q)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (r0 + i < rows) at.load(src + (r0 + i) * vx.sh * ES, p[i], q[i]);
  };
  fetch(0, x, y);

  const bool norm = n.norm && which != 2;
  const void* w = which == 0 ? n.wq : n.wk;
  // y = (a ac - b bs, b bc + a as), times r
  if (coded) {
    if (!kept) return;  // (whole rows of threads)
    double ac[E], as[E], bc[E], bs[E];
#pragma unroll
    for (int e = 0; e < E; ++e) ac[e] = bc[e] = 1.0, as[e] = bs[e] = 0.0;
    if (which != 2) {
      double cs[E], sn[E];
      at.turns(a, pos, cs, sn);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double wa = norm ? weight_at<T>(w, n.w_wide, at.first(e)) : 1.f;
        const double wb = norm ? weight_at<T>(w, n.w_wide, at.second(e)) : 1.f;
        ac[e] = wa * cs[e], as[e] = wa * sn[e], bc[e] = wb * cs[e], bs[e] = wb * sn[e];
      }
    }
    // A weight, or an angle's frequency, that is an infinity or NaN makes every row one that is
    // not of numbers (0 times an infinity too), which the maximum of the rows would not show.
    double odd = 0.0, none = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) odd += 0.0 * ac[e] + 0.0 * as[e] + 0.0 * bc[e] + 0.0 * bs[e];
    row_join<UPR>(odd, none);
    const bool sound = odd == 0.0;
    for (int r0 = 0; r0 < rows; ++r0) {
      fetch(r0 + 1, nx, ny);
      double ya[E], yb[E], sq = 0.0, top = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double p = P::a_of(x[0], y[0], e), q = P::b_of(x[0], y[0], e);
        sq = __builtin_fma(p, p, sq);
        sq = __builtin_fma(q, q, sq);
        ya[e] = __builtin_fma(p, ac[e], -(q * bs[e]));
        yb[e] = __builtin_fma(q, bc[e], p * as[e]);
        top = fmax(top, fmax(fabs(ya[e]), fabs(yb[e])));
      }
      row_join<UPR>(sq, top);
      double r = 1.0, root = 1.0;
      if (norm) {  // r = m^-1/2, m of any size: of the approximate one in 64 bits one step more leaves 2e-14
        const double m = __builtin_fma(sq, 1.0 / D, (double)n.eps);
        r = __builtin_amdgcn_rsq(m);
        r *= __builtin_fma(-0.5 * m * r, r, 1.5);
        root = m * r;
      }
      top *= r;
      // (sq: of an infinity or NaN it is none of the numbers that 32 bits give)
      const bool fine = sound && sq < 0x1p300 && top <= (double)FLT_MAX;
      // (the largest numbers a little less, so that code * scale is one)
      const double size = fmin(fmax(top, 0x1p-100), 0x1.fffffp127);
      const float scale = (float)(size * (n.kind == FLEXATT_E4M3 ? 1.0 / 448 : 1.0 / 127));
      // y r / scale: the quotient by (scale / r), with its rest (exact where r is 1)
      const double by = (double)scale * root;
      double inv = __builtin_amdgcn_rcpf(scale);
      inv *= __builtin_fma(-inv, (double)scale, 2.0) * r;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const auto over = [&](double v) {
          const double t = v * inv;
          return __builtin_fma(__builtin_fma(-t, by, v), inv, t);
        };
        ya[e] = over(ya[e]), yb[e] = over(yb[e]);
      }
      if (!fine) {
#pragma unroll
        for (int e = 0; e < E; ++e) ya[e] = yb[e] = 0.0;
      }
      char* to = dst + r0 * vy.sh;
      if (at.u == 0) scales[(int64_t)r0 * a.cache_rows] = fine ? scale : __builtin_nanf("");
      if constexpr (MODE == kAny) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const unsigned c = code4(n.kind, ya[e], yb[e], ya[e + 1], yb[e + 1]);
          to[at.first(e)] = (char)c, to[at.second(e)] = (char)(c >> 8);
          to[at.first(e + 1)] = (char)(c >> 16), to[at.second(e + 1)] = (char)(c >> 24);
        }
      } else if constexpr (MODE == kInter) {  // 2 E neighbours
        unsigned c[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) c[e] = code4(n.kind, ya[2 * e], yb[2 * e], ya[2 * e + 1], yb[2 * e + 1]);
        if constexpr (E == 8) *(i32x4*)(to + at.c0) = i32x4{(int)c[0], (int)c[1], (int)c[2], (int)c[3]};
        else *(i32x2*)(to + at.c0) = i32x2{(int)c[0], (int)c[1]};
      } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const double* v = g ? yb : ya;
          char* d = to + (g ? at.c1 : at.c0);
          const unsigned c = code4(n.kind, v[0], v[1], v[2], v[3]);
          if constexpr (E == 8) *(i32x2*)d = i32x2{(int)c, (int)code4(n.kind, v[4], v[5], v[6], v[7])};
          else *(int*)d = (int)c;
        }
      }
      x[0] = nx[0], y[0] = ny[0];
    }
    return;
  }
  float ac[E], as[E], bc[E], bs[E];
  if (which != 2) {
    float cs[E], sn[E];
    at.turns(a, pos, cs, sn);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float wa = norm ? weight_at<T>(w, n.w_wide, at.first(e)) : 1.f;
      const float wb = norm ? weight_at<T>(w, n.w_wide, at.second(e)) : 1.f;
      ac[e] = wa * cs[e], as[e] = wa * sn[e], bc[e] = wb * cs[e], bs[e] = wb * sn[e];
    }
  }
  for (int r0 = 0; r0 < rows; r0 += U) {
    fetch(r0 + U, nx, ny);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (r0 + i >= rows) break;
      char* to = dst + (r0 + i) * vy.sh * ES;
      if (which != 2) {
        float ya[E], yb[E], m = 0.f;
        for (bool again = false;; again = true) {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float p = P::a_of(x[i], y[i], e), q = P::b_of(x[i], y[i], e);
            sq = __builtin_fmaf(p, p, sq);
            sq = __builtin_fmaf(q, q, sq);
            const bool t = at.turned(e);
            ya[e] = t ? __builtin_fmaf(p, ac[e], -(q * bs[e])) : p * ac[e];
            yb[e] = t ? __builtin_fmaf(q, bc[e], p * as[e]) : q * bc[e];
          }
          if (!norm) break;
          m = __builtin_fmaf(row_sum<UPR>(sq), 1.0f / D, again && m == kInf ? n.eps * kLess * kLess : n.eps);
          if (again || !passes<T>(m)) break;
          at.shrink(x[i], y[i], m);
        }
        if (norm) {
          const float r = __builtin_amdgcn_rsqf(m);
#pragma unroll
          for (int e = 0; e < E; ++e) ya[e] *= r, yb[e] *= r;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) P::put(x[i], y[i], e, ya[e], yb[e]);
      }
      if (kept) at.store(to, x[i], y[i]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = nx[i], y[i] = ny[i];
  }
}

// Gradients.  A workgroup has the heads of one weight (grid.y: groups of a.hpt q heads,
// then of k heads) and every grid.x-th set of tokens.  Three waves a SIMD are what its plan
// counts on (neighbouring pairs in bf16 else take the registers of two: D=128 94 -> 99 us).
template <class T, int D, int MODE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(MODE == kAny ? 2 : 3)))
void norm_rotary_grad_kernel(NormRotaryArgs n) {
  using C = NormCfg<T, D>;
  using P = Place<T, D, MODE>;
  typedef typename P::vec vec;
  constexpr int E = C::E, UPR = C::UPR, TPB = C::TPB;
  const RotaryArgs& a = n.r;
  const int which = (int)blockIdx.y < n.q_groups ? 0 : 1;
  const int lo = ((int)blockIdx.y - (which ? n.q_groups : 0)) * a.hpt, hi = min(lo + a.hpt, which ? a.Hkv : a.Hq);
  const View& vx = which ? a.k : a.q;
  const View& vg = which ? n.gk : n.gq;
  const MutView& vd = which ? a.ko : a.qo;
  const void* w = which ? n.wk : n.wq;
  const P at(a, threadIdx.x % UPR);
  float wa[E], wb[E], da[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    wa[e] = weight_at<T>(w, n.w_wide, at.first(e));
    wb[e] = weight_at<T>(w, n.w_wide, at.second(e));
    da[e] = db[e] = 0.f;
  }
  const int64_t tokens = (int64_t)a.B * a.S;
  for (int64_t t0 = (int64_t)blockIdx.x * TPB; t0 < tokens; t0 += (int64_t)gridDim.x * TPB) {
    const int64_t tok = t0 + threadIdx.x / UPR;
    if (tok >= tokens) break;  // (whole rows of threads)
    int b, s;
    int64_t slot;
    double pos;
    token_of(a, tok, b, s, slot, pos);
    float cs[E], sn[E];
    at.turns(a, pos, cs, sn);
    const char* px = (const char*)vx.data + (b * vx.sb + lo * vx.sh + s * vx.ss) * (int)sizeof(T);
    const char* pg = (const char*)vg.data + (b * vg.sb + lo * vg.sh + s * vg.ss) * (int)sizeof(T);
    char* pd = (char*)vd.data + (b * vd.sb + lo * vd.sh + s * vd.ss) * (int)sizeof(T);
    constexpr int U = 2;  // heads loaded before the first is stored
    for (int hh = lo; hh < hi; hh += U) {
      vec x[U], y[U], gx[U], gy[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (hh + i >= hi) break;
        at.load(px, x[i], y[i]);
        at.load(pg, gx[i], gy[i]);
        px += vx.sh * (int)sizeof(T);
        pg += vg.sh * (int)sizeof(T);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (hh + i >= hi) break;
        float ga[E], gb[E], ms = 0.f, dot, down = 1.f;  // (x of a row that is shrunk: r x is as it was)
        for (bool again = false;; again = true) {
          float sq = 0.f;
          dot = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float p = P::a_of(x[i], y[i], e), q = P::b_of(x[i], y[i], e);
            const float u = P::a_of(gx[i], gy[i], e), v = P::b_of(gx[i], gy[i], e);
            const bool t = at.turned(e);
            ga[e] = t ? __builtin_fmaf(u, cs[e], v * sn[e]) : u;
            gb[e] = t ? __builtin_fmaf(v, cs[e], -(u * sn[e])) : v;
            sq = __builtin_fmaf(p, p, sq);
            sq = __builtin_fmaf(q, q, sq);
            dot = __builtin_fmaf(ga[e] * wa[e], p, dot);
            dot = __builtin_fmaf(gb[e] * wb[e], q, dot);
          }
          ms = __builtin_fmaf(row_sum<UPR>(sq), 1.0f / D, n.eps * down * down);
          if (again || !passes<T>(ms)) break;
          at.shrink(x[i], y[i], ms);
          if (ms == kInf) down = kLess;
        }
        const float r = __builtin_amdgcn_rsqf(ms), rd = r * down;
        const float m = row_sum<UPR>(dot) * (1.0f / D) * r * r;  // mean(g w x r) r
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float p = P::a_of(x[i], y[i], e), q = P::b_of(x[i], y[i], e);
          da[e] = __builtin_fmaf(ga[e] * r, p, da[e]);
          db[e] = __builtin_fmaf(gb[e] * r, q, db[e]);
          P::put(gx[i], gy[i], e, rd * __builtin_fmaf(-m, p, ga[e] * wa[e]), rd * __builtin_fmaf(-m, q, gb[e] * wb[e]));
        }
        at.store(pd, gx[i], gy[i]);
        pd += vd.sh * (int)sizeof(T);
      }
    }
  }

  // the workgroup's sums: over the rows of a wave by lane shifts, over the waves in order
  __shared__ float sums[kThreads / 64][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int e = 0; e < E; ++e) {
#pragma unroll
    for (int y = UPR; y < 64; y *= 2) da[e] += __shfl_xor(da[e], y), db[e] += __shfl_xor(db[e], y);
    if (lane < UPR) sums[wave][at.first(e)] = da[e], sums[wave][at.second(e)] = db[e];
  }
  __syncthreads();
  float* part = n.part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * D;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < kThreads / 64; ++v) t += sums[v][d];
    part[d] = t;
  }
}

// dw of both weights from the workgroups' sums: a workgroup has 32 elements of one, a
// thread four of them of every 128th row.
template <class T, int D>
__global__ __launch_bounds__(1024) void norm_weight_grad_kernel(NormRotaryArgs n, int rows_q, int rows_k) {
  const int which = blockIdx.x / (D / 32), c0 = blockIdx.x % (D / 32) * 32;
  const int rows = which ? rows_k : rows_q;
  const float* part = n.part + (which ? (int64_t)rows_q * D : 0) + c0 + (threadIdx.x & 7) * 4;
  f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r = threadIdx.x >> 3; r < rows; r += 128) {
    const f32x4 v = *(const f32x4*)(part + (int64_t)r * D);
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] += v[j];
  }
  __shared__ f32x4 sums[16][8];
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int y = 8; y < 64; y *= 2) t[j] += __shfl_xor(t[j], y);
  if ((threadIdx.x & 63) < 8) sums[wave][threadIdx.x & 7] = t;
  __syncthreads();
  if (threadIdx.x < 32) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += sums[i][threadIdx.x >> 2][threadIdx.x & 3];
    void* out = which ? n.dwk : n.dwq;
    if (n.w_wide) ((float*)out)[c0 + threadIdx.x] = v;
    else ((T*)out)[c0 + threadIdx.x] = from_f32<T>(v);
  }
}

template <class T, int D>
int mode_of(const RotaryArgs& a) {
  return a.rotary % (2 * NormCfg<T, D>::E) ? kAny : a.inter ? kInter : kPlain;
}

template <class T, int D, bool CODED>
hipError_t launch(NormRotaryArgs n, hipStream_t st) {
  RotaryArgs& a = n.r;
  const int64_t nb = ((int64_t)a.B * a.S + NormCfg<T, D>::TPB - 1) / NormCfg<T, D>::TPB;
  // heads per thread: all of them once the tokens alone make four workgroups a CU, and
  // whole rounds of the loads (rotary.hip)
  int64_t groups = (1024 + nb - 1) / nb;
  if (groups > a.heads) groups = a.heads;
  a.hpt = (int)((a.heads + groups - 1) / groups);
  if (a.hpt > 2) a.hpt = (a.hpt + 3) / 4 * 4;
  n.q_groups = (a.Hq + a.hpt - 1) / a.hpt;
  n.k_groups = (a.Hkv + a.hpt - 1) / a.hpt;
  const int v_groups = a.cache_rows > 0 ? n.k_groups : 0;
  const dim3 grid((unsigned)nb, (unsigned)(n.q_groups + n.k_groups + v_groups)), block(kThreads);
  switch (mode_of<T, D>(a)) {
    case kPlain: hipLaunchKernelGGL((norm_rotary_kernel<T, D, kPlain, CODED>), grid, block, 0, st, n); break;
    case kInter: hipLaunchKernelGGL((norm_rotary_kernel<T, D, kInter, CODED>), grid, block, 0, st, n); break;
    default: hipLaunchKernelGGL((norm_rotary_kernel<T, D, kAny, CODED>), grid, block, 0, st, n);
  }
  return hipGetLastError();
}

template <class T, int D>
hipError_t launch_grad(NormRotaryArgs n, hipStream_t st) {
  RotaryArgs& a = n.r;
  const NormGradPlan p = norm_grad_plan(a.B, a.S, a.Hq, a.Hkv, D, (int)sizeof(T));
  a.hpt = p.hpt;
  n.q_groups = p.q_groups;
  const dim3 grid((unsigned)p.columns, (unsigned)(p.q_groups + p.k_groups)), block(kThreads);
  switch (mode_of<T, D>(a)) {
    case kPlain: hipLaunchKernelGGL((norm_rotary_grad_kernel<T, D, kPlain>), grid, block, 0, st, n); break;
    case kInter: hipLaunchKernelGGL((norm_rotary_grad_kernel<T, D, kInter>), grid, block, 0, st, n); break;
    default: hipLaunchKernelGGL((norm_rotary_grad_kernel<T, D, kAny>), grid, block, 0, st, n);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((norm_weight_grad_kernel<T, D>), dim3((a.Hkv > 0 ? 2 : 1) * (D / 32)), dim3(1024), 0, st, n,
                     p.columns * p.q_groups, p.columns * p.k_groups);
  return hipGetLastError();
}
}  // namespace

#define FLEXATT_CAT2(a, b) a##b
#define FLEXATT_CAT(a, b) FLEXATT_CAT2(a, b)
hipError_t FLEXATT_CAT(norm_rotary_d, FLEXATT_D)(int dtype, const NormRotaryArgs& n, hipStream_t st) {
  switch (dtype) {
    case FLEXATT_F32: return n.kind ? launch<float, FLEXATT_D, true>(n, st) : launch<float, FLEXATT_D, false>(n, st);
    case FLEXATT_F16:
      return n.kind ? launch<_Float16, FLEXATT_D, true>(n, st) : launch<_Float16, FLEXATT_D, false>(n, st);
    case FLEXATT_BF16: return n.kind ? launch<__bf16, FLEXATT_D, true>(n, st) : launch<__bf16, FLEXATT_D, false>(n, st);
    default: return hipErrorInvalidValue;
  }
}
hipError_t FLEXATT_CAT(norm_rotary_grad_d, FLEXATT_D)(int dtype, const NormRotaryArgs& n, hipStream_t st) {
  switch (dtype) {
    case FLEXATT_F32: return launch_grad<float, FLEXATT_D>(n, st);
    case FLEXATT_F16: return launch_grad<_Float16, FLEXATT_D>(n, st);
    case FLEXATT_BF16: return launch_grad<__bf16, FLEXATT_D>(n, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace flexatt
