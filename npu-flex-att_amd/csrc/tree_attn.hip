// Attention of a tree of drafted tokens over a K/V cache (speculative decoding;
// with one token, ordinary decoding over a batch of caches of unequal lengths).
// No counterpart in the reference, which has no cache.
//
// Semantics: those of the forward (npu_flash_attention.py:17-166: scale, soft-cap,
// mask, online softmax in the log2 domain, LSE in natural log) with, for drafted
// token t of a sequence of n cached tokens, the keys j < n (with a window,
// n + depth[t] - j <= W) and those slots n + u, u < T, whose mask[t][u] is set
// (no mask: u <= t).  A row without keys is 0 with LSE -inf; a sequence whose
// n + T rows do not fit the cache (or n < 0) is NaN.
//
// Decomposition (that of fwd_split.hip)
//  * the G * T query rows of one KV head are packed with the heads innermost into
//    tiles of 32, the columns of an MFMA tile, so heads and tokens share K and V;
//  * a workgroup has one row tile of one (b, hkv) and a contiguous chunk of 32-key
//    tiles; wave w takes tiles w, w + NW, ... with its own LDS stages and online
//    softmax, no barriers; the waves' states are combined through LDS;
//  * the chunks are cut on the device from the sequence's own length, so that a
//    cache of large capacity that holds little costs what it holds; the partials
//    of a row (O over its row sum, LSE) are merged in a fixed order.
//  * rows behind n + T are never read: the copies repeat the last row instead, so
//    what a cache holds there (NaN too) does not matter.
// What bounds it: K and V from HBM for long caches.
#include "flexatt_device.h"
#include "flexatt_kernels.h"

#ifndef FLEXATT_D
#error "FLEXATT_D (head dim) must be defined"
#endif

namespace flexatt {

namespace {
constexpr float kTreeRescale = 8.0f;  // lazy rescale threshold, log2 units (as the forward)

// LDS stages by the bytes of a row: two of a K and a V tile per wave, so that the
// next tile is in flight during the whole of this one, where four waves' fit
// 160 KB (rows up to 256 bytes); one above, K refilled after the scores and V
// after P V; two waves of 1 KB rows.
template <class T, int D>
struct TreeCfg {
  static constexpr int BN = 32;                       // keys per tile
  static constexpr int ROWB = D * (int)sizeof(T);     // bytes per row
  static constexpr int KC = ROWB / 32;                // 32-byte steps of S^T = K Q^T
  static constexpr int DB = D / 32;                   // 32-row blocks of O^T
  static constexpr int CPR = ROWB / 16;               // 16-byte chunks per row
  static constexpr int TB = BN * ROWB;                // bytes of one K or V tile
  static constexpr int E = TB / 1024;                 // 1 KB copies per tile
  static constexpr int NW = ROWB <= 512 ? 4 : 2;      // waves per workgroup
  static constexpr int ST = ROWB <= 256 ? 2 : 1;      // stages
  static constexpr int WAVEB = ST * 2 * TB;
  static constexpr int COMBB = NW * 64 * 4 * (2 + 16 * DB);
  static constexpr int LDSB = NW * WAVEB > COMBB ? NW * WAVEB : COMBB;
  static_assert(E * 1024 == TB && LDSB <= 160 * 1024, "LDS");
};

// V tiles of 32-bit elements are read one element per lane, 32 of a row by each
// half wave from rows 4 apart: the second one's chunks sit in the other half of
// a 256-byte bank row.
template <int CPR>
__device__ __forceinline__ int swz_v32(int r, int c) {
  if constexpr (CPR >= 16) return c ^ (((r >> 2) & 1) << 3);
  else return c;
}
template <class T, int CPR>
__device__ __forceinline__ int swz_v(int r, int p) {  // logical chunk at physical chunk p
  if constexpr (sizeof(T) == 4) return swz_v32<CPR>(r, p);
  else return swz_tr_inv<CPR>(r, p);
}

// One 32-byte step of the scores: A rows are keys, B columns query rows; lane half
// h has the bytes 16 h .. 16 h + 15 of the step of its row.
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

// The key tiles [t0, t1) of sequence b and how they are cut: ns chunks of `chunk`.
struct TreePlan {
  int n, t0, t1, ns, chunk;
  bool bad;
};
template <int NW>
__device__ __forceinline__ TreePlan tree_plan(const TreeArgs& a, int b) {
  TreePlan x;
  x.n = __builtin_amdgcn_readfirstlane(a.lengths[b]);
  x.bad = x.n < 0 || x.n > a.p.Skv - a.p.Sq;
  if (x.bad) x.n = 0;
  x.t0 = a.p.window > 0 ? max(x.n - a.p.window, 0) / 32 : 0;
  x.t1 = (x.n + a.p.Sq + 31) / 32;
  const int nt = x.t1 - x.t0;
  int ns = x.bad ? 1 : min(a.nsplit, nt / (2 * NW));  // at least two tiles per wave
  if (ns < 1) ns = 1;
  x.chunk = (nt + ns - 1) / ns;
  x.ns = (nt + x.chunk - 1) / x.chunk;
  return x;
}
}  // namespace

template <class T, int D, int NW, bool CAP>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(D * sizeof(T) >= 512 ? 1 : 2)))
void tree_attn_kernel(TreeArgs a) {
  using C = TreeCfg<T, D>;
  constexpr int ST = C::ST;
  __shared__ __attribute__((aligned(1024))) char smem[C::LDSB];

  const Shape& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, l32 = lane & 31;

  // (b, hkv, row tile, split): the row tiles of one chunk are neighbours
  int item = blockIdx.x;
  const int rt = item % a.nrt;
  item /= a.nrt;
  const int s = item % a.nsplit;
  const int bh = item / a.nsplit;
  const int hk = bh % p.Hkv, b = bh / p.Hkv;
  const TreePlan pl = tree_plan<NW>(a, b);
  if (s >= pl.ns) return;

  // packed query row of this lane
  const int R = p.G * p.Sq;
  const int r = min(32 * rt + l32, R - 1);
  const int g = r % p.G, qi = r / p.G;
  const int hq = hk * p.G + g;
  const int64_t row = ((int64_t)b * p.Hq + hq) * p.Sq + qi;

  if (pl.bad) {
    if (32 * rt + l32 < R) {
      const float nan = __builtin_nanf("");
      T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss;
      for (int d = wave * 2 + h; d < D; d += NW * 2) out[d] = from_f32<T>(nan);
      if (wave == 0 && h == 0) a.lse[row] = nan;
    }
    return;
  }

  i32x4 qf[C::KC];
  {
    const char* src = (const char*)((const T*)a.q.data + b * a.q.sb + hq * a.q.sh + (int64_t)qi * a.q.ss) + 16 * h;
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) qf[kc] = ld_global16(src + 32 * kc);
  }

  // This row sees the cached keys [row_lo, n); the tiles that hold only keys every
  // row of the tile sees need no mask.
  const int n = pl.n;
  int row_lo = 0, full_lo = 0;
  if (p.window > 0) {
    const int depth = a.depths ? max(a.depths[(int64_t)b * p.Sq + qi], 0) : qi;
    // (n + depth - window without leaving 32 bits: depth at most the window counts)
    row_lo = max(n - (p.window - min(depth, p.window)), 0);
    full_lo = row_lo;
#pragma unroll
    for (int x = 32; x; x >>= 1) full_lo = max(full_lo, __shfl_xor(full_lo, x));
    full_lo = __builtin_amdgcn_readfirstlane(full_lo);
  }
  const unsigned char* mrow = a.mask ? a.mask + b * a.mask_sb + (int64_t)qi * p.Sq : nullptr;

  // this wave's tiles: first + NW * j, j < nt
  const int t_lo = pl.t0 + s * pl.chunk, t_hi = min(pl.t1, t_lo + pl.chunk);
  const int first = t_lo + wave;
  const int nt = __builtin_amdgcn_readfirstlane(max((t_hi - first + NW - 1) / NW, 0));

  const T* kp = (const T*)a.k.data + b * a.k.sb + hk * a.k.sh;
  const T* vp = (const T*)a.v.data + b * a.v.sb + hk * a.v.sh;
  const int last = n + p.Sq - 1;
  const unsigned wbase = lds_addr_of(smem) + wave * C::WAVEB;
  auto issue_k = [&](int t, int st) {
#pragma unroll
    for (int e = 0; e < C::E; ++e) {
      const int q = e * 64 + lane, kr = q / C::CPR, pc = q % C::CPR;
      const int64_t j = min(t * C::BN + kr, last);
      load_lds16((const char*)(kp + j * a.k.ss) + swz_col<C::CPR>(kr, pc) * 16, wbase + st * 2 * C::TB + e * 1024);
    }
  };
  auto issue_v = [&](int t, int st) {
#pragma unroll
    for (int e = 0; e < C::E; ++e) {
      const int q = e * 64 + lane, kr = q / C::CPR, pc = q % C::CPR;
      const int64_t j = min(t * C::BN + kr, last);
      load_lds16((const char*)(vp + j * a.v.ss) + swz_v<T, C::CPR>(kr, pc) * 16,
                 wbase + st * 2 * C::TB + C::TB + e * 1024);
    }
  };
  // this wave's LDS reads have returned: the buffer they read may be refilled
  auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  if (nt > 0) {
    issue_k(first, 0);
    issue_v(first, 0);
  }

  float c2 = p.scale_log2;
  if constexpr (!CAP) {  // as in the forward: a negative scale moves into Q
    if (c2 < 0.f) {
      constexpr int kSign = sizeof(T) == 4 ? (int)0x80000000 : (int)0x80008000;
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc) qf[kc] ^= i32x4{kSign, kSign, kSign, kSign};
      c2 = -c2;
    }
    if (c2 == 0.f) c2 = 1e-30f;
  }
  // wait for Q here, once: see fwd_split.hip
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) pin(qf[kc]);

  int koff[C::KC], voff[C::DB];
#pragma unroll
  for (int kc = 0; kc < C::KC; ++kc) koff[kc] = l32 * C::ROWB + swz_col<C::CPR>(l32, 2 * kc + h) * 16;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int db = 0; db < C::DB; ++db)  // row 4 h (rows 8 i + 4 h + j have its swizzle)
      voff[db] = 4 * h * C::ROWB + swz_v32<C::CPR>(4 * h, 8 * db + (l32 >> 2)) * 16 + (l32 & 3) * 4;
  } else {
    const int tr_row = 4 * h + ((lane & 15) >> 2);
    const int tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
      voff[db] = tr_row * C::ROWB + swz_tr<C::CPR>(tr_row, 4 * db + (tr_col >> 3)) * 16 + (tr_col & 7) * 2;
  }

  f32x16 acc[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x16{};
  float m_run = kNegInf, l_run = 0.f;

  for (int j = 0; j < nt; ++j) {
    const int t = first + NW * j;
    const bool more = j + 1 < nt;
    if constexpr (ST == 2) {
      if (more) {  // into the stage of tile j - 1, read in the previous iteration
        reads_done();
        issue_k(t + NW, (j + 1) & 1);
        issue_v(t + NW, (j + 1) & 1);
        wait_vmcnt<2 * C::E>();  // tile j landed, the next in flight
      } else {
        wait_vmcnt<0>();
      }
    } else {
      wait_vmcnt<C::E>();  // K of tile j landed (its V, issued later, may be in flight)
    }
    const char* sK = smem + wave * C::WAVEB + (ST == 2 ? (j & 1) * 2 * C::TB : 0);
    const char* sV = sK + C::TB;
    const int n0 = t * C::BN;

    f32x16 sc = f32x16{};
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) sc = mma_step<T>(lds_read16(sK + koff[kc]), qf[kc], sc);
    if constexpr (ST == 1) {
      reads_done();
      if (more) issue_k(t + NW, 0);
    }

    // element e is key n0 + 8(e/4) + 4h + e%4
    if constexpr (CAP) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float tv;
        if constexpr (sizeof(T) == 4) sc[e] = p.cap_log2 * tanhf(sc[e] * p.scale * p.inv_cap);
        else sc[e] = score_log2<true, false>(sc[e], p, 0.f, 0, 0, tv);
      }
    }
    if (n0 < full_lo || n0 + C::BN > n) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int jj = n0 + 8 * (e >> 2) + 4 * h + (e & 3), u = jj - n;
        bool ok;
        if (u < 0) ok = jj >= row_lo;
        else if (u >= p.Sq) ok = false;
        else ok = mrow ? mrow[u] != 0 : u <= qi;
        if (!ok) sc[e] = kNegInf;
      }
    }
    float mx, mx2;
    max16_partial(sc, mx, mx2);
    mx = max2(mx, mx2);
    if constexpr (!CAP) mx *= c2;
    mx = fmaxf(mx, swap_halves(mx));
    if (mx != mx) mx = kNegInf;
    const bool grow = mx > m_run + kTreeRescale;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float m_new = grow ? mx : m_run;
      const float alpha = grow ? fast_exp2(m_run - m_new) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < C::DB; ++db) scale_inplace(acc[db], alpha);
      m_run = m_new;
    }
    const float m_use = (m_run == kNegInf) ? 0.f : m_run;
    f32x16 pe;
    float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if constexpr (!CAP) pe[e] = fast_exp2(__builtin_fmaf(sc[e], c2, -m_use));
      else pe[e] = fast_exp2(sc[e] - m_use);
      rs[e & 3] += pe[e];
    }
    l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    if constexpr (ST == 1) {  // V of tile j landed (the next K may be in flight)
      if (more) wait_vmcnt<C::E>();
      else wait_vmcnt<0>();
    }
    if constexpr (sizeof(T) == 4) {
      // key 8 i + 4 h + j of lane half h is accumulator element 4 i + j: P is its own B operand
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const char* vr = sV + (8 * (i >> 2) + (i & 3)) * C::ROWB;
#pragma unroll
        for (int db = 0; db < C::DB; ++db) {
          const float v = *(const float*)(vr + voff[db]);
          acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, pe[i], acc[db], 0, 0, 0);
        }
      }
    } else {
      typedef typename Mfma<T>::v8 V8;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const V8 pb = pack8<T>(pe, 8 * c);
        const char* vr = sV + 16 * c * C::ROWB;
#pragma unroll
        for (int db = 0; db < C::DB; ++db) {
          const i16x4 lo = lds_read_tr4(vr + voff[db]);
          const i16x4 hi = lds_read_tr4(vr + 8 * C::ROWB + voff[db]);
          acc[db] = Mfma<T>::mma(cat_tr<V8>(lo, hi), pb, acc[db]);
        }
      }
    }
    if constexpr (ST == 1) {
      reads_done();
      if (more) issue_v(t + NW, 0);
    }
  }

  // The NW waves' (m, l, acc) combined in wave order through LDS (every wave's
  // copies have landed: its last tile waited for vmcnt 0), then O / l and LSE.
  const float l_tot = l_run + swap_halves(l_run);
  __syncthreads();
  float* xm = (float*)smem;  // [NW][64]
  float* xl = xm + NW * 64;  // [NW][64]
  float* xa = xl + NW * 64;  // [NW][DB][16][64]
  xm[wave * 64 + lane] = m_run;
  xl[wave * 64 + lane] = l_tot;
#pragma unroll
  for (int db = 0; db < C::DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) xa[((wave * C::DB + db) * 16 + e) * 64 + lane] = acc[db][e];
  __syncthreads();
  float mw[NW], mall = kNegInf;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    mw[w] = xm[w * 64 + lane];
    mall = fmaxf(mall, mw[w]);
  }
  float al[NW], L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    // a wave whose maximum stayed -inf has weights of 0, or NaN scores
    al[w] = mw[w] == kNegInf ? (xl[w * 64 + lane] == 0.f ? 0.f : 1.f) : fast_exp2(mw[w] - mall);
    L = __builtin_fmaf(al[w], xl[w * 64 + lane], L);
  }
  const bool empty = L == 0.f;  // no key; NaN (a NaN query row or key) is not
  const float inv = empty ? 0.f : 1.0f / L;
  if (32 * rt + l32 < R) {
    float* po = a.part_o + (row * a.nsplit + s) * D + 4 * h;
    T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)qi * a.o.ss + 4 * h;
    for (int x = wave; x < 4 * C::DB; x += NW) {  // 4 columns of this row per half wave
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(al[w], xa[(w * C::DB * 16 + 4 * x + j) * 64 + lane], o[j]);
      o *= inv;
      if (pl.ns > 1) *(f32x4*)(po + 8 * x) = o;
      else if constexpr (sizeof(T) == 4) *(f32x4*)(out + 8 * x) = o;
      else st_global8(out + 8 * x, pack4<T>(o[0], o[1], o[2], o[3]));
    }
    if (wave == 0 && h == 0) {
      const float lse = empty ? kNegInf : mall + log2f(L);
      if (pl.ns > 1) a.part_lse[row * a.nsplit + s] = lse;
      else a.lse[row] = lse * kLn2;
    }
  }
}

// Merge of a row's partials, one workgroup per row, four columns per thread:
// M = max LSE_s, O = sum 2^(LSE_s - M) O_s / sum 2^(LSE_s - M).  A partial without
// keys has LSE -inf and is left out; one with a NaN score makes the row NaN.
template <class T, int D>
__global__ __launch_bounds__(64) void tree_merge_kernel(TreeArgs a) {
  constexpr int TPR = D / 4;
  const Shape& p = a.p;
  const int64_t row = blockIdx.x;
  const int i = (int)(row % p.Sq);
  const int64_t bh = row / p.Sq;
  const int hq = (int)(bh % p.Hq), b = (int)(bh / p.Hq);
  const int ns = tree_plan<TreeCfg<T, D>::NW>(a, b).ns;
  if (ns == 1) return;  // (and a sequence that does not fit) written by its workgroup
  const float* pl = a.part_lse + row * a.nsplit;
  float mx = kNegInf;
  for (int s = 0; s < ns; ++s) mx = fmaxf(mx, pl[s]);
  const float m0 = mx == kNegInf ? 0.f : mx;
  float ws = 0.f;
  for (int s = 0; s < ns; ++s) ws += fast_exp2(pl[s] - m0);
  const bool none = ws == 0.f;
  const int c = threadIdx.x;
  if (c < TPR) {
    const f32x4* po = (const f32x4*)(a.part_o + row * a.nsplit * D) + c;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ns; ++s) {
      const float lw = pl[s], w = fast_exp2(lw - m0);
      const f32x4 v = po[(int64_t)s * TPR];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = lw != kNegInf ? __builtin_fmaf(w, v[j], acc[j]) : acc[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = none ? 0.f : acc[j] / ws;
    T* out = (T*)a.o.data + b * a.o.sb + hq * a.o.sh + (int64_t)i * a.o.ss + 4 * c;
    if constexpr (sizeof(T) == 4) *(f32x4*)out = acc;
    else st_global8(out, pack4<T>(acc[0], acc[1], acc[2], acc[3]));
  }
  if (c == 0) a.lse[row] = none ? kNegInf : (mx + log2f(ws)) * kLn2;
}

template <class T, int D>
hipError_t launch_tree(TreeArgs a, hipStream_t st) {
  using C = TreeCfg<T, D>;
  a.nrt = (int)(((int64_t)a.p.G * a.p.Sq + 31) / 32);
  const dim3 grid((unsigned)((int64_t)a.nsplit * a.nrt * a.p.B * a.p.Hkv)), block(C::NW * 64);
  if (a.p.cap > 0.f) hipLaunchKernelGGL((tree_attn_kernel<T, D, C::NW, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((tree_attn_kernel<T, D, C::NW, false>), grid, block, 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nsplit == 1) return e;
  hipLaunchKernelGGL((tree_merge_kernel<T, D>), dim3((unsigned)((int64_t)a.p.B * a.p.Hq * a.p.Sq)), dim3(64), 0, st, a);
  return hipGetLastError();
}

#define FLEXATT_CAT2(a, b) a##b
#define FLEXATT_CAT(a, b) FLEXATT_CAT2(a, b)
hipError_t FLEXATT_CAT(tree_attn_bf16_d, FLEXATT_D)(const TreeArgs& a, hipStream_t st) {
  return launch_tree<__bf16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(tree_attn_f16_d, FLEXATT_D)(const TreeArgs& a, hipStream_t st) {
  return launch_tree<_Float16, FLEXATT_D>(a, st);
}
hipError_t FLEXATT_CAT(tree_attn_f32_d, FLEXATT_D)(const TreeArgs& a, hipStream_t st) {
  return launch_tree<float, FLEXATT_D>(a, st);
}

}  // namespace flexatt
