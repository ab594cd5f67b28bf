// Attention of new tokens over a paged key/value cache.
//
//   o = sum_j softmax_j(cap(scale q . k_j)) v_j   over the keys j that the
//   token sees, cap(x) = softcap tanh(x / softcap) or x
//
// A token at position t sees the keys [lo, hi): hi = max(t + 1, prefix) (at
// most the sequence's length), lo = t - window + 1 with a window, else 0.
//
// The query heads of one key/value head are rows of one problem (row r is
// token r / G, head r % G of the group), so that its keys and values are read
// once for all of them.  Scores are computed transposed, S^T = K Q^T, and the
// output too, O^T = V^T P^T: a lane's scores, its statistics and its output
// columns then belong to one query row, and with the keys of a block dealt to
// the rows of the S^T tiles as below, the probabilities a lane holds are the
// ones the second product wants from it -- no exchange between the products.
#include <math.h>

#include "capi_util.h"
#include "common.h"
#include "paged.h"

namespace fvx {

constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttn {
  PagedBatch b;
  const bf16_t* q;
  int64_t ldq;
  bf16_t* o;
  int64_t ldo;
  const unsigned char* k;
  const unsigned char* v;
  const float* k_scale;
  const float* v_scale;
  const int32_t* prefix_len;
  int32_t kv_heads, group, window;
  float scale, softcap;
  int32_t* rec;  // [n_wg][8] problems that cross workgroups
  float* part;   // [n_wg][2][16 rows x (D + 2)] partials
};

// Max / sum of the four lanes l, l ^ 16, l ^ 32, l ^ 48 (one query row's
// lanes), in all of them: v_permlane16_swap, then v_permlane32_swap.
__device__ __forceinline__ void row_pair(float v, float& a, float& b) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                  false, false);
  a = __uint_as_float(s[0]);
  b = __uint_as_float(s[1]);
}
__device__ __forceinline__ float quad_max(float v) {
  float a, b;
  row_pair(v, a, b);
  return half_pair_max(fmaxf(a, b));
}
__device__ __forceinline__ float quad_sum(float v) {
  float a, b;
  row_pair(v, a, b);
  return half_pair_sum(a + b);
}

// Length of sequence b's visible cache and the interval of keys that its new
// token i (of n) sees; empty for a token before the sequence's start.
struct PagedSeq {
  int q0, n, raw, len, pre;
  __device__ __forceinline__ void load(const PagedAttn& p, int b) {
    paged_rows(p.b, b, q0, n);
    raw = p.b.kv_len[b];
    pre = p.prefix_len ? p.prefix_len[b] : 0;
    const int64_t most = (int64_t)p.b.max_pages << p.b.lg_page;
    len = raw < 0 ? 0 : (raw < most ? raw : (int)most);
  }
  __device__ __forceinline__ void keys(const PagedAttn& p, int i, int& lo, int& hi) const {
    const int64_t t = (int64_t)raw - n + i;
    if (t < 0) {
      lo = hi = 0;
      return;
    }
    const int64_t h = t + 1 > pre ? t + 1 : pre;
    hi = h < len ? (int)h : len;
    const int64_t l = p.window > 0 ? t - p.window + 1 : 0;
    lo = l < 0 ? 0 : (l < hi ? (int)l : hi);
  }
};

// ---------------------------------------------------------------------------
// Few rows per sequence: up to 16 rows a problem on 16x16x32 MFMAs
// ---------------------------------------------------------------------------
// Bound by the cache's bytes.  All (sequence, key/value head, 16 rows)
// problems form one line of units of kUnitBlocks key blocks, which is cut
// evenly over the workgroups: lengths may differ as they like, and the host
// need not know them.  A workgroup walks its piece problem by problem, its
// four waves taking the key blocks in turn; a problem that crosses workgroups
// leaves fp32 partials (rows, maxima, sums) and the merge kernel adds them in
// workgroup order.
//
// Key blocks: 32 keys of bf16, 64 of e4m3 -- 16 bytes per lane and load.  Lane
// (m = l % 16, g = l / 16) reads, for S^T tile t, key GS (m / 4) + 4 t + m % 4
// (GS = 8 or 16 keys) and, for O^T, dim m, keys GS g ... + GS - 1.  Then lane
// (row m, g)'s scores, S^T rows 4 g + j of tile t, are keys GS g + 4 t + j:
// the keys whose values the lane group g brings to O^T.  Operands go from
// memory to registers; the next block's keys are requested once S^T has used
// the current ones, its values once O^T has.
constexpr int kDecRows = 16;
constexpr int kUnitBlocks = 4;
constexpr int kPageIds = 1024;  // page ids of a walk held in LDS

template <int D, bool F8>
struct DecShape {
  static constexpr int ES = F8 ? 1 : 2;        // bytes per cache value
  static constexpr int KB = F8 ? 64 : 32;      // keys per block
  static constexpr int GS = KB / 4;            // keys per lane group
  static constexpr int NT = KB / 16;           // S^T tiles
  static constexpr int NK = D * ES / 64;       // 16-byte loads per key row
  static constexpr int NS = D / 32;            // MFMA steps over the dims
  static constexpr int ND = D / 16;            // O^T tiles
  static constexpr int PF = kDecRows * (D + 2);  // floats of a partial
};

template <int D, bool F8, bool CAP>
__global__ __launch_bounds__(256, 2) void paged_decode_kernel(PagedAttn p) {
  using S = DecShape<D, F8>;
  constexpr int LDO = D + 4;
  __shared__ __align__(16) float sO[4 * kDecRows * LDO];
  __shared__ float sM[4][kDecRows], sL[4][kDecRows];
  __shared__ int sPid[kPageIds + 4];
  __shared__ int64_t sScan[4];
  __shared__ int64_t sBase;
  __shared__ int sSeq;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int wg = blockIdx.x, n_wg = gridDim.x;
  const int lg = p.b.lg_page, G = p.group;

  // Units of sequence b: key/value heads x 16-row tiles x units of its keys
  // (one for a sequence that sees nothing: its rows are still written).
  auto seq_units = [&](int b, int& per, int& tiles) {
    PagedSeq s;
    s.load(p, b);
    tiles = (int)(((int64_t)s.n * G + kDecRows - 1) / kDecRows);
    int lo, hi, x;
    s.keys(p, 0, lo, x);
    s.keys(p, s.n - 1, x, hi);
    const int ub = S::KB * kUnitBlocks;
    per = hi > lo ? (hi + ub - 1) / ub - lo / ub : 1;
    return (int64_t)per * tiles * p.kv_heads;
  };

  // this workgroup's piece [g0, g1) of all units, and the sequence of g0
  int64_t g0, g1, total;
  int wgs;
  {
    const int each = (p.b.n_seqs + 255) / 256, first = tid * each;
    int64_t mine = 0;
    int per, tiles;
    for (int i = 0; i < each; ++i)
      if (first + i < p.b.n_seqs) mine += seq_units(first + i, per, tiles);
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    if (lane == 63) sScan[wave] = incl;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < wave) before += sScan[i];
      total += sScan[i];
    }
    wgs = total < n_wg ? (int)total : n_wg;
    if (wg >= wgs) {
      if (tid == 0) p.rec[wg * 8] = -1;
      return;
    }
    g0 = total * wg / wgs;
    g1 = total * (wg + 1) / wgs;
    int64_t at = before + incl - mine;
    if (g0 >= at && g0 < at + mine) {
      int b = first;
      for (;; ++b) {
        const int64_t u = seq_units(b, per, tiles);
        if (g0 < at + u) break;
        at += u;
      }
      sSeq = b;
      sBase = at;
    }
    __syncthreads();
  }

  int b = sSeq;
  int64_t base = sBase, at = g0;
  bool crosses = false;
  while (at < g1) {
    int per, tiles;
    const int64_t units = seq_units(b, per, tiles);
    if (at >= base + units) {
      base += units;
      ++b;
      continue;
    }
    // problem j of the sequence (key/value head fastest), its units [u0, u1)
    const int j = (int)((at - base) / per);
    const int h = j % p.kv_heads, rt = j / p.kv_heads;
    const int64_t p0 = base + (int64_t)j * per, p1 = p0 + per;
    const int u0 = (int)(at - p0), u1 = (int)((p1 < g1 ? p1 : g1) - p0);
    const bool whole = p0 >= g0 && p1 <= g1;

    PagedSeq s;
    s.load(p, b);
    const int rows = s.n * G - rt * kDecRows < kDecRows ? s.n * G - rt * kDecRows : kDecRows;
    // this lane's row, its keys, and those of the first and last row
    const int r = rt * kDecRows + (m < rows ? m : rows - 1);
    const int tok = r / G, head = h * G + r - tok * G;
    int lo, hi, lo_min, lo_max, hi_min, hi_max, seq_lo, x;
    s.keys(p, tok, lo, hi);
    s.keys(p, rt * kDecRows / G, lo_min, hi_min);
    s.keys(p, (rt * kDecRows + rows - 1) / G, lo_max, hi_max);
    s.keys(p, 0, seq_lo, x);
    constexpr int UB = S::KB * kUnitBlocks;
    const int k_first = (seq_lo / UB + u0) * UB, k_last = (seq_lo / UB + u1) * UB;
    // key blocks of this piece that some row sees
    const int kb0 = (k_first > lo_min ? k_first : lo_min) / S::KB;
    const int k_end = k_last < hi_max ? k_last : hi_max;
    const int kb1 = (k_end + S::KB - 1) / S::KB;

    bf16x8 qf[S::NS];
    {
      const bf16_t* qr = p.q + (int64_t)(s.q0 + tok) * p.ldq + (int64_t)head * D;
#pragma unroll
      for (int i = 0; i < S::NS; ++i)
        qf[i] = ld8(qr + (F8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g));
    }
    float sc = p.scale * (F8 && p.k_scale ? p.k_scale[h] : 1.f);
    // CAP: cap tanh(x / cap) = cap (1 - 2 / (exp(2 x / cap) + 1))
    sc *= CAP ? 2.f * kLog2e / p.softcap : kLog2e;
    const float cap = CAP ? p.softcap * kLog2e : 0.f;

    f32x4_t o[S::ND];
#pragma unroll
    for (int d = 0; d < S::ND; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    bf16x8 kr[S::NT][S::NK], vr[S::ND];
    int vpid = 0;
    const int kq = S::GS * (m >> 2) + (m & 3);

    constexpr int CB = kPageIds * 16 / S::KB;  // blocks per walk (pages hold 16 tokens or more)
    for (int c0 = kb0; c0 < kb1; c0 += CB) {
      const int c1 = c0 + CB < kb1 ? c0 + CB : kb1;
      const int pg0 = (int)(((int64_t)c0 * S::KB) >> lg);
      const int pg1 = (int)(((int64_t)c1 * S::KB - 1) >> lg);
      __syncthreads();
      for (int i = tid; i <= pg1 - pg0; i += 256) sPid[i] = paged_page(p.b, b, pg0 + i);
      __syncthreads();

      auto load_k = [&](int kb) {
        const int key = kb * S::KB + kq;
        const int id = sPid[(key >> lg) - pg0];
        const unsigned char* a =
            p.k + ((((int64_t)(id < 0 ? 0 : id) * p.kv_heads + h) << lg) + (key & ((1 << lg) - 1))) *
                      (D * S::ES) + 16 * g;
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
#pragma unroll
          for (int i = 0; i < S::NK; ++i)
            kr[t][i] = *(const bf16x8*)(a + t * 4 * D * S::ES + i * 64);
      };
      auto load_v = [&](int kb) {
        const int key = kb * S::KB + S::GS * g;
        vpid = sPid[(key >> lg) - pg0];
        const unsigned char* a =
            p.v + (((((int64_t)(vpid < 0 ? 0 : vpid) * p.kv_heads + h) * D + m) << lg) +
                   (key & ((1 << lg) - 1))) * S::ES;
#pragma unroll
        for (int d = 0; d < S::ND; ++d) vr[d] = *(const bf16x8*)(a + ((int64_t)(d * 16 * S::ES) << lg));
      };
      auto block = [&](int kb, auto more) {
        f32x4_t sa[S::NT];
#pragma unroll
        for (int t = 0; t < S::NT; ++t) sa[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < S::NK; ++i)
#pragma unroll
          for (int t = 0; t < S::NT; ++t) {
            if constexpr (F8) {
              sa[t] = mfma16x16x32(e4m3x8_to_bf16(kr[t][i].w[0], kr[t][i].w[1]), qf[2 * i], sa[t]);
              sa[t] = mfma16x16x32(e4m3x8_to_bf16(kr[t][i].w[2], kr[t][i].w[3]), qf[2 * i + 1], sa[t]);
            } else {
              sa[t] = mfma16x16x32(kr[t][i], qf[i], sa[t]);
            }
          }
        // (the next block's keys take the registers of this one's, not others)
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(more)::value) load_k(kb + 4);
        __builtin_amdgcn_sched_barrier(0);

        const int k0 = kb * S::KB, kg = k0 + S::GS * g;
        const bool edge = k0 < lo_max || k0 + S::KB > hi_min || __any(vpid < 0);
        float sv[4 * S::NT];
#pragma unroll
        for (int e = 0; e < 4 * S::NT; ++e) {
          float a = sa[e >> 2][e & 3] * sc;
          if (CAP) a = cap - 2.f * cap * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(a) + 1.f);
          sv[e] = a;
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 4 * S::NT; ++e)
            if (kg + e < lo || kg + e >= hi || vpid < 0) sv[e] = -INFINITY;
          // what no row sees may hold anything: 0 x infinity is not 0
          const int a = lo_min - kg, z = vpid < 0 ? 0 : hi_max - kg;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t keep = 0;
#pragma unroll
            for (int e = 0; e < 4 / S::ES; ++e) {
              const int key = w * (4 / S::ES) + e;
              if (key >= a && key < z) keep |= (F8 ? 0xffu : 0xffffu) << (8 * S::ES * e);
            }
#pragma unroll
            for (int d = 0; d < S::ND; ++d) vr[d].w[w] &= keep;
          }
        }
        float mb = sv[0];
#pragma unroll
        for (int e = 1; e < 4 * S::NT; ++e) mb = fmaxf(mb, sv[e]);
        mb = quad_max(mb);
        if (__any(mb > m_run)) {
          const float mn = fmaxf(m_run, mb);
          const float f = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - mn);
          m_run = mn;
          l_run *= f;
#pragma unroll
          for (int d = 0; d < S::ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] *= f;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run;
        // probabilities are rounded to bf16 for the product (half a step of
        // 2^-8 each, and independent over the keys); the sum takes them as
        // they are in fp32
        bf16x8 pt[S::NT / 2];
#pragma unroll
        for (int t = 0; t < S::NT / 2; ++t) {
          float pv[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pv[e] = __builtin_amdgcn_exp2f(sv[8 * t + e] - ref);
            l_run += pv[e];
          }
          pt[t] = pack8(pv);
        }
#pragma unroll
        for (int d = 0; d < S::ND; ++d) {
          if constexpr (F8) {
            o[d] = mfma16x16x32(e4m3x8_to_bf16(vr[d].w[0], vr[d].w[1]), pt[0], o[d]);
            o[d] = mfma16x16x32(e4m3x8_to_bf16(vr[d].w[2], vr[d].w[3]), pt[S::NT / 2 - 1], o[d]);
          } else {
            o[d] = mfma16x16x32(vr[d], pt[0], o[d]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(more)::value) load_v(kb + 4);
        __builtin_amdgcn_sched_barrier(0);
      };
      int kb = c0 + wave;
      if (kb < c1) {
        load_k(kb);
        load_v(kb);
        for (; kb + 4 < c1; kb += 4) block(kb, BoolC<true>{});
        block(kb, BoolC<false>{});
      }
    }

    // the four waves' rows together: weights exp2(m_w - M)
    l_run = quad_sum(l_run);
    if (g == 0) {
      sM[wave][m] = m_run;
      sL[wave][m] = l_run;
    }
    if (m < rows) {
      const float vs = F8 && p.v_scale ? p.v_scale[h] : 1.f;
      float* row = &sO[(wave * kDecRows + m) * LDO + 4 * g];
#pragma unroll
      for (int d = 0; d < S::ND; ++d) {
        f32x4_t t = o[d];
        if (F8) t = f32x4_t{t[0] * vs, t[1] * vs, t[2] * vs, t[3] * vs};
        *(f32x4_t*)(row + 16 * d) = t;
      }
    }
    __syncthreads();
    const int slot = at > g0 ? 1 : 0;
    float* part = p.part + ((int64_t)wg * 2 + slot) * S::PF;
    for (int c = tid; c < rows * (D / 4); c += 256) {
      const int i = c / (D / 4), d0 = (c % (D / 4)) * 4;
      float top = sM[0][i];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, sM[w][i]);
      f32x4_t a = f32x4_t{0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (sM[w][i] == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(sM[w][i] - top);
        const f32x4_t t = *(const f32x4_t*)&sO[(w * kDecRows + i) * LDO + d0];
        l += f * sL[w][i];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += f * t[e];
      }
      if (whole) {
        const int rr = rt * kDecRows + i, tk = rr / G;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        uint2 w2;
        w2.x = f2bf2(a[0] * inv, a[1] * inv);
        w2.y = f2bf2(a[2] * inv, a[3] * inv);
        *(uint2*)(p.o + (int64_t)(s.q0 + tk) * p.ldo + (int64_t)(h * G + rr - tk * G) * D + d0) = w2;
      } else {
        *(f32x4_t*)(part + i * D + d0) = a;
        if (d0 == 0) {
          part[kDecRows * D + i] = top;
          part[kDecRows * D + kDecRows + i] = l;
        }
      }
    }
    __syncthreads();  // the rows in LDS are read
    // a problem that starts here and ends in a later workgroup: what the
    // merge has to know
    if (p1 > g1 && p0 >= g0) {
      crosses = true;
      if (tid == 0) {
        int32_t* rec = p.rec + wg * 8;
        rec[0] = (int)((p1 * wgs - 1) / total);  // the workgroup of its last unit
        rec[1] = slot;
        rec[2] = s.q0;
        rec[3] = rt;
        rec[4] = h;
        rec[5] = rows;
      }
    }
    at = p0 + u1;
  }
  if (!crosses && tid == 0) p.rec[wg * 8] = -1;
}

// Rows blockIdx.y, + gridDim.y, ... of the problem that crosses out of
// workgroup blockIdx.x: its partials (slot rec[1] there, slot 0 in the
// workgroups after it) are added in a fixed order, a quarter (256 / (D / 4)
// groups) of them per group of threads, weighted by exp2(m_w - M).
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttn p) {
  constexpr int V = D / 4, NG = 256 / V;
  constexpr int64_t PF = kDecRows * (D + 2);
  __shared__ float sT[4];
  __shared__ __align__(16) float sA[NG][D];
  __shared__ float sW[NG];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = blockIdx.x;
  const int32_t* rec = p.rec + first * 8;
  const int last = rec[0];
  if (last < 0) return;
  const int slot = rec[1], q0 = rec[2], rt = rec[3], h = rec[4], rows = rec[5];
  const int n = last - first + 1;
  auto partial = [&](int i) {
    return p.part + ((int64_t)(first + i) * 2 + (i == 0 ? slot : 0)) * PF;
  };
  for (int i = blockIdx.y; i < rows; i += gridDim.y) {
    float top = -INFINITY;
    for (int w = tid; w < n; w += 256) top = fmaxf(top, partial(w)[kDecRows * D + i]);
    top = wave_max(top);
    __syncthreads();  // the previous row's sums are read
    if (lane == 0) sT[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sT[0], sT[1]), fmaxf(sT[2], sT[3]));
    const int v = tid % V, gr = tid / V;
    f32x4_t a = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 4
    for (int w = gr; w < n; w += NG) {
      const float* pt = partial(w);
      const float mw = pt[kDecRows * D + i];
      const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
      const f32x4_t t = *(const f32x4_t*)(pt + i * D + 4 * v);
      l += f * pt[kDecRows * D + kDecRows + i];
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += f * t[e];
    }
    *(f32x4_t*)&sA[gr][4 * v] = a;
    if (v == 0) sW[gr] = l;
    __syncthreads();
    if (tid < V) {
      float den = 0.f;
      f32x4_t t = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < NG; ++u) {
        den += sW[u];
        const f32x4_t x = *(const f32x4_t*)&sA[u][4 * tid];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += x[e];
      }
      const float inv = den > 0.f ? 1.f / den : 0.f;
      const int rr = rt * kDecRows + i, tk = rr / p.group;
      uint2 w2;
      w2.x = f2bf2(t[0] * inv, t[1] * inv);
      w2.y = f2bf2(t[2] * inv, t[3] * inv);
      *(uint2*)(p.o + (int64_t)(q0 + tk) * p.ldo +
                (int64_t)(h * p.group + rr - tk * p.group) * D + 4 * tid) = w2;
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Workgroups of the decode kernel: as many as run at once (two per CU by
// registers).
static int decode_wgs() { return 2 * device_cus(); }

static int64_t decode_ws_bytes(int64_t d, int n_wg) {
  return (int64_t)n_wg * 8 * 4 + (int64_t)n_wg * 2 * kDecRows * (d + 2) * 4;
}

template <int D>
static void launch_decode(const PagedAttn& p, bool f8, bool cap, int n_wg, unsigned ry,
                          hipStream_t s) {
  const dim3 grid((unsigned)n_wg), block(256);
  if (f8 && cap) hipLaunchKernelGGL((paged_decode_kernel<D, true, true>), grid, block, 0, s, p);
  else if (f8) hipLaunchKernelGGL((paged_decode_kernel<D, true, false>), grid, block, 0, s, p);
  else if (cap) hipLaunchKernelGGL((paged_decode_kernel<D, false, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_decode_kernel<D, false, false>), grid, block, 0, s, p);
  hipLaunchKernelGGL((paged_merge_kernel<D>), dim3((unsigned)n_wg, ry), block, 0, s, p);
}

static int check_paged_attention(const fvx_paged_attn_desc* d) {
  FVX_REQUIRE(d, FVX_ERR_NULL, "paged_attention: descriptor is NULL");
  FVX_REQUIRE(d->n_rows >= 0 && d->n_seqs >= 0 && d->max_pages >= 0, FVX_ERR_SHAPE,
              "paged_attention: n_rows, n_seqs and max_pages must not be negative");
  FVX_REQUIRE(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, FVX_ERR_SHAPE,
              "paged_attention: head_dim=%lld must be 64, 128 or 256", (long long)d->head_dim);
  FVX_REQUIRE(d->page_size >= 16 && d->page_size <= 1024 &&
                  (d->page_size & (d->page_size - 1)) == 0,
              FVX_ERR_SHAPE, "paged_attention: page_size=%lld must be a power of two, 16 to 1024",
              (long long)d->page_size);
  FVX_REQUIRE(d->kv_heads > 0 && d->q_heads > 0 && d->q_heads % d->kv_heads == 0 &&
                  d->q_heads <= 4096,
              FVX_ERR_SHAPE,
              "paged_attention: q_heads=%lld must be a positive multiple of kv_heads=%lld, at "
              "most 4096", (long long)d->q_heads, (long long)d->kv_heads);
  const int64_t big = 1ll << 30;
  FVX_REQUIRE(d->n_rows < big && d->n_rows * d->q_heads < 2 * big && d->n_seqs < big &&
                  d->n_pages > 0 && d->n_pages < 2 * big && d->max_pages < big &&
                  d->max_pages * d->page_size < big && d->window >= 0 && d->window < 2 * big,
              FVX_ERR_SHAPE,
              "paged_attention: n_rows, n_seqs and max_pages * page_size must be below 2^30, "
              "n_rows * q_heads, n_pages (> 0) and window (>= 0) below 2^31");
  FVX_REQUIRE(d->max_q >= 0, FVX_ERR_SHAPE, "paged_attention: max_q must not be negative");
  FVX_REQUIRE(d->q_start || d->n_rows == d->n_seqs, FVX_ERR_SHAPE,
              "paged_attention: without q_start n_rows (%lld) must be n_seqs (%lld)",
              (long long)d->n_rows, (long long)d->n_seqs);
  FVX_REQUIRE(d->e4m3 == 0 || d->e4m3 == 1, FVX_ERR_ARG, "paged_attention: e4m3 must be 0 or 1");
  FVX_REQUIRE(d->softcap >= 0.f && isfinite(d->softcap) && isfinite(d->scale), FVX_ERR_ARG,
              "paged_attention: scale must be finite, softcap finite and >= 0");
  return FVX_OK;
}

}  // namespace fvx

using namespace fvx;

extern "C" int64_t fvx_paged_attention_workspace_bytes(const fvx_paged_attn_desc* d) {
  clear_error();
  const int st = check_paged_attention(d);
  if (st) return st;
  if (d->n_rows == 0 || d->n_seqs == 0) return 0;
  return decode_ws_bytes(d->head_dim, decode_wgs());
}

extern "C" int fvx_paged_attention(const fvx_paged_attn_desc* d, void* stream) {
  clear_error();
  int st = check_paged_attention(d);
  if (st) return st;
  if (d->n_rows == 0 || d->n_seqs == 0) return FVX_OK;
  FVX_REQUIRE(d->q && d->o && d->k && d->v && d->kv_len && (d->page_table || d->max_pages == 0),
              FVX_ERR_NULL, "paged_attention: q, o, k, v, kv_len and page_table required");
  FVX_REQUIRE(!d->e4m3 || (d->k_scale && d->v_scale), FVX_ERR_NULL,
              "paged_attention: an e4m3 cache needs k_scale and v_scale");
  FVX_REQUIRE(aligned16(d->q) && aligned16(d->o) && aligned16(d->k) && aligned16(d->v) &&
                  aligned16(d->workspace) && d->ldq % 8 == 0 && d->ldo % 8 == 0,
              FVX_ERR_ALIGN,
              "paged_attention: q, o, k, v and workspace must be 16B aligned, ldq and ldo "
              "multiples of 8");
  FVX_REQUIRE(d->ldq >= d->q_heads * d->head_dim && d->ldo >= d->q_heads * d->head_dim &&
                  (d->table_stride >= d->max_pages || d->n_seqs == 1),
              FVX_ERR_SHAPE,
              "paged_attention: ldq and ldo must hold q_heads * head_dim values, table_stride "
              "max_pages entries");
  const int n_wg = decode_wgs();
  FVX_REQUIRE(d->workspace && d->workspace_bytes >= decode_ws_bytes(d->head_dim, n_wg),
              FVX_ERR_WORKSPACE, "paged_attention: workspace of %lld bytes required",
              (long long)decode_ws_bytes(d->head_dim, n_wg));
  PagedAttn p;
  p.b.page_table = d->page_table;
  p.b.table_stride = d->table_stride;
  p.b.kv_len = d->kv_len;
  p.b.q_start = d->q_start;
  p.b.n_rows = (int)d->n_rows;
  p.b.n_seqs = (int)d->n_seqs;
  p.b.max_pages = (int)d->max_pages;
  p.b.n_pages = (int)d->n_pages;
  p.b.lg_page = __builtin_ctzll((unsigned long long)d->page_size);
  p.q = (const bf16_t*)d->q;
  p.ldq = d->ldq;
  p.o = (bf16_t*)d->o;
  p.ldo = d->ldo;
  p.k = (const unsigned char*)d->k;
  p.v = (const unsigned char*)d->v;
  p.k_scale = d->k_scale;
  p.v_scale = d->v_scale;
  p.prefix_len = d->prefix_len;
  p.kv_heads = (int)d->kv_heads;
  p.group = (int)(d->q_heads / d->kv_heads);
  p.window = (int)d->window;
  p.scale = d->scale;
  p.softcap = d->softcap;
  p.part = (float*)d->workspace;
  p.rec = (int32_t*)(p.part + (int64_t)n_wg * 2 * kDecRows * (d->head_dim + 2));
  hipStream_t s = (hipStream_t)stream;
  const bool cap = d->softcap > 0.f;
  const int64_t most = p.group * (d->max_q > 0 ? d->max_q : 16);
  const unsigned ry = (unsigned)(most < kDecRows ? most : kDecRows);
  if (d->head_dim == 64) launch_decode<64>(p, d->e4m3 != 0, cap, n_wg, ry, s);
  else if (d->head_dim == 128) launch_decode<128>(p, d->e4m3 != 0, cap, n_wg, ry, s);
  else launch_decode<256>(p, d->e4m3 != 0, cap, n_wg, ry, s);
  return launch_status("paged_attention");
}
