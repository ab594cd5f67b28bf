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

// n / d for n < 2^31 by one multiplication
struct FastDiv {
  uint32_t d, mul, shift;
  static FastDiv of(uint32_t d) {
    FastDiv f;
    f.d = d;
    f.shift = 0;
    while ((1ull << f.shift) < d) ++f.shift;
    f.mul = (uint32_t)((((1ull << f.shift) - d) << 32) / d + 1);
    return f;
  }
  __device__ __forceinline__ int div(int n) const {
    return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
  }
};

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
  FastDiv by_group, by_kv;
  float scale, softcap;
  // few rows: sequences of at most most_rows query rows per key/value head
  int32_t most_rows;
  int32_t by_problem;  // records by problem, not by workgroup
  int32_t extra;  // units that a problem counts beside its key blocks
  int32_t* rec;  // [8 each] problems that cross workgroups
  float* part;   // [n_wg][2][16 rows x (D + 2)] partials
  // many rows: the others; problems and key ranges of the launch
  int32_t problems, splits;
  int32_t* prec;  // [problems][4]
  float* ppart;   // [problems][splits][rows x (D + 2)]
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
    raw = max(p.b.kv_len[b], 0);
    pre = p.prefix_len ? p.prefix_len[b] : 0;
    len = min(raw, p.b.max_pages << p.b.lg_page);
  }
  __device__ __forceinline__ void keys(const PagedAttn& p, int i, int& lo, int& hi) const {
    const int t = raw - n + i;  // below raw
    hi = t < 0 ? 0 : min(max(t + 1, pre), len);
    lo = clampi(p.window > 0 ? t - p.window + 1 : 0, 0, hi);
    lo = t < 0 ? 0 : lo;
  }
};

// ---------------------------------------------------------------------------
// Few rows per sequence: up to 16 rows a problem on 16x16x32 MFMAs
// ---------------------------------------------------------------------------
// Bound by the cache's bytes: 64 sequences of 1 to 8192 tokens, 32 heads on 8
// of 128 dims, 1.07 GB: 185 us + 5 of the merge, 5.6 TB/s where reading alone
// reaches 5.7; short caches by a chain of dependent loads (817 tokens: 7 us
// and 3.3).  All (sequence, key/value head, 16 rows)
// problems form one line of units, a key block each, which is cut evenly
// over the workgroups, one per CU: lengths may differ as they like, and the
// host need not know them.  A workgroup walks its piece problem by problem,
// its waves taking the key blocks in turn; a problem that crosses workgroups
// leaves fp32 partials (rows, maxima, sums) and the merge kernel adds them in
// workgroup order.  (With two workgroups of 4 waves per CU the memory serves
// the older one first: it was done at 145 us of 187 and left the other alone
// with half the loads in flight.)
//
// Key blocks: 32 keys of bf16, 64 of e4m3 -- 16 bytes per lane and load.  Lane
// (m = l % 16, g = l / 16) reads, for S^T tile t, key GS (m / 4) + 4 t + m % 4
// (GS = 8 or 16 keys) and, for O^T, dim m, keys GS g ... + GS - 1.  Then lane
// (row m, g)'s scores, S^T rows 4 g + j of tile t, are keys GS g + 4 t + j:
// the keys whose values the lane group g brings to O^T.  Operands go from
// memory to registers; the next block's keys are requested once S^T has used
// the current ones, its values once O^T has.
constexpr int kDecRows = 16;
constexpr int kWaves = 8;
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

// a / b for a >= 0, b > 0; almost always in 32 bits
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
  if ((uint64_t)(a | b) >> 32 == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// The line of units cut into `parts` pieces as even as they go: the first
// `more` of them have `each` + 1 units.
struct Pieces {
  int64_t each, more;
  __device__ __forceinline__ Pieces(int64_t total, int parts) {
    each = div64(total, parts);
    more = total - each * parts;
  }
  __device__ __forceinline__ int64_t start(int w) const {
    return w * each + (w < more ? w : more);
  }
  __device__ __forceinline__ int holder(int64_t unit) const {
    const int64_t big = more * (each + 1);
    return (int)(unit < big ? div64(unit, each + 1) : more + div64(unit - big, each));
  }
};

template <int D, bool F8, bool CAP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_decode_kernel(PagedAttn p) {
  using S = DecShape<D, F8>;
  constexpr int LDO = D + 4, NTH = 64 * kWaves;
  __shared__ __align__(16) float sO[kWaves * kDecRows * LDO];
  __shared__ float sM[kWaves][kDecRows], sL[kWaves][kDecRows];
  // head dim 256: the queries, whose registers the loads in flight need
  constexpr bool QL = D == 256;
  __shared__ __align__(16) bf16_t sQ[QL ? S::NS * 64 * 8 : 8];
  __shared__ int sPid[kPageIds + 4];
  __shared__ int64_t sScan[kWaves];
  __shared__ int64_t sBase;
  __shared__ int sSeq;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int wg = blockIdx.x, n_wg = gridDim.x;
  const int lg = p.b.lg_page, G = p.group;

  // A sequence's units: key/value heads x 16-row tiles x `per`, its key
  // blocks (one if it sees nothing: its rows are still written) after `extra`
  // units that stand for the time a problem takes to begin and end.
  struct Units {
    int per, tiles;
    int64_t all;
  };
  auto units_of = [&](const PagedSeq& s) {
    Units u;
    const int64_t rows = (int64_t)s.n * G;
    u.tiles = rows <= p.most_rows ? (int)((rows + kDecRows - 1) / kDecRows) : 0;
    int lo, hi, x;
    s.keys(p, 0, lo, x);
    s.keys(p, s.n - 1, x, hi);
    u.per = p.extra + (hi > lo ? (hi + S::KB - 1) / S::KB - lo / S::KB : 1);
    u.all = (int64_t)u.per * u.tiles * p.kv_heads;
    return u;
  };

  // this workgroup's piece [g0, g1) of all units, and the sequence of g0: up
  // to 64 sequences by every wave for itself, a lane each; more by the
  // workgroup, a run of sequences per thread
  int64_t total = 0, base = 0, g0, g1;
  int b = 0;
  PagedSeq s;
  const bool lanes = p.b.n_seqs <= 64;
  int64_t at = 0, mine = 0;
  const int each = lanes ? 1 : (p.b.n_seqs + NTH - 1) / NTH, first = (lanes ? lane : tid) * each;
  for (int i = 0; i < each; ++i)
    if (first + i < p.b.n_seqs) {
      s.load(p, first + i);
      mine += units_of(s).all;
    }
  {
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    at = incl - mine;
    total = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(incl >> 32), 63) << 32) |
                      (uint32_t)__builtin_amdgcn_readlane((int)incl, 63));
    if (!lanes) {
      if (lane == 63) sScan[wave] = incl;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        if (i < wave) at += sScan[i];
        total += sScan[i];
      }
    }
  }
  const int wgs = total < n_wg ? (int)total : n_wg;
  if (wg >= wgs) {
    if (tid == 0 && !p.by_problem) p.rec[wg * 8] = -1;
    return;
  }
  const Pieces pieces(total, wgs);
  g0 = pieces.start(wg);
  g1 = pieces.start(wg + 1);
  if (lanes) {
    b = __builtin_ctzll(__ballot(g0 >= at && g0 < at + mine));
    base = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), b) << 32) |
                     (uint32_t)__builtin_amdgcn_readlane((int)at, b));
    s.q0 = __builtin_amdgcn_readlane(s.q0, b);
    s.n = __builtin_amdgcn_readlane(s.n, b);
    s.raw = __builtin_amdgcn_readlane(s.raw, b);
    s.len = __builtin_amdgcn_readlane(s.len, b);
    s.pre = __builtin_amdgcn_readlane(s.pre, b);
  } else {
    if (g0 >= at && g0 < at + mine) {
      int c = first;
      for (;; ++c) {
        s.load(p, c);
        const int64_t n = units_of(s).all;
        if (g0 < at + n) break;
        at += n;
      }
      sSeq = c;
      sBase = at;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(sSeq);
    base = sBase;
    base = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(base >> 32)) << 32) |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)base));
    s.load(p, b);
  }
  Units u = units_of(s);
  bool starts = false, again = false;  // a problem starts here
  at = g0;
  while (at < g1) {
    if (at >= base + u.all) {
      base += u.all;
      s.load(p, ++b);
      u = units_of(s);
      continue;
    }
    // problem j of the sequence (key/value head fastest), its units [u0, u1)
    const int per = u.per;
    const int j = at - base < per ? 0 : (int)div64(at - base, per);
    const int rt = p.by_kv.div(j), h = j - rt * p.kv_heads;
    const int64_t p0 = base + (int64_t)j * per, p1 = p0 + per;
    const int u0 = (int)(at - p0), u1 = (int)((p1 < g1 ? p1 : g1) - p0);
    const bool whole = p0 >= g0 && p1 <= g1;
    starts = starts || p0 >= g0;

    const int rows = s.n * G - rt * kDecRows < kDecRows ? s.n * G - rt * kDecRows : kDecRows;
    // this lane's row, its keys, and those of the first and last row
    const int r = rt * kDecRows + (m < rows ? m : rows - 1);
    const int tok = p.by_group.div(r), head = h * G + r - tok * G;
    int lo, hi, lo_min, lo_max, hi_min, hi_max, seq_lo, x;
    s.keys(p, tok, lo, hi);
    s.keys(p, p.by_group.div(rt * kDecRows), lo_min, hi_min);
    s.keys(p, p.by_group.div(rt * kDecRows + rows - 1), lo_max, hi_max);
    s.keys(p, 0, seq_lo, x);
    auto key_of = [&](int unit) {
      return (seq_lo / S::KB + (unit > p.extra ? unit - p.extra : 0)) * S::KB;
    };
    const int k_first = key_of(u0), k_last = key_of(u1);
    // key blocks of this piece that some row sees
    const int kb0 = (k_first > lo_min ? k_first : lo_min) / S::KB;
    const int k_end = k_last < hi_max ? k_last : hi_max;
    const int kb1 = (k_end + S::KB - 1) / S::KB;

    // Q's fragment i: dims 32 i + 8 g ... of row m (e4m3: the order of the
    // keys' loads, 16 dims of a pair of fragments per lane)
    bf16x8 qf[QL ? 1 : S::NS];
    {
      const bf16_t* qr = p.q + (int64_t)(s.q0 + tok) * p.ldq + (int64_t)head * D;
      auto dim = [&](int i) { return F8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g; };
      if constexpr (QL) {
        static_assert(!QL || S::NS == kWaves, "a fragment per wave");
        qf[0] = ld8(qr + dim(wave));  // to LDS behind the page ids' loads
      } else {
#pragma unroll
        for (int i = 0; i < S::NS; ++i) qf[i] = ld8(qr + dim(i));
      }
    }
    auto q_frag = [&](int i) {
      if constexpr (QL) return ld8(&sQ[(i * 64 + lane) * 8]);
      else return qf[i];
    };
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
      if (again) __syncthreads();  // the ids before these are read
      again = true;
      for (int i = tid; i <= pg1 - pg0; i += NTH) sPid[i] = paged_page(p.b, b, pg0 + i);
      if constexpr (QL) st8(&sQ[(wave * 64 + lane) * 8], qf[0]);
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
        for (int d = 0; d < S::ND; ++d) {
          vr[d] = *(const bf16x8*)a;
          a += (uint32_t)(16 * S::ES) << lg;
        }
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
              sa[t] = mfma16x16x32(e4m3x8_to_bf16(kr[t][i].w[0], kr[t][i].w[1]), q_frag(2 * i), sa[t]);
              sa[t] = mfma16x16x32(e4m3x8_to_bf16(kr[t][i].w[2], kr[t][i].w[3]), q_frag(2 * i + 1), sa[t]);
            } else {
              sa[t] = mfma16x16x32(kr[t][i], q_frag(i), sa[t]);
            }
          }
        // (the next block's keys take the registers of this one's, not others)
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(more)::value) load_k(kb + kWaves);
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
        if constexpr (decltype(more)::value) load_v(kb + kWaves);
        __builtin_amdgcn_sched_barrier(0);
      };
      int kb = c0 + wave;
      if (kb < c1) {  // (all of it in one branch: exact waits for the loads)
        load_k(kb);
        load_v(kb);
        for (; kb + kWaves < c1; kb += kWaves) block(kb, BoolC<true>{});
        block(kb, BoolC<false>{});
      }
    }

    // the waves' rows together: weights exp2(m_w - M)
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
    for (int c = tid; c < rows * (D / 4); c += NTH) {
      const int i = c / (D / 4), d0 = (c % (D / 4)) * 4;
      float mw[kWaves], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, mw[w] = sM[w][i]);
      f32x4_t a = f32x4_t{0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        // (a wave without keys holds zeros)
        const float f = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[w] - top);
        const f32x4_t t = *(const f32x4_t*)&sO[(w * kDecRows + i) * LDO + d0];
        l += f * sL[w][i];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += f * t[e];
      }
      if (whole) {
        const int rr = rt * kDecRows + i, tk = p.by_group.div(rr);
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
    if (p0 >= g0 && tid == 0) {
      int32_t* rec = p.rec + (p.by_problem ? (b * u.tiles + rt) * p.kv_heads + h : wg) * 8;
      if (p1 > g1) {
        rec[0] = pieces.holder(p1 - 1) - wg + 1;  // workgroups
        rec[1] = slot;
        rec[2] = s.q0;
        rec[3] = rt;
        rec[4] = h;
        rec[5] = rows;
        rec[6] = wg;
      } else {
        rec[0] = -1;
      }
    }
    at = p0 + u1;
  }
  if (!p.by_problem && !starts && tid == 0) p.rec[wg * 8] = -1;
}

// Rows blockIdx.y, + gridDim.y, ... of the problem of record blockIdx.x, if it
// crosses workgroups: its partials (slot rec[1] of workgroup rec[6], slot 0 of
// the ones after it) weighted by exp2(m_w - M), and added by NT / (D / 4)
// groups of threads, then over the groups, in a fixed order.
template <int D, int NT>
__global__ __launch_bounds__(NT) void paged_merge_kernel(PagedAttn p) {
  constexpr int V = D / 4, NG = NT / V;
  constexpr int64_t PF = kDecRows * (D + 2);
  __shared__ float sT[NT / 64];
  __shared__ __align__(16) float sA[NG][D];
  __shared__ float sW[NG];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* rec = p.rec + (int64_t)blockIdx.x * 8;
  const int n = rec[0];
  if (n < 0) return;
  const int slot = rec[1], q0 = rec[2], rt = rec[3], h = rec[4], rows = rec[5], first = rec[6];
  auto partial = [&](int i) {
    return p.part + ((int64_t)(first + i) * 2 + (i == 0 ? slot : 0)) * PF;
  };
  for (int i = blockIdx.y; i < rows; i += gridDim.y) {
    float top = -INFINITY;
    for (int w = tid; w < n; w += NT) top = fmaxf(top, partial(w)[kDecRows * D + i]);
    top = wave_max(top);
    __syncthreads();  // the previous row's sums are read
    if (lane == 0) sT[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) top = fmaxf(top, sT[w]);
    const int v = tid % V, gr = tid / V;
    f32x4_t a = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 8
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
      const int groups = n < NG ? n : NG;
      float den = 0.f;
      f32x4_t t = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int u = 0; u < groups; ++u) {
        den += sW[u];
        const f32x4_t x = *(const f32x4_t*)&sA[u][4 * tid];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += x[e];
      }
      const float inv = den > 0.f ? 1.f / den : 0.f;
      const int rr = rt * kDecRows + i, tk = p.by_group.div(rr);
      uint2 w2;
      w2.x = f2bf2(t[0] * inv, t[1] * inv);
      w2.y = f2bf2(t[2] * inv, t[3] * inv);
      *(uint2*)(p.o + (int64_t)(q0 + tk) * p.ldo +
                (int64_t)(h * p.group + rr - tk * p.group) * D + 4 * tid) = w2;
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows per sequence: 32x32x16 MFMAs, keys and values through LDS
// ---------------------------------------------------------------------------
// Bound by what a SIMD issues: products, the exponentials and their packing
// (four prompts of 4000 tokens, causal: 880 TFLOP/s at 128 dims, 765 at 256,
// 730 at 64, where a large matrix product reaches 1390; with capped scores,
// three transcendentals each, 740, 710 and 550).  A workgroup owns 128 query
// rows of one key/value head, a wave 32 of them, and walks the keys they see
// (or one of `splits` ranges of them) in tiles of 64.  (64 rows per wave: 851
// for 880, and 655 for 740 capped.)  As many workgroups share a CU as
// registers allow: their waves are each other's cover.  Tiles arrive in LDS
// by DMA, one barrier per tile, keys one tile ahead of values.  A wave
// goes on in halves of 32 keys, three of which are in work at once: the
// scores of half h + 1 and the output of half h - 1 are on the matrix cores
// while the exponentials of half h are taken.
//
// Scores refer to a row's reference, its running maximum when that last rose
// by more than kSlack above it: probabilities stay below 2^kSlack, and the
// output is rescaled a few times per row, not once per tile.
constexpr int kProTile = 64;
// Page ids in LDS: two runs of kProRun tiles (of at most 4 pages each), the
// second of which is refilled while the first is walked.
constexpr int kProRun = 128;
constexpr int kProPages = 2 * kProRun * kProTile / 16;
constexpr float kSlack = 8.f;

// 16 bytes per lane straight into LDS (lane l's at m0 + OFF + 16 l), from
// 64-bit addresses or from a uniform base and 32-bit offsets (+ OFF); waited
// for with wait_vmcnt, like load_lds16.
__device__ __forceinline__ void load_lds16_at(const void* a, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(a)
               : "memory");
}
template <int OFF>
__device__ __forceinline__ void load_lds16_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3"
               :
               : "s"(lds), "v"(off), "s"(base), "n"(OFF)
               : "memory");
}

// max(a, b, c), without the compiler's quieting of each
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// l + the two bf16 values of w, as the second product reads them.
__device__ __forceinline__ float add_pair(uint32_t w, float l) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w),
                                         __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l, false);
}

// The products with their operands where the kernel wants them: scores in
// vector registers, which the exponentials read; output and queries in
// accumulation registers, which nothing else reads in the common path.  (The
// compiler by itself copies scores or output from one file to the other in
// every half.)  It does not know when these products finish: what reads their results must come 20 wait
// states or more behind the last one (mfma_settle).  NOP: the operand of the
// vector registers is just computed, which needs two wait states.
template <bool FIRST, bool NOP>
__device__ __forceinline__ void mfma_scores(f32x16_t& d, const bf16x8& k, const bf16x8& q) {
  const i32x4_t a = __builtin_bit_cast(i32x4_t, k), c = __builtin_bit_cast(i32x4_t, q);
  if constexpr (FIRST && NOP)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(c));
  else if constexpr (FIRST)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(c));
  else if constexpr (NOP)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "a"(c));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "a"(c));
}

template <bool NOP>
__device__ __forceinline__ void mfma_output(f32x16_t& d, const bf16x8& v, const bf16x8& pr) {
  const i32x4_t a = __builtin_bit_cast(i32x4_t, v), c = __builtin_bit_cast(i32x4_t, pr);
  if constexpr (NOP)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(d) : "v"(a), "v"(c));
  else
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(d) : "v"(a), "v"(c));
}
__device__ __forceinline__ void mfma_settle() { asm volatile("s_nop 15\n\ts_nop 15"); }

template <int D, bool F8>
struct ProShape {
  static constexpr int BM = 128;                // rows per workgroup
  // workgroups per CU that registers and LDS allow
  static constexpr int WGS = D == 256 ? 1 : (D == 128 ? 2 : 3);
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int KROW = D * ES;           // bytes of a key in LDS
  static constexpr int VROW = kProTile * ES;    // bytes of a dim in LDS
  static constexpr int TB = kProTile * D * ES;  // bytes of a tile of keys (of values)
  static constexpr int NDB = D / 32;            // output blocks
  static constexpr int NS = D / 16;             // MFMA steps of a score
  static constexpr int PF = BM * (D + 2);       // floats of a partial

  // Products of a half: JA steps of the output, the scores' NC, the rest of
  // the output's NO.  Their operand fragments come from LDS in that order,
  // through a ring of registers, read kAhead fragments before their product.
  // An output step is (block pair, step u, block); e4m3 fragments hold both
  // steps u of a block, or two steps of the scores.
  static constexpr int NVR = F8 ? NDB : 2 * NDB;  // fragments of values
  static constexpr int NKR = F8 ? NS / 2 : NS;    // fragments of keys
  static constexpr int NO = 2 * NDB, NC = NS, JA = NO / 2;
  static constexpr int NVA = F8 && D == 64 ? NVR : NVR / 2;  // values' that the first JA use
  static constexpr int kRing = D == 64 ? 4 : 8, kAhead = D == 64 ? 3 : 6;
  // the output's fragment of its step j
  static constexpr int out_frag(int j) {
    return F8 ? 2 * (j >> 2) + (j & 1) : j;
  }
  // the fragment, in reading order, of step j of a half
  static constexpr int frag_at(int j) {
    if (j >= JA && j < JA + NC) return NVA + (j - JA) / (F8 ? 2 : 1);
    const int r = out_frag(j < JA ? j : j - NC);
    return r < NVA ? r : r + NKR;
  }
  // fragments read by the start of step j's product
  static constexpr int frags_to(int j) {
    int m = 0;
    for (int i = 0; i <= j; ++i) m = frag_at(i) + 1 > m ? frag_at(i) + 1 : m;
    return m;
  }
};

// 16-byte slot of logical chunk c of LDS row `row` (RB bytes long): rows that
// lanes read together lie in different banks.
template <int RB>
__device__ __forceinline__ int swz(int row, int c) {
  constexpr int RP = RB >= 256 ? 1 : 256 / RB, M = RB / 16 < 16 ? RB / 16 - 1 : 15;
  return c ^ ((row / RP) & M);
}

// Problem `item` of the launch: the tiles of BM rows of the sequences with
// more than most_rows rows, key/value head fastest, a sequence's last tile
// (which sees most keys) first.  Returns false past the last one.
template <int BM>
__device__ bool find_tile(const PagedAttn& p, int item, int* scan, int* found, int& b, int& t,
                          int& h) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // up to 64 sequences: every wave by itself, a lane each; more: a run of
  // sequences per thread
  const bool lanes = p.b.n_seqs <= 64;
  const int each = lanes ? 1 : (p.b.n_seqs + 255) / 256, first = (lanes ? lane : tid) * each;
  auto tiles = [&](int s) {
    int q0, n;
    paged_rows(p.b, s, q0, n);
    const int64_t rows = (int64_t)n * p.group;
    return rows > p.most_rows ? (int)((rows + BM - 1) / BM) : 0;
  };
  // Starts that run backwards make sequences overlap: sums that saturate keep
  // every problem of the launch in the one run [at, incl) that holds it.
  int mine = 0;
  for (int i = 0; i < each; ++i)
    if (first + i < p.b.n_seqs) mine = __builtin_elementwise_add_sat(mine, tiles(first + i));
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl = __builtin_elementwise_add_sat(incl, v);
  }
  int at = __shfl_up(incl, 1, 64), total = __builtin_amdgcn_readlane(incl, 63);
  if (lane == 0) at = 0;
  if (!lanes) {
    if (lane == 63) scan[wave] = incl;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < wave) {
        at = __builtin_elementwise_add_sat(at, scan[i]);
        incl = __builtin_elementwise_add_sat(incl, scan[i]);
      }
      total = __builtin_elementwise_add_sat(total, scan[i]);
    }
  }
  const int want = p.by_kv.div(item);
  h = item - want * p.kv_heads;
  if (want >= total) return false;
  const bool here = want >= at && want < incl;
  if (lanes) {
    b = __builtin_ctzll(__ballot(here));
    t = __builtin_amdgcn_readlane(mine - 1 - (want - at), b);
    return true;
  }
  if (here) {
    int s = first, n;
    for (;; ++s) {
      n = tiles(s);
      if (want - at < n) break;
      at += n;
    }
    found[0] = s;
    found[1] = n - 1 - (want - at);
  }
  __syncthreads();
  b = __builtin_amdgcn_readfirstlane(found[0]);
  t = __builtin_amdgcn_readfirstlane(found[1]);
  return true;
}

template <int D, bool F8, bool CAP>
__global__ __launch_bounds__(256, (ProShape<D, F8>::WGS)) void paged_prompt_kernel(PagedAttn p) {
  using S = ProShape<D, F8>;
  __shared__ __align__(16) unsigned char smem[4 * S::TB];
  __shared__ int sPid[kProPages];
  __shared__ int sScan[4], sFound[2], sMissing;

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 31, hh = lane >> 5;
  const int prob = blockIdx.x, split = blockIdx.y;
  const int lg = p.b.lg_page, G = p.group;
  int b, rt, h;
  if (!find_tile<S::BM>(p, prob, sScan, sFound, b, rt, h)) {
    if (split == 0 && tid == 0 && p.splits > 1) p.prec[prob * 4] = -1;
    return;
  }
  PagedSeq s;
  s.load(p, b);
  const int all = s.n * G;
  const int r_tile = rt * S::BM, rows = all - r_tile < S::BM ? all - r_tile : S::BM;
  int lo_min, lo_tile, hi_tile, hi_max;
  s.keys(p, p.by_group.div(r_tile), lo_min, hi_tile);
  s.keys(p, p.by_group.div(r_tile + rows - 1), lo_tile, hi_max);
  // tiles of this key range
  int t0 = lo_min / kProTile, t1 = (hi_max + kProTile - 1) / kProTile;
  if (t1 < t0) t1 = t0;
  {
    const int64_t n = t1 - t0;
    t1 = t0 + (int)(n * (split + 1) / p.splits);
    t0 = t0 + (int)(n * split / p.splits);
  }

  // this wave's rows: those past the tile's last repeat it and store nothing
  const int r_wave = r_tile + 32 * w;
  const bool active = 32 * w < rows;
  const int row = 32 * w + qi;  // of the tile
  const int r = r_tile + (row < rows ? row : rows - 1);
  const int tok = p.by_group.div(r), head = h * G + r - tok * G;
  int lo, hi;
  s.keys(p, tok, lo, hi);
  bf16x8 qf[S::NS];
  // a negative scale turns the queries' signs (exact), a zero one clears
  // them: the scores' maximum can then be taken before scaling
  const float ks = F8 ? p.k_scale[h] : 1.f;
  const float raw = p.scale * ks;
  const float sc = (raw == 0.f ? 1.f : fabsf(raw)) * (CAP ? 2.f / p.softcap : 1.f) * kLog2e;
  const float cap = CAP ? p.softcap * kLog2e : 0.f;
  {
    const bf16_t* qr = p.q + (int64_t)(s.q0 + tok) * p.ldq + (int64_t)head * D;
#pragma unroll
    for (int x = 0; x < S::NS; ++x) {
      qf[x] = ld8(qr + (F8 ? 32 * (x >> 1) + 16 * hh + 8 * (x & 1) : 16 * x + 8 * hh));
      if (raw <= 0.f)
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[x].w[e] = raw == 0.f ? 0u : qf[x].w[e] ^ 0x80008000u;
    }
  }
  // into accumulation registers here, two wait states or more before a product
#pragma unroll
  for (int x = 0; x < S::NS; ++x) {
    i32x4_t v = __builtin_bit_cast(i32x4_t, qf[x]);
    asm volatile("" : "+a"(v));
    qf[x] = __builtin_bit_cast(bf16x8, v);
  }
  asm volatile("s_nop 1");
  // the wave's rows all see keys [lo_max, hi_min)
  int lo_max = lo_tile, hi_min = hi_tile;
  if (active) {
    int x;
    const int last = min(r_wave + 31, r_tile + rows - 1);
    s.keys(p, p.by_group.div(r_wave), x, hi_min);
    s.keys(p, p.by_group.div(last), lo_max, x);
  }

  // O^T, the scores of a tile's halves (sa[half]) and their probabilities
  f32x16_t o[S::NDB], sa[2];
  bf16x8 pt[2][2];
  float ref = -INFINITY, l_run = 0.f;
#pragma unroll
  for (int db = 0; db < S::NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;

  // DMA: a wave brings 16 keys and D / 4 dims of a tile, LPW instructions of
  // 1 KiB each: RPK keys or RPV dims.  Its keys share a page.  A tile's
  // values share one when pages hold a tile or more; otherwise a lane's keys
  // do, at a place in the page that is the same in every tile.
  constexpr int LPW = S::TB / 1024 / 4;
  constexpr int CK = S::KROW / 16, CV = S::VROW / 16, RPK = 64 / CK, RPV = 64 / CV;
  constexpr int NV = LPW > 1 && !F8 ? 2 : 1;  // key chunks that differ over i
  const uint32_t lds = lds_addr(smem) + 1024 * LPW * w;
  const int mask = (1 << lg) - 1;
  const bool big_page = (1 << lg) >= kProTile;
  const uint32_t page_bytes = ((uint32_t)p.kv_heads * D * S::ES) << lg;  // at most 2^31
  const unsigned char* k_head = p.k + (((int64_t)h * D * S::ES) << lg);
  const unsigned char* v_head = p.v + (((int64_t)h * D * S::ES) << lg);
  uint32_t koff[LPW];
#pragma unroll
  for (int i = 0; i < LPW; ++i)
    koff[i] = (lane / CK) * S::KROW + 16 * swz<S::KROW>(16 * w + RPK * i + lane / CK, lane % CK) +
              1024 * (i & ~3);
  int vchunk[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) vchunk[i] = swz<S::VROW>(RPV * (LPW * w + i) + lane / CV, lane % CV);
  const uint32_t vrow = ((uint32_t)(RPV * LPW * w + lane / CV) * S::ES) << lg;

  // the page of a token, -1 for none
  auto page_of = [&](int key) { return sPid[(key >> lg) & (kProPages - 1)]; };
  // ids of the pages of tiles [ta, ta + kProRun), by all threads
  auto fill_ids = [&](int ta) {
    const int first = (ta * kProTile) >> lg, n = (kProRun * kProTile) >> lg;
    for (int i = tid; i < n; i += 256) {
      const int id = paged_page(p.b, b, first + i);
      sPid[(first + i) & (kProPages - 1)] = id;
      if (id < 0 && (int64_t)(first + i) << lg < hi_max) sMissing = 1;
    }
  };
  bool missing = false;  // has a page so far not existed?
  struct Ids {
    int k, v[NV], none;
  };
  // page ids for load_k(tk) and load_v(tv), ahead of them
  auto fetch_ids = [&](int tk, int tv) {
    Ids d;
    d.k = page_of(tk * kProTile + 16 * w);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      d.v[i] = page_of(tv * kProTile + (big_page ? 0 : vchunk[i] * (16 / S::ES)));
    d.none = sMissing;
    return d;
  };
  auto load_k = [&](int t, const Ids& d) {
    const uint32_t id = __builtin_amdgcn_readfirstlane(d.k < 0 ? 0 : d.k);
    const unsigned char* at =
        k_head + (uint64_t)id * page_bytes + ((t * kProTile + 16 * w) & mask) * S::KROW;
    const uint32_t to = lds + (t & 1) * S::TB;
    static_for<0, LPW>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      load_lds16_at<1024 * (i & 3)>(at, koff[i], to + 1024 * (i & ~3));
    });
  };
  auto load_v = [&](int t, const Ids& d) {
    const uint32_t to = lds + (2 + (t & 1)) * S::TB;
    if (big_page) {
      const uint32_t id = __builtin_amdgcn_readfirstlane(d.v[0] < 0 ? 0 : d.v[0]);
      const unsigned char* at = v_head + (uint64_t)id * page_bytes + ((t * kProTile) & mask) * S::ES;
#pragma unroll
      for (int i = 0; i < LPW; ++i)
        load_lds16_at<0>(at + (((uint32_t)i * RPV * S::ES) << lg), vrow + 16 * vchunk[i % NV],
                         to + 1024 * i);
    } else {
      const unsigned char* at[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i)
        at[i] = v_head + (uint64_t)(uint32_t)(d.v[i] < 0 ? 0 : d.v[i]) * page_bytes + vrow +
                ((vchunk[i] * (16 / S::ES)) & mask) * S::ES;
#pragma unroll
      for (int i = 0; i < LPW; ++i)
        load_lds16_at(at[i % NV] + (((uint32_t)i * RPV * S::ES) << lg), to + 1024 * i);
    }
  };
  // values that no row of the tile sees (unwritten slots, missing pages) may
  // be anything: they are cleared in LDS, by the wave that loaded them
  auto clear_v = [&](int t) {
    if (t * kProTile >= lo_min && (t + 1) * kProTile <= hi_max && !missing) return;
#pragma unroll 1
    for (int i = 0; i < LPW; ++i) {
      const int c = 64 * (LPW * w + i) + lane, d = c / CV;
      const int key = t * kProTile + swz<S::VROW>(d, c % CV) * (16 / S::ES);
      const bool gone = page_of(key) < 0;
      bf16x8* x = (bf16x8*)(smem + (2 + (t & 1)) * S::TB + 16 * c);
      bf16x8 v = *x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t keep = 0;
#pragma unroll
        for (int y = 0; y < 4 / S::ES; ++y) {
          const int k = key + e * (4 / S::ES) + y;
          if (k >= lo_min && k < hi_max && !gone) keep |= (F8 ? 0xffu : 0xffffu) << (8 * S::ES * y);
        }
        v.w[e] &= keep;
      }
      *x = v;
    }
  };

  constexpr int NVR = S::NVR, NKR = S::NKR, NVA = S::NVA, NO = S::NO, NC = S::NC, JA = S::JA;
  constexpr int kRing = S::kRing, kAhead = S::kAhead;
  const int kperm = F8 ? 16 * ((qi >> 2) & 1) + 8 * (qi >> 4) + 4 * ((qi >> 3) & 1) + (qi & 3)
                       : 16 * (qi >> 4) + 8 * ((qi >> 2) & 1) + 4 * ((qi >> 3) & 1) + (qi & 3);
  auto read_k = [&](int t, int hf, int x) {
    const int row = 32 * hf + kperm;
    return *(const bf16x8*)(smem + (t & 1) * S::TB + row * S::KROW +
                            16 * swz<S::KROW>(row, 2 * x + hh));
  };
  auto read_v = [&](int t, int hf, int r) {
    const int d = 32 * (F8 ? r : 2 * (r >> 2) + (r & 1)) + qi;
    const int ch = F8 ? 2 * hf + hh : 4 * hf + 2 * ((r >> 1) & 1) + hh;
    return *(const bf16x8*)(smem + (2 + (t & 1)) * S::TB + d * S::VROW + 16 * swz<S::VROW>(d, ch));
  };
  auto out_step = [&](auto jc, const bf16x8& f, const bf16x8* pr) {
    constexpr int j = decltype(jc)::value;
    constexpr int u = (j >> 1) & 1, db = 2 * (j >> 2) + (j & 1);
    if constexpr (F8)
      mfma_output<true>(o[db], e4m3x8_to_bf16(f.w[2 * u], f.w[2 * u + 1]), pr[u]);
    else
      mfma_output<false>(o[db], f, pr[u]);
  };
  auto score_step = [&](auto jc, const bf16x8& f, f32x16_t& d) {
    constexpr int x = decltype(jc)::value;
    if constexpr (F8)
      mfma_scores<x == 0, true>(d, e4m3x8_to_bf16(f.w[2 * (x & 1)], f.w[2 * (x & 1) + 1]), qf[x]);
    else
      mfma_scores<x == 0, false>(d, f, qf[x]);
  };
  auto capped = [&](float x) {  // in exponents of 2, of a score
    return cap - 2.f * cap * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * sc) + 1.f);
  };
  // key of element e of a half's scores, from the half's first
  auto key_at = [&](int e) { return F8 ? 16 * hh + e : 16 * (e >> 3) + 8 * hh + (e & 7); };

  // Half hf of tile t: its scores are in sa[hf].  Output of the half before
  // (probabilities pt[hf ^ 1], which also enter the row sums here) and scores
  // of the next one (to sa[hf ^ 1]).  The first JA products run over the
  // maximum of the scores, the others over the exponentials.
  auto half = [&](int t, auto hfc) {
    constexpr int hf = decltype(hfc)::value;
    f32x16_t& sv = sa[hf];
    f32x16_t& sn = sa[hf ^ 1];
    bf16x8* pr = pt[hf ^ 1];
    const int tv = hf ? t : t - 1, tk = hf ? t + 1 : t;
    bf16x8 ring[kRing];
    auto read = [&](auto rc) {
      constexpr int r = decltype(rc)::value;
      if constexpr (r < NVA) ring[r % kRing] = read_v(tv, hf ^ 1, r);
      else if constexpr (r < NVA + NKR) ring[r % kRing] = read_k(tk, hf ^ 1, r - NVA);
      else if constexpr (r < NVR + NKR) ring[r % kRing] = read_v(tv, hf ^ 1, r - NKR);
    };
    static_for<0, kAhead>([&](auto rc) { read(rc); });

    const int k0 = t * kProTile + 32 * hf;
    const bool edge = k0 < lo_max || k0 + 32 > hi_min || missing;
    // keys of this lane that exist, bit e
    auto there = [&] {
      uint32_t m = 0xffffu;
      if (missing) {
        m = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) m |= (page_of(k0 + key_at(e)) < 0 ? 0u : 1u) << e;
      }
      return m;
    };
    if (edge) {
      const uint32_t ok = there();
      const uint32_t span = (uint32_t)(hi - lo), at = (uint32_t)(k0 - lo);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool in = (at + (uint32_t)key_at(e) < span) & ((ok >> e & 1) != 0);
        sv[e] = in ? sv[e] : -INFINITY;
      }
    }

    constexpr int JB = NO - JA + NC;
    float mx;
    static_for<0, JA>([&](auto jc) {
      constexpr int j = decltype(jc)::value;
      static_for<j ? kAhead + S::frags_to(j - 1) : kAhead, kAhead + S::frags_to(j)>([&](auto rc) { read(rc); });
      out_step(jc, ring[S::frag_at(j) % kRing], pr);
      static_for<8 * j / JA, 8 * (j + 1) / JA>([&](auto qc) {
        constexpr int q = decltype(qc)::value, e = 2 * q;
        mx = max3(q == 0 ? sv[0] : mx, sv[e], sv[e + 1]);
        l_run = add_pair(pr[q >> 2].w[q & 3], l_run);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    mx = half_pair_max(mx);
    if (mx != -INFINITY) mx = CAP ? capped(mx) : mx * sc;
    if (__any(mx > ref + kSlack)) {
      // the probabilities not yet in the output follow it to the new
      // reference (a second rounding to bf16, on the halves where it rises)
      mfma_settle();
      const float nr = fmaxf(ref, mx);
      const float f = ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - nr);
      ref = nr;
      l_run *= f;
#pragma unroll
      for (int db = 0; db < S::NDB; ++db) {
        asm volatile("" : "+a"(o[db]));  // not copied before it is settled
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= f;
        asm volatile("" : "+a"(o[db]));  // and back before the paths join
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[8];
        unpack8(pr[u], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f;
        pr[u] = pack8(x);
      }
    }
    // the wave that has its maximum goes first: the SIMD's other one is then
    // between its products (capped scores, e4m3: 692 -> 647 us)
    __builtin_amdgcn_s_setprio(1);
    const float nm = (CAP ? cap : 0.f) - (ref == -INFINITY ? 0.f : ref);
    float even = 0.f;
    static_for<0, JB>([&](auto jc) {
      constexpr int j = JA + decltype(jc)::value, jb = decltype(jc)::value;
      static_for<kAhead + S::frags_to(j - 1), kAhead + S::frags_to(j)>([&](auto rc) { read(rc); });
      const bf16x8& f = ring[S::frag_at(j) % kRing];
      if constexpr (jb < NC) score_step(IntC<jb>{}, f, sn);
      else out_step(IntC<j - NC>{}, f, pr);
      static_for<16 * jb / JB, 16 * (jb + 1) / JB>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        const float x = sv[e];
        float pv;
        if constexpr (CAP) {
          const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * sc) + 1.f);
          pv = __builtin_amdgcn_exp2f(fmaf(-2.f * cap, r, nm));
        } else {
          pv = __builtin_amdgcn_exp2f(fmaf(x, sc, nm));
        }
        if constexpr (e % 2 == 0) {
          even = pv;
        } else {
          uint32_t w2 = f2bf2(even, pv);
          asm volatile("" : "+v"(w2));  // here, under the products, not behind them
          pt[hf][e >> 3].w[(e & 7) >> 1] = w2;
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
    // (a capped score of minus infinity is minus the cap)
    if (CAP && edge) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        pt[hf][e >> 3].w[(e & 7) >> 1] &=
            sv[e] == -INFINITY ? (e & 1 ? 0xffffu : 0xffff0000u) : 0xffffffffu;
    }
  };

  if (t0 < t1) {
    // runs begin at whole runs, and so at whole pages (of up to 1024 tokens)
    const int run0 = t0 & ~(kProRun - 1);
    if (tid == 0) sMissing = 0;
    __syncthreads();
    fill_ids(run0);
    if (t1 > run0 + kProRun) fill_ids(run0 + kProRun);
    // the first half's "previous" values: zeros (with zero probabilities)
    for (int i = tid; i < S::TB / 16; i += 256)
      *(bf16x8*)(smem + (2 + ((t0 + 1) & 1)) * S::TB + 16 * i) = zero8();
    pt[1][0] = pt[1][1] = zero8();
    __syncthreads();
    {
      const Ids d = fetch_ids(t0, t0);
      load_k(t0, d);
      load_v(t0, d);
    }
    wait_vmcnt<LPW>();
    __syncthreads();  // everyone's first keys
    {
      const Ids d = fetch_ids(t0 + 1, t0);
      missing = __builtin_amdgcn_readfirstlane(d.none) != 0;
      if (t0 + 1 < t1) load_k(t0 + 1, d);
    }

    // what a wave does at the turn of tile t: everyone's keys of tile t + 1
    // and values of tile t are there behind the barrier, and the keys of tile
    // t and the values of tile t - 1 have been used
    auto turn = [&](int t, const Ids& d) {
      wait_vmcnt<0>();
      clear_v(t);
      if ((t & (kProRun - 1)) == 2 && t - 2 > run0 && t - 2 + kProRun < t1)
        fill_ids(t - 2 + kProRun);
      // (a run's pages are looked up a hundred tiles before they are used)
      missing = __builtin_amdgcn_readfirstlane(d.none) != 0;
      __syncthreads();
      if (t + 2 < t1) load_k(t + 2, d);
      if (t + 1 < t1) load_v(t + 1, d);
    };
    if (!active) {  // no rows: this wave only loads
      for (int t = t0; t < t1; ++t) {
        turn(t, fetch_ids(t + 2, t + 1));
      }
    } else {
      static_for<0, NC>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        score_step(jc, read_k(t0, 0, j / (F8 ? 2 : 1)), sa[0]);
      });
      mfma_settle();
      for (int t = t0; t < t1; ++t) {
        const Ids d = fetch_ids(t + 2, t + 1);
        half(t, IntC<0>{});
        turn(t, d);
        half(t, IntC<1>{});
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) l_run = add_pair(pt[1][e >> 2].w[e & 3], l_run);
      static_for<0, NO>([&](auto jc) {
        out_step(jc, read_v(t1 - 1, 1, S::out_frag(decltype(jc)::value)), pt[1]);
      });
      mfma_settle();
    }
  }

  if (!active && p.splits == 1) return;
  const float vs = F8 ? p.v_scale[h] : 1.f;
  float* part = p.ppart + ((int64_t)prob * p.splits + split) * S::PF;
  if (p.splits > 1 && split == 0 && tid == 0) {
    p.prec[prob * 4] = rows;
    p.prec[prob * 4 + 1] = s.q0;
    p.prec[prob * 4 + 2] = r_tile;
    p.prec[prob * 4 + 3] = h;
  }
  const float l = half_pair_sum(l_run);
#pragma unroll
  for (int db = 0; db < S::NDB; ++db) asm volatile("" : "+a"(o[db]));
  if (row >= rows) return;
  if (p.splits == 1) {
    const float inv = l > 0.f ? vs / l : 0.f;
    bf16_t* out = p.o + (int64_t)(s.q0 + tok) * p.ldo + (int64_t)head * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < S::NDB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint2 v;
        v.x = f2bf2(o[db][4 * j] * inv, o[db][4 * j + 1] * inv);
        v.y = f2bf2(o[db][4 * j + 2] * inv, o[db][4 * j + 3] * inv);
        *(uint2*)(out + 32 * db + 8 * j) = v;
      }
    return;
  }
  float* out = part + row * D + 4 * hh;
#pragma unroll
  for (int db = 0; db < S::NDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *(f32x4_t*)(out + 32 * db + 8 * j) = f32x4_t{o[db][4 * j] * vs, o[db][4 * j + 1] * vs,
                                                   o[db][4 * j + 2] * vs, o[db][4 * j + 3] * vs};
  if (hh == 0) {
    part[S::BM * D + row] = ref;
    part[S::BM * D + S::BM + row] = l;
  }
}

// The key ranges of a problem together: rows blockIdx.y * 256 / D ... of
// problem blockIdx.x, four dims per thread, a quarter of the ranges for each
// of four groups of threads, which are then added in a fixed order.
template <int D>
__global__ __launch_bounds__(256) void paged_prompt_merge_kernel(PagedAttn p) {
  using S = ProShape<D, false>;
  constexpr int V = D / 4, NR = 64 / V;  // threads of a row, rows per group
  __shared__ __align__(16) float sA[4][NR][D];
  __shared__ float sT[4][NR], sW[4][NR];
  const int prob = blockIdx.x, rows = p.prec[prob * 4];
  const int gr = threadIdx.x / 64, ir = threadIdx.x % 64 / V, d0 = threadIdx.x % V * 4;
  if ((int)blockIdx.y * NR >= rows) return;
  const int i = blockIdx.y * NR + ir;
  const int q0 = p.prec[prob * 4 + 1], r_tile = p.prec[prob * 4 + 2], h = p.prec[prob * 4 + 3];
  const float* part = p.ppart + (int64_t)prob * p.splits * S::PF;
  float top = -INFINITY, l = 0.f;
  f32x4_t a = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (i < rows) {
#pragma unroll 4
    for (int k = gr; k < p.splits; k += 4) {
      const float* x = part + (int64_t)k * S::PF;
      const float m = x[S::BM * D + i], w = x[S::BM * D + S::BM + i];
      const f32x4_t t = *(const f32x4_t*)(x + i * D + d0);
      const float nt = fmaxf(top, m);
      const float fo = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - nt);
      const float fn = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - nt);
      top = nt;
      l = l * fo + fn * w;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = a[e] * fo + fn * t[e];
    }
  }
  *(f32x4_t*)&sA[gr][ir][d0] = a;
  if (d0 == 0) {
    sT[gr][ir] = top;
    sW[gr][ir] = l;
  }
  __syncthreads();
  if (gr || i >= rows) return;
  top = fmaxf(fmaxf(sT[0][ir], sT[1][ir]), fmaxf(sT[2][ir], sT[3][ir]));
  l = 0.f;
  a = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float f = sT[u][ir] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sT[u][ir] - top);
    const f32x4_t t = *(const f32x4_t*)&sA[u][ir][d0];
    l += f * sW[u][ir];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] += f * t[e];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int r = r_tile + i, tk = p.by_group.div(r);
  uint2 v;
  v.x = f2bf2(a[0] * inv, a[1] * inv);
  v.y = f2bf2(a[2] * inv, a[3] * inv);
  *(uint2*)(p.o + (int64_t)(q0 + tk) * p.ldo + (int64_t)(h * p.group + r - tk * p.group) * D + d0) = v;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Workgroups of the decode kernel: one per CU.
static int decode_wgs() { return device_cus(); }

// Which kernels a call launches, their grids and their parts of the
// workspace.  The host knows the number of rows and sequences and, as a hint,
// the most rows of one sequence, not who has how many.
struct PagedPlan {
  bool few, many;          // kernels launched
  int most_rows;           // query rows up to which a sequence is the few kernel's
  int n_wg;                // few: workgroups
  int64_t problems;        // many: upper bound of the problems
  int splits;
  int64_t rec, part, prec, ppart, bytes;  // workspace offsets
};

static PagedPlan paged_plan(const fvx_paged_attn_desc* d) {
  PagedPlan a = {};
  const int64_t G = d->q_heads / d->kv_heads;
  const int64_t most = d->q_start ? d->max_q : 1;
  // Up to 16 rows are one tile of the few kernel, which would read keys again
  // for each further one (20 to 64 rows, per sequence 1000 to 4000 keys: 1.2
  // to 2.7 times the many kernel's time throughout; 16 sequences of 40 rows
  // of 256 dims: 36 us and 25; one of 20 rows of 64 dims: 27 and 16).
  a.many = most == 0 || most * G > kDecRows;
  // every sequence has most rows: none is left to the few kernel
  a.few = !a.many || most == 0 || d->n_rows != d->n_seqs * most;
  a.most_rows = !a.many ? 0x7fffffff : (a.few ? kDecRows : 0);
  a.n_wg = a.few ? decode_wgs() : 0;
  a.rec = 0;
  a.part = (int64_t)a.n_wg * 32;
  a.prec = a.part + (int64_t)a.n_wg * 2 * kDecRows * (d->head_dim + 2) * 4;
  a.ppart = a.bytes = a.prec;
  if (a.many) {
    constexpr int64_t bm = ProShape<64, false>::BM;  // of any
    a.problems = (d->n_rows * G / bm + (d->n_seqs < d->n_rows ? d->n_seqs : d->n_rows)) * d->kv_heads;
    // With fewer problems than workgroups that run at once their keys are
    // split.  Each range costs the merge a partial, and saves the walk of the
    // others a share of the T tiles of 64 keys that the tables can hold: both
    // are even at a number of ranges like sqrt(T), 4 sqrt(T) by measurement.
    // One sequence, 5 tokens of 8 heads of 256 dims (32, 64, 128 ranges):
    // 4000 keys 18.9, 19.3, 19.1 us; 16000 31.2, 25.3, 24.2; 64000 76.0,
    // 48.3, 35.6; 16 of 16 heads of 64 dims: 14.0, 15.3, 15.6; 20.0, 18.3,
    // 22.1; 45.3, 30.2, 27.1.  (Tables may hold more than the lengths use:
    // 128 at most.)  Fewer ranges than run at once are slower: 16 sequences
    // of 40 rows of 256 dims 26.8 us, 32.2 with half as many; one of 816
    // tokens of 8 heads 33.8 and 38.0.
    const int64_t at_once =
        device_cus() * (d->head_dim == 256 ? ProShape<256, false>::WGS
                                           : (d->head_dim == 128 ? ProShape<128, false>::WGS
                                                                 : ProShape<64, false>::WGS));
    const int64_t tiles = (d->max_pages * d->page_size + 63) / 64;
    int64_t s = at_once / a.problems;
    s = s < 128 ? s : 128;
    while (s > 1 && s * s > 16 * tiles) --s;
    s = s < tiles ? s : tiles;
    a.splits = s < 1 ? 1 : (int)s;
    if (a.splits > 1) {
      a.ppart = a.prec + (a.problems * 16 + 15) / 16 * 16;
      a.bytes = a.ppart + a.problems * a.splits * bm * (d->head_dim + 2) * 4;
    }
  }
  return a;
}

template <int D>
static void launch_many(const PagedAttn& p, bool f8, bool cap, hipStream_t s) {
  const dim3 grid((unsigned)p.problems, (unsigned)p.splits), block(256);
  if (f8 && cap) hipLaunchKernelGGL((paged_prompt_kernel<D, true, true>), grid, block, 0, s, p);
  else if (f8) hipLaunchKernelGGL((paged_prompt_kernel<D, true, false>), grid, block, 0, s, p);
  else if (cap) hipLaunchKernelGGL((paged_prompt_kernel<D, false, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_prompt_kernel<D, false, false>), grid, block, 0, s, p);
  if (p.splits > 1)
    hipLaunchKernelGGL((paged_prompt_merge_kernel<D>),
                       dim3((unsigned)p.problems, ProShape<D, false>::BM * D / 256), block, 0, s, p);
}

template <int D>
static void launch_few(const PagedAttn& p, bool f8, bool cap, int n_wg, unsigned ry,
                       hipStream_t s) {
  const dim3 grid((unsigned)n_wg), block(64 * kWaves);
  if (f8 && cap) hipLaunchKernelGGL((paged_decode_kernel<D, true, true>), grid, block, 0, s, p);
  else if (f8) hipLaunchKernelGGL((paged_decode_kernel<D, true, false>), grid, block, 0, s, p);
  else if (cap) hipLaunchKernelGGL((paged_decode_kernel<D, false, true>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_decode_kernel<D, false, false>), grid, block, 0, s, p);
  // Few problems: long lines of partials, more threads for each (256 partials
  // of 8 x 256: 8.2 us with 1024 threads, 29 with 256; two partials of 4 x
  // 128, 512 times: 9.1 and 4.7).
  const int64_t tiles = (p.group + kDecRows - 1) / kDecRows;
  const dim3 merge(p.by_problem ? (unsigned)(p.b.n_seqs * tiles * p.kv_heads) : (unsigned)n_wg, ry);
  if ((int64_t)p.b.n_seqs * p.kv_heads * 8 < n_wg)
    hipLaunchKernelGGL((paged_merge_kernel<D, 1024>), merge, dim3(1024), 0, s, p);
  else
    hipLaunchKernelGGL((paged_merge_kernel<D, 256>), merge, dim3(256), 0, s, p);
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
              "paged_attention: scale and softcap must be finite, softcap >= 0");
  // cap(x) is formed as softcap (1 - 2 / (exp(2 x / softcap) + 1)), which
  // costs a score 3 * 2^-24 softcap: 2e-4 at most
  FVX_REQUIRE(d->softcap <= 1024.f, FVX_ERR_ARG, "paged_attention: softcap=%g must be at most 1024",
              (double)d->softcap);
  const float per_cap = d->softcap > 0.f ? 2.f * kLog2e / d->softcap : 0.f;
  FVX_REQUIRE(isfinite(per_cap) && isfinite(per_cap * d->scale), FVX_ERR_ARG,
              "paged_attention: softcap=%g is too small for scale=%g", (double)d->softcap,
              (double)d->scale);
  return FVX_OK;
}

}  // namespace fvx

using namespace fvx;

extern "C" int64_t fvx_paged_attention_workspace_bytes(const fvx_paged_attn_desc* d) {
  clear_error();
  const int st = check_paged_attention(d);
  if (st) return st;
  if (d->n_rows == 0 || d->n_seqs == 0) return 0;
  return paged_plan(d).bytes;
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
  const PagedPlan plan = paged_plan(d);
  FVX_REQUIRE(plan.problems < 1ll << 24, FVX_ERR_SHAPE,
              "paged_attention: (n_rows * q_heads / kv_heads / 128 + n_seqs) * kv_heads must be "
              "below 2^24");
  FVX_REQUIRE(plan.bytes == 0 || (d->workspace && d->workspace_bytes >= plan.bytes),
              FVX_ERR_WORKSPACE,
              "paged_attention: workspace of %lld bytes required", (long long)plan.bytes);
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
  p.by_group = FastDiv::of((uint32_t)p.group);
  p.by_kv = FastDiv::of((uint32_t)p.kv_heads);
  p.window = (int)d->window;
  p.scale = d->scale;
  p.softcap = d->softcap;
  char* ws = (char*)d->workspace;
  // With a problem or more per workgroup short ones lie behind each other:
  // each counts 128 KiB more, which is what a CU reads while one begins and
  // ends (about 5 us; 64 sequences of 1 to 8192 tokens, 8 heads of 128 dims:
  // 209 us without, 191 with).
  p.extra = d->n_seqs * d->kv_heads >= plan.n_wg
                ? (int)((128 << 10) / (2 * d->head_dim * 64)) : 0;
  p.most_rows = plan.most_rows;
  // one row per sequence: the problems are known; fewer than workgroups, each
  // has its record
  p.by_problem = !d->q_start && d->n_seqs * ((p.group + kDecRows - 1) / kDecRows) * d->kv_heads < plan.n_wg;
  p.rec = (int32_t*)(ws + plan.rec);
  p.part = (float*)(ws + plan.part);
  p.problems = (int)plan.problems;
  p.splits = plan.splits;
  p.prec = (int32_t*)(ws + plan.prec);
  p.ppart = (float*)(ws + plan.ppart);
  hipStream_t s = (hipStream_t)stream;
  const bool cap = d->softcap > 0.f;
  const int64_t most = (d->q_start ? d->max_q : 1) * p.group;
  const unsigned ry = (unsigned)(most > 0 && most < kDecRows ? most : kDecRows);
#define FVX_PAGED(D)                                                        \
  do {                                                                      \
    if (plan.many) launch_many<D>(p, d->e4m3 != 0, cap, s);                 \
    if (plan.few) launch_few<D>(p, d->e4m3 != 0, cap, plan.n_wg, ry, s);    \
  } while (0)
  if (d->head_dim == 64) FVX_PAGED(64);
  else if (d->head_dim == 128) FVX_PAGED(128);
  else FVX_PAGED(256);
#undef FVX_PAGED
  return launch_status("paged_attention");
}
