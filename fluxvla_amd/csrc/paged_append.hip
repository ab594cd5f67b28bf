// New tokens into a paged key/value cache: queries and keys rotated to their
// positions, keys and values written into their pages.
//
// Bound by bytes: each Q|K|V value is read once and written once (20800 rows
// of 32 + 8 + 8 heads of 128 dims, 361 MB with e4m3 pages: 85 us, 4.2 TB/s of
// the 5.1 that a large copy reaches); a few rows by the chain of loads from
// the row to its sequence, its length, its page (1 row: 3 us).  One
// workgroup takes RB consecutive rows of HB query and key heads, or of one
// value head.  Its first Q|K|V loads do not depend
// on where the rows go and are issued first; meanwhile one wave finds the
// rows' sequences and pages.  The rows' rotations are read once for all its
// heads (fp32 rotations weigh twice a head's bf16 values).  Rotations are two
// products and a sum per value, each rounded to fp32 (no fused multiply-add),
// then one rounding to bf16 or e4m3: the value does not depend on how the
// compiler contracts.  Values are turned in LDS: up to eight tokens of one
// dim are one store of the transposed page.
#include "capi_util.h"
#include "common.h"
#include "paged.h"

namespace fvx {

struct PagedAppend {
  PagedBatch b;
  const bf16_t* qkv;
  int64_t ld_qkv;
  bf16_t* q_out;
  int64_t ld_q;
  unsigned char* k;
  unsigned char* v;
  const float* k_scale;
  const float* v_scale;
  const float* rope;
  int64_t max_pos;
  const int32_t* positions;
  int32_t q_heads, kv_heads;
};

// e4m3 of x, rounded to nearest even, at most 448 in magnitude (NaN stays
// NaN), two values per instruction.
__device__ __forceinline__ float e4m3_sat(float x) {
  x = x > 448.f ? 448.f : x;
  return x < -448.f ? -448.f : x;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_sat(a), e4m3_sat(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_sat(c), e4m3_sat(d), r, true);
}

// Four pairs (a, b) turned by (cos, sin): (a c - b s, b c + a s), every
// operation rounded to fp32.
__device__ __forceinline__ void rotate8(const float* f, const float* cs, float* w) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    w[e] = f[e] * cs[e] - f[e + 1] * cs[e + 1];
    w[e + 1] = f[e + 1] * cs[e] + f[e] * cs[e + 1];
  }
}

constexpr int kEndsLds = 1024;  // sequence ends held in LDS for the search

// RB rows; blockIdx.y: groups of HB query and key heads, then value heads.
template <int D, bool F8, int RB, int HB>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend p) {
  constexpr int V = D / 8, RP = 256 / V;        // vectors of a row, rows per pass
  constexpr int NP = RB > RP ? RB / RP : 1;     // passes
  constexpr int LD = D + 2;
  constexpr int ES = F8 ? 1 : 2;
  __shared__ int sEnd[kEndsLds];
  __shared__ int sPos[RB], sPage[RB], sSlot[RB], sLead[RB], sCount[RB];
  __shared__ int sLeads;
  __shared__ __align__(16) bf16_t sV[RB * LD];

  const int tid = threadIdx.x, c = tid % V, i0 = tid / V;
  const int64_t r0 = (int64_t)blockIdx.x * RB;
  const int turned = p.q_heads + p.kv_heads, groups = (turned + HB - 1) / HB;
  const bool is_v = (int)blockIdx.y >= groups;
  const int y0 = is_v ? turned + (int)blockIdx.y - groups : (int)blockIdx.y * HB;
  const int y1 = is_v ? y0 + 1 : (y0 + HB < turned ? y0 + HB : turned);

  bf16x8 x[NP];
  auto load = [&](int y) {
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int i = i0 + RP * u;
      x[u] = i < RB && r0 + i < p.b.n_rows
                 ? ld8(p.qkv + (r0 + i) * p.ld_qkv + (int64_t)y * D + 8 * c)
                 : zero8();
    }
  };
  load(y0);

  const bool lds_ends = p.b.q_start && p.b.n_seqs <= kEndsLds;
  if (lds_ends) {
    for (int i = tid; i < p.b.n_seqs; i += 256) sEnd[i] = p.b.q_start[i + 1];
    __syncthreads();
  }
  if (tid < 64) {
    const int64_t row = r0 + tid;
    int pos = -1, page = -1, slot = 0, seq = -1;
    if (tid < RB && row < p.b.n_rows) {
      seq = (int)row;
      if (p.b.q_start) {  // the first sequence that ends behind the row
        int lo = 0, hi = p.b.n_seqs;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if ((lds_ends ? sEnd[mid] : p.b.q_start[mid + 1]) > row) hi = mid;
          else lo = mid + 1;
        }
        seq = lo;
      }
      int q0 = 0, n = 0;
      if (seq < p.b.n_seqs) paged_rows(p.b, seq, q0, n);
      if (row >= q0 && row < (int64_t)q0 + n) {
        const int64_t t = (int64_t)p.b.kv_len[seq] - n + (row - q0);
        const int64_t at = p.positions ? p.positions[row] : t;
        if (at >= 0 && at < p.max_pos) {
          pos = (int)at;
          if (t >= 0) page = paged_page(p.b, seq, (int)(t >> p.b.lg_page));
          slot = (int)(t & ((1 << p.b.lg_page) - 1));
        }
      }
    }
    if (tid < RB) {
      sPos[tid] = pos;
      sPage[tid] = page;
      sSlot[tid] = slot;
    }
    // runs of rows that share eight slots of a page: their first rows
    const int pseq = __shfl_up(seq, 1, 64), ppage = __shfl_up(page, 1, 64);
    const bool lead = page >= 0 && (tid == 0 || ppage != page || pseq != seq || slot % 8 == 0);
    const uint64_t leads = __ballot(lead), stops = leads | __ballot(page < 0);
    if (lead) {
      const uint64_t after = tid == 63 ? 0 : stops >> (tid + 1);
      const int run = after ? __builtin_ctzll(after) + 1 : 64 - tid;
      const int at = __builtin_popcountll(leads & ((1ull << tid) - 1));
      sLead[at] = tid;
      sCount[at] = run < 8 ? run : 8;
    }
    if (tid == 0) sLeads = __builtin_popcountll(leads);
  }
  __syncthreads();

  if (!is_v) {
    float cs[NP][8];
    int pos[NP], page[NP], slot[NP];
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int i = i0 + RP * u;
      pos[u] = i < RB ? sPos[i] : -1;
      page[u] = i < RB ? sPage[i] : -1;
      slot[u] = i < RB ? sSlot[i] : 0;
      const float* rp = p.rope + (int64_t)(pos[u] < 0 ? 0 : pos[u]) * D + 8 * c;
      f32x4_t a = f32x4_t{0.f, 0.f, 0.f, 0.f}, b = a;
      if (pos[u] >= 0) {
        a = *(const f32x4_t*)rp;
        b = *(const f32x4_t*)(rp + 4);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cs[u][e] = a[e];
        cs[u][4 + e] = b[e];
      }
    }
    for (int y = y0; y < y1; ++y) {
      const bool is_q = y < p.q_heads;
      const int h = is_q ? y : y - p.q_heads;
      const float ks = F8 && !is_q ? p.k_scale[h] : 1.f;
      bf16x8 now[NP];
#pragma unroll
      for (int u = 0; u < NP; ++u) now[u] = x[u];
      if (y + 1 < y1) load(y + 1);
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        if (pos[u] < 0 || (!is_q && page[u] < 0)) continue;
        float f[8], w[8];
        unpack8(now[u], f);
        rotate8(f, cs[u], w);
        if (is_q) {
          if (p.q_out) st8(p.q_out + (r0 + i0 + RP * u) * p.ld_q + (int64_t)h * D + 8 * c, pack8(w));
          continue;
        }
        unsigned char* a =
            p.k + ((((((int64_t)page[u] * p.kv_heads + h) << p.b.lg_page) + slot[u]) * D) + 8 * c) * ES;
        if constexpr (F8) {
          uint2 o;
          o.x = e4m3x4(w[0] / ks, w[1] / ks, w[2] / ks, w[3] / ks);
          o.y = e4m3x4(w[4] / ks, w[5] / ks, w[6] / ks, w[7] / ks);
          *(uint2*)a = o;
        } else {
          st8((bf16_t*)a, pack8(w));
        }
      }
    }
    return;
  }
  const int h = y0 - turned;
#pragma unroll
  for (int u = 0; u < NP; ++u) {
    const int i = i0 + RP * u;
    if (i >= RB) continue;
#pragma unroll
    for (int w = 0; w < 4; ++w) *(uint32_t*)&sV[i * LD + 8 * c + 2 * w] = x[u].w[w];
  }
  __syncthreads();
  const float vs = F8 ? p.v_scale[h] : 1.f;
  const int nl = sLeads;
  for (int e = tid; e < nl * D; e += 256) {
    const int d = e / nl, l = e - d * nl;  // neighbours: one dim's runs of tokens
    const int i = sLead[l], n = sCount[l], slot = sSlot[i];
    unsigned char* a =
        p.v + (((((int64_t)sPage[i] * p.kv_heads + h) * D + d) << p.b.lg_page) + slot) * ES;
    if (n == 8) {
      bf16_t t[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) t[w] = sV[(i + w) * LD + d];
      if constexpr (F8) {
        uint2 o;
        o.x = e4m3x4(bf2f(t[0]) / vs, bf2f(t[1]) / vs, bf2f(t[2]) / vs, bf2f(t[3]) / vs);
        o.y = e4m3x4(bf2f(t[4]) / vs, bf2f(t[5]) / vs, bf2f(t[6]) / vs, bf2f(t[7]) / vs);
        *(uint2*)a = o;
      } else {
        bf16x8 o;
#pragma unroll
        for (int w = 0; w < 4; ++w) o.w[w] = (uint32_t)t[2 * w] | ((uint32_t)t[2 * w + 1] << 16);
        st8((bf16_t*)a, o);
      }
    } else {
      for (int w = 0; w < n; ++w) {
        const bf16_t t = sV[(i + w) * LD + d];
        if constexpr (F8) a[w] = (unsigned char)e4m3x4(bf2f(t) / vs, 0.f, 0.f, 0.f);
        else ((bf16_t*)a)[w] = t;
      }
    }
  }
}

template <int D, bool F8, int RB, int HB>
static void launch_append_rows(const PagedAppend& p, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)p.b.n_rows + RB - 1) / RB),
                  (unsigned)((p.q_heads + p.kv_heads + HB - 1) / HB + p.kv_heads));
  hipLaunchKernelGGL((paged_append_kernel<D, F8, RB, HB>), grid, dim3(256), 0, s, p);
}

template <int D>
static void launch_append(const PagedAppend& p, bool f8, bool small, hipStream_t s) {
  if (f8 && small) launch_append_rows<D, true, 8, 1>(p, s);
  else if (f8) launch_append_rows<D, true, 32, 8>(p, s);
  else if (small) launch_append_rows<D, false, 8, 1>(p, s);
  else launch_append_rows<D, false, 32, 8>(p, s);
}

}  // namespace fvx

using namespace fvx;

extern "C" int fvx_paged_append(const fvx_paged_append_desc* d, void* stream) {
  clear_error();
  FVX_REQUIRE(d, FVX_ERR_NULL, "paged_append: descriptor is NULL");
  FVX_REQUIRE(d->n_rows >= 0 && d->n_seqs >= 0 && d->max_pages >= 0 && d->max_pos >= 0,
              FVX_ERR_SHAPE,
              "paged_append: n_rows, n_seqs, max_pages and max_pos must not be negative");
  FVX_REQUIRE(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, FVX_ERR_SHAPE,
              "paged_append: head_dim=%lld must be 64, 128 or 256", (long long)d->head_dim);
  FVX_REQUIRE(d->page_size >= 16 && d->page_size <= 1024 &&
                  (d->page_size & (d->page_size - 1)) == 0,
              FVX_ERR_SHAPE, "paged_append: page_size=%lld must be a power of two, 16 to 1024",
              (long long)d->page_size);
  FVX_REQUIRE(d->kv_heads > 0 && d->q_heads >= 0 && d->q_heads + 2 * d->kv_heads <= 16384,
              FVX_ERR_SHAPE,
              "paged_append: kv_heads (> 0) and q_heads (>= 0) out of range: %lld, %lld",
              (long long)d->kv_heads, (long long)d->q_heads);
  const int64_t big = 1ll << 30;
  FVX_REQUIRE(d->n_rows < big / 16 && d->n_seqs < big && d->n_pages > 0 && d->n_pages < 2 * big &&
                  d->max_pages < big && d->max_pages * d->page_size < big && d->max_pos < 2 * big,
              FVX_ERR_SHAPE,
              "paged_append: n_rows must be below 2^26, n_seqs and max_pages * page_size below "
              "2^30, n_pages (> 0) and max_pos below 2^31");
  FVX_REQUIRE(d->q_start || d->n_rows == d->n_seqs, FVX_ERR_SHAPE,
              "paged_append: without q_start n_rows (%lld) must be n_seqs (%lld)",
              (long long)d->n_rows, (long long)d->n_seqs);
  FVX_REQUIRE(d->e4m3 == 0 || d->e4m3 == 1, FVX_ERR_ARG, "paged_append: e4m3 must be 0 or 1");
  if (d->n_rows == 0 || d->n_seqs == 0) return FVX_OK;
  FVX_REQUIRE(d->qkv && d->k && d->v && d->rope && d->kv_len &&
                  (d->page_table || d->max_pages == 0),
              FVX_ERR_NULL, "paged_append: qkv, k, v, rope, kv_len and page_table required");
  FVX_REQUIRE(!d->e4m3 || (d->k_scale && d->v_scale), FVX_ERR_NULL,
              "paged_append: an e4m3 cache needs k_scale and v_scale");
  FVX_REQUIRE(aligned16(d->qkv) && aligned16(d->q_out) && aligned16(d->k) && aligned16(d->v) &&
                  aligned16(d->rope) && d->ld_qkv % 8 == 0 && d->ld_q % 8 == 0,
              FVX_ERR_ALIGN,
              "paged_append: qkv, q_out, k, v and rope must be 16B aligned, ld_qkv and ld_q "
              "multiples of 8");
  const int heads = (int)(d->q_heads + 2 * d->kv_heads);
  FVX_REQUIRE(d->ld_qkv >= heads * d->head_dim &&
                  (!d->q_out || d->ld_q >= d->q_heads * d->head_dim) &&
                  (d->table_stride >= d->max_pages || d->n_seqs == 1),
              FVX_ERR_SHAPE,
              "paged_append: ld_qkv and ld_q must hold their heads' values, table_stride "
              "max_pages entries");
  PagedAppend p;
  p.b.page_table = d->page_table;
  p.b.table_stride = d->table_stride;
  p.b.kv_len = d->kv_len;
  p.b.q_start = d->q_start;
  p.b.n_rows = (int)d->n_rows;
  p.b.n_seqs = (int)d->n_seqs;
  p.b.max_pages = (int)d->max_pages;
  p.b.n_pages = (int)d->n_pages;
  p.b.lg_page = __builtin_ctzll((unsigned long long)d->page_size);
  p.qkv = (const bf16_t*)d->qkv;
  p.ld_qkv = d->ld_qkv;
  p.q_out = (bf16_t*)d->q_out;
  p.ld_q = d->ld_q;
  p.k = (unsigned char*)d->k;
  p.v = (unsigned char*)d->v;
  p.k_scale = d->k_scale;
  p.v_scale = d->v_scale;
  p.rope = d->rope;
  p.max_pos = d->max_pos;
  p.positions = d->positions;
  p.q_heads = (int)d->q_heads;
  p.kv_heads = (int)d->kv_heads;
  hipStream_t s = (hipStream_t)stream;
  // Few rows, or one per sequence (scattered value stores, one per token and
  // dim): 8 rows of one head per workgroup, else 32 rows of eight.  150 to 300
  // rows of 48 heads of 128 dims: 10.2 us small, 12.6 large; 4900 rows of 10
  // heads of 256: 17.0 and 14.1; 4900 of 48 of 128: 60 and 28.
  const bool small = !d->q_start || d->n_rows * heads < 32 * 4 * 256;
  if (d->head_dim == 64) launch_append<64>(p, d->e4m3 != 0, small, s);
  else if (d->head_dim == 128) launch_append<128>(p, d->e4m3 != 0, small, s);
  else launch_append<256>(p, d->e4m3 != 0, small, s);
  return launch_status("paged_append");
}
