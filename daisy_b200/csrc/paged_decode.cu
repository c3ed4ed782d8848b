// One new token of every sequence against a paged cache: the work of a batch of uneven lengths dealt out in equal shares, one launch.
//
// Bound by HBM: 512 bytes for every cached row and key head, read once for all query heads of the group (from card to card 64 sequences x 4096
// rows x 16 heads 319-350 us, 6.1-6.7 TB/s, the least where the same rows are read again and L2 still holds some; 1 x 131071 x 16 164-177; 24 of
// up to 16384 rows, 32 query heads over 8, 133-144; 1 x 511 rows x 6 8.7-9.2, four of them the chain length -> page -> rows and the join).  The cached rows
// of all (sequence, key head) pairs lie end to end in blocks of four 16-row tiles; every CTA takes an equal run of blocks, whatever sequences it
// cuts, so neither uneven lengths nor a wide block table leaves an SM idle (the host knows no lengths).  A pair that
// several CTAs share is joined by the last of them, from partial sums in a fixed order: the same bits every run.  That last one,
// or the only one, also prepares the token's own row, adds it and stores it.
//
// A warp takes a tile straight from memory into the operands of mma.m16n8k16 (keys or channels are the 16, query heads the 8; every lane
// loads whole 16-byte pieces, the order of channels in a product is free): scores S^T = K Q^T, then O^T += V^T P^T.  On CUDA cores
// the same work is 22 instructions for 16 bytes and lane, a third of the SM's issue slots for one query head and over all of them for
// four.  Queries and weights go in as sums of two 16-bit values (two products each): scores and weights keep 16 bits and more, weights of float16
// pages down to 2^-16 of the largest, below that 2^-32 of it (WEIGHT_ROOM).
#include "paged.cuh"

//
// FEW: a few queries of every sequence instead of one (drafted tokens), prepared, their keys and values in the pages already; the
// columns of a product are then (query, head) pairs, 8 a pass, each with its own last key.
namespace daisy {

constexpr int PD_WARPS = 4;
constexpr int PD_TILE = 16;
constexpr float PD_NEG = -1.0e30f;

struct PagedDecodeParams {
  PagedCache c;
  const __nv_bfloat16 *q, *k, *v, *ve;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, ve_sb, ve_sh, o_sb, o_sh;
  __nv_bfloat16* out;
  const int *lens, *cu;
  const float *cos, *sin, *ve_gate;
  int window, table_rows, Hq, G;     // G query heads of one key head; columns (heads, or queries x heads) come in up to n_grp groups of 8 NT
  int n_grp;
  int T;                             // FEW: queries of a sequence, or of the packed row; q_st, o_st: from query to query
  int64_t q_st, o_st;
  float qscale, eps;
  unsigned flags;
  int* status;
  float* part;                       // [2 grid][8 NT][PD_PART]: 128 sums, reference, denominator
  int *tickets, *tickets_grp;        // [n_seq H n_grp], [2 grid], zero between calls
};
constexpr int PD_PART = 132;
// What a pair costs beside its rows (queries, sums of the warps, the token's own row, output), in blocks of 64 rows: the deal counts it
// as so many blocks without rows in front of the pair's.
constexpr int PD_HEAD = 2;
// FEW: columns (queries x heads of a key head) that one pass over the rows serves, and the most of a packed call: four passes where one
// sequence has them all.  8 sequences of 9000 rows x 16 heads: 4 queries 97 us here, 121 on tcgen05 (paged_prefill.cu); 16 queries in one
// pass of 16 columns 139, 121 there.
constexpr int PD_FEW = 8, PD_FEW_PACKED = 32;
constexpr int PD_JOIN = 16;          // shares that one CTA joins
constexpr __host__ __device__ int pd_ctas(int cols) { return cols == 8 ? 3 : 2; }              // CTAs a SM, by registers

// Where a sequence stands: its cached length, or -1 if it is idle or cannot have the position; rows lo .. len-1 are seen by some query.
// blocks: PD_HEAD, then one for every PD_WARPS tiles, the last one maybe short.  FEW: n queries from row row0 of q, the first at position pos0.
struct SeqRange { int len, lo, tile0, tiles, blocks, n, row0, pos0; };
struct SeqIndex { int len, first, end; };                            // as the index arrays say; FEW: its queries first .. end - 1 of the row
template <bool FEW>
__device__ __forceinline__ SeqIndex seq_index(const PagedDecodeParams& p, int b) {          // L2: this grid may have been there before they were written
  SeqIndex i{__ldcg(p.lens + b), 0, FEW ? p.T : 1};
  if (FEW && p.cu) { i.first = __ldcg(p.cu + b); i.end = __ldcg(p.cu + b + 1); }
  return i;
}
template <bool FEW>
__device__ __forceinline__ SeqRange seq_range(const PagedDecodeParams& p, const SeqIndex& i) {
  SeqRange r;
  r.len = i.len;
  bool bad;
  if (FEW) {
    const bool sane = i.first >= 0 && i.end >= i.first && i.end <= p.T;                      // offsets outside the row: no queries
    r.n = sane ? i.end - i.first : 0;
    r.row0 = sane ? i.first : 0;
    bad = !sane || (r.n > 0 && r.len >= 0 && (r.len < r.n || r.len > p.c.capacity()));
  } else {
    r.n = 1; r.row0 = 0;
    bad = r.len >= p.c.capacity() || ((p.flags & DAISY_ROPE) && r.len >= p.table_rows);
  }
  if (bad && p.status) p.status[0] = DAISY_EINVAL;
  if (r.len < 0 || bad) r.len = -1;
  r.pos0 = FEW ? r.len - r.n : r.len;
  r.lo = p.window > 0 && r.pos0 > p.window - 1 ? r.pos0 - (p.window - 1) : 0;
  r.tile0 = r.lo / PD_TILE;
  r.tiles = r.len <= r.lo ? 1 : (r.len + PD_TILE - 1) / PD_TILE - r.tile0;      // one without rows: the token alone
  r.blocks = PD_HEAD + (r.tiles + PD_WARPS - 1) / PD_WARPS;
  return r;
}
// (key head, group of columns) pairs of a sequence
template <bool FEW>
__device__ __forceinline__ int pairs_of(const PagedDecodeParams& p, const SeqRange& r, int cols) {
  return p.c.H * (FEW ? (r.n * p.G + cols - 1) / cols : p.n_grp);
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Four channels 4 lane .. 4 lane + 3 of a row, normalised and rotated by the whole warp.
__device__ __forceinline__ void row_of_warp(const __nv_bfloat16* src, bool norm, bool rope, float eps, const float* cos_row, const float* sin_row,
                                            int lane, float (&x)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(src + 4 * lane);
  x[0] = bf16_lo(u.x); x[1] = bf16_hi(u.x); x[2] = bf16_lo(u.y); x[3] = bf16_hi(u.y);
  if (norm) {
    const float r = rsqrtf(warp_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]) * (1.0f / DAISY_HEAD_DIM) + eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= r;
  }
  if (rope) {
    const float4 c = *reinterpret_cast<const float4*>(cos_row + 4 * (lane & 15)), s = *reinterpret_cast<const float4*>(sin_row + 4 * (lane & 15));
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
    const float sgn = lane < 16 ? 1.f : -1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float other = __shfl_xor_sync(0xffffffffu, x[e], 16);
      x[e] = x[e] * cc[e] + sgn * other * ss[e];
    }
  }
}

// Index entries of the first PD_KEPT sequences stay in shared memory.
constexpr int PD_KEPT = 32 * PD_WARPS;
struct DealSmem { int warp_sum[PD_WARPS]; int before, b; SeqIndex kept[PD_KEPT]; };

// This CTA's run of blocks [t, t_end) of the batch, the sequence b that holds t, and where b's blocks begin.  The whole block calls it.
struct Deal { int t, t_end, share, b_at, b; };
template <bool FEW>
__device__ __forceinline__ Deal deal_tiles(const PagedDecodeParams& p, int cols, DealSmem* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Deal d;
  int base, x, t, total = 0;
  // blocks of sequences b0 .. b0 + PD_KEPT - 1: this thread's, their inclusive prefix sum, what lies in front of its warp
  auto scan = [&](int b0) {
    const int b = b0 + threadIdx.x;
    x = t = 0;
    if (b < p.c.n_seq) {
      const SeqIndex at = seq_index<FEW>(p, b);
      if (b0 == 0) sm->kept[threadIdx.x] = at;
      const SeqRange r = seq_range<FEW>(p, at);
      x = t = r.blocks * pairs_of<FEW>(p, r, cols);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sm->warp_sum[warp] = x;
    __syncthreads();
    base = 0;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < PD_WARPS; ++w) { if (w < warp) base += sm->warp_sum[w]; sum += sm->warp_sum[w]; }
    return sum;
  };
  if (threadIdx.x == 0) sm->b = -1;
  total = scan(0);
  const int first_sum = total;
  for (int b0 = PD_KEPT; b0 < p.c.n_seq; b0 += PD_KEPT) {
    __syncthreads();
    total += scan(b0);
  }
  d.share = (int)(((unsigned)total + gridDim.x - 1) / gridDim.x);
  d.t = min((unsigned)blockIdx.x * (unsigned)d.share, (unsigned)total);
  d.t_end = (int)min((unsigned)d.t + (unsigned)d.share, (unsigned)total);
  d.b = -1;
  if (d.t >= d.t_end) return d;
  const int want = d.t;
  int front = 0;
  for (int b0 = 0; b0 < p.c.n_seq; b0 += PD_KEPT) {
    int sum = first_sum;
    if (p.c.n_seq > PD_KEPT) { __syncthreads(); sum = scan(b0); }
    if (want < front + sum) {
      const int at = front + base + x - t;
      if (t > 0 && at <= want && want < at + t) { sm->b = b0 + threadIdx.x; sm->before = at; }
      break;
    }
    front += sum;
  }
  __syncthreads();
  d.b = sm->b;
  d.b_at = sm->before;
  return d;
}

// Sums of one head: channels 4 lane .. of the numerator, reference, denominator.
struct Sums { float4 num; float ref, den; };

// Shares of CTAs from, from + step, .. <= to, every fourth to a warp, into the warps' places in shared memory (acc [4][NQ][128], m, l [4][NQ]).
// A function of its own: inlined, what it computes ahead takes the registers of the main loop (spills, 322 -> 458 us); with four heads at once
// its own registers do (322 -> 550 us).
template <int NQ>
__device__ __noinline__ void join_shares(const float* part, float* acc, float* m, float* l, int n_q, int from, int to, int step, int first_cta) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int col = 0; col < n_q; col += 2) {
    Sums x[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) x[k] = Sums{make_float4(0.f, 0.f, 0.f, 0.f), PD_NEG, 0.f};
    for (int cc = from + warp * step; cc <= to; cc += 4 * PD_WARPS * step) {
      float4 n1[4][2];
      float2 rd[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ci = cc + i * PD_WARPS * step <= to ? cc + i * PD_WARPS * step : cc;
        const float* src = part + ((int64_t)ci * 2 + (ci == first_cta ? 1 : 0)) * NQ * PD_PART + col * PD_PART;
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (k == 0 || col + 1 < n_q) {
            n1[i][k] = __ldcg(reinterpret_cast<const float4*>(src + k * PD_PART) + lane);
            rd[i][k] = __ldcg(reinterpret_cast<const float2*>(src + k * PD_PART + 128));
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (cc + i * PD_WARPS * step <= to) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (k == 0 || col + 1 < n_q) {
              Sums& y = x[k];
              const float top = fmaxf(y.ref, rd[i][k].x), a = fast_exp2(y.ref - top), e = fast_exp2(rd[i][k].x - top);
              y.num = make_float4(y.num.x * a + e * n1[i][k].x, y.num.y * a + e * n1[i][k].y, y.num.z * a + e * n1[i][k].z, y.num.w * a + e * n1[i][k].w);
              y.den = y.den * a + e * rd[i][k].y;
              y.ref = top;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k == 0 || col + 1 < n_q) {
        *reinterpret_cast<float4*>(acc + (warp * NQ + col + k) * DAISY_HEAD_DIM + 4 * lane) = x[k].num;
        if (lane == 0) { m[warp * NQ + col + k] = x[k].ref; l[warp * NQ + col + k] = x[k].den; }
      }
  }
}

// The token's own row of pair (b, h) and its scores, by all warps but the first: k and v as they will lie in the page, its page, v in fp32, the
// scores of query heads q_h0 .. q_h0 + n_q - 1 (in the exp2 domain).
struct OwnRow { float4 v[32]; uint2 k16[32], v16[32]; int page; };
template <bool F16>
__device__ __forceinline__ void own_row(const PagedDecodeParams& p, int b, int h, int q_h0, int n_q, int len, OwnRow* own, float* scores) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float *cos_row = p.cos + (int64_t)len * 64, *sin_row = p.sin + (int64_t)len * 64;
  int page = 0;
  if (warp == PD_WARPS - 1) page = __ldcg(p.c.table + b * p.c.table_sb + (len >> p.c.lg));
  float kr[4];
  row_of_warp(p.k + b * p.k_sb + h * p.k_sh, p.flags & DAISY_NORM_K, p.flags & DAISY_ROPE, p.eps, cos_row, sin_row, lane, kr);
  const uint2 k16 = make_uint2(pack16<F16>(kr[0], kr[1]), pack16<F16>(kr[2], kr[3]));
  const float2 ka = unpack16<F16>(k16.x), kc = unpack16<F16>(k16.y);
  for (int col = warp - 1; col < n_q; col += PD_WARPS - 1) {
    float x[4];
    row_of_warp(p.q + b * p.q_sb + (q_h0 + col) * p.q_sh, p.flags & DAISY_NORM_Q, p.flags & DAISY_ROPE, p.eps, cos_row, sin_row, lane, x);
    const float s = warp_sum(x[0] * ka.x + x[1] * ka.y + x[2] * kc.x + x[3] * kc.y) * p.qscale;
    if (lane == 0) scores[col] = s;
  }
  if (warp == PD_WARPS - 1) {
    float vr[4];
    row_of_warp(p.v + b * p.v_sb + h * p.v_sh, p.flags & DAISY_NORM_V, false, p.eps, cos_row, sin_row, lane, vr);
    if (p.ve) {
      const float gate = 1.0f / (1.0f + __expf(-*p.ve_gate));
      const uint2 u = *reinterpret_cast<const uint2*>(p.ve + b * p.ve_sb + h * p.ve_sh + 4 * lane);
      const float e[4] = {bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)};
#pragma unroll
      for (int i = 0; i < 4; ++i) vr[i] = gate * vr[i] + (1.0f - gate) * e[i];
    }
    const uint2 v16 = make_uint2(pack16<F16>(vr[0], vr[1]), pack16<F16>(vr[2], vr[3]));
    const float2 va = unpack16<F16>(v16.x), vc = unpack16<F16>(v16.y);
    own->v[lane] = make_float4(va.x, va.y, vc.x, vc.y);
    own->k16[lane] = k16;
    own->v16[lane] = v16;
    if (lane == 0) own->page = page;
  }
}

template <int NT, bool F16, bool FEW>
__global__ void __launch_bounds__(32 * PD_WARPS, pd_ctas(8 * NT)) paged_decode_kernel(const __grid_constant__ PagedDecodeParams p) {
  constexpr int NQ = 8 * NT;                                         // query heads of a pass, the last ones maybe absent
  __shared__ DealSmem sm_deal;
  __shared__ __align__(16) float sm_acc[PD_WARPS][NQ][DAISY_HEAD_DIM];
  __shared__ float sm_m[PD_WARPS][NQ], sm_l[PD_WARPS][NQ];
  __shared__ float sm_self[NQ];
  __shared__ OwnRow sm_own;
  __shared__ int sm_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  grid_dep_launch();
  grid_dep_wait();

  const Deal deal = deal_tiles<FEW>(p, NQ, &sm_deal);                // pairs are (sequence, head)-major
  if (deal.b < 0) return;
  const int t_end = deal.t_end, share = deal.share;
  int t = deal.t, b_at = deal.b_at;
  int b = deal.b;
  auto range_of = [&](int i) { return seq_range<FEW>(p, i < PD_KEPT ? sm_deal.kept[i] : seq_index<FEW>(p, i)); };
  SeqRange r = range_of(b);

  while (t < t_end) {
    while (t >= b_at + r.blocks * pairs_of<FEW>(p, r, NQ)) {
      if (b + 1 >= p.c.n_seq) return;                                // lengths that changed under the call
      b_at += r.blocks * pairs_of<FEW>(p, r, NQ);
      r = range_of(++b);
    }
    const int n_grp = FEW ? (r.n * p.G + NQ - 1) / NQ : p.n_grp;
    const int hh = (t - b_at) / r.blocks, h = hh / n_grp, grp = hh % n_grp;
    const int u_at = b_at + hh * r.blocks;                           // this pair's blocks: u_at .. u_end - 1
    const int u_end = u_at + r.blocks, s_end = min(u_end, t_end);
    const int r_at = max(t, u_at + PD_HEAD);                         // this CTA's blocks with rows: r_at .. s_end - 1
    if (r_at >= s_end) { t = s_end; continue; }
    const int q_h0 = h * p.G + grp * NQ, n_q = min(NQ, (FEW ? r.n * p.G : p.G) - grp * NQ);
    // FEW: column -> query of the sequence
    auto query_of = [&](int col) { return (grp * NQ + col) / p.G; };
    auto q_at = [&](int col) -> const __nv_bfloat16* {
      if (!FEW) return p.q + b * p.q_sb + (q_h0 + col) * p.q_sh;
      const int i = query_of(col);
      return p.q + (p.cu ? 0 : b) * p.q_sb + (int64_t)(r.row0 + i) * p.q_st + (h * p.G + grp * NQ + col - i * p.G) * p.q_sh;
    };
    const float *cos_row = p.cos + (int64_t)max(r.len, 0) * 64, *sin_row = p.sin + (int64_t)max(r.len, 0) * 64;

    // what the queries are made of is asked for first: the table's entry and the rows behind it take longer
    uint4 q_raw[NT][4];
    float4 cs4[2][2], sn4[2][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        q_raw[n][j] = 8 * n + g < n_q ? ld_cg16(q_at(8 * n + g) + 32 * j + 8 * c) : make_uint4(0, 0, 0, 0);
    if constexpr (!FEW)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cs4[j][i] = make_float4(1.f, 1.f, 1.f, 1.f);
        sn4[j][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.flags & DAISY_ROPE) {
          cs4[j][i] = *reinterpret_cast<const float4*>(cos_row + 32 * j + 8 * c + 4 * i);
          sn4[j][i] = *reinterpret_cast<const float4*>(sin_row + 32 * j + 8 * c + 4 * i);
        }
      }
    const int* table = p.c.table + b * p.c.table_sb;
    const int first = r.tile0 + (r_at - u_at - PD_HEAD) * PD_WARPS, last = r.tile0 + min((s_end - u_at - PD_HEAD) * PD_WARPS, r.tiles);    // tiles of the sequence
    auto page_of = [&](int tile) -> int {                            // a row outside the pool is taken from page 0
      int pg = tile < last && r.len > r.lo ? __ldcg(table + ((tile * PD_TILE) >> p.c.lg)) : 0;
      if ((unsigned)pg >= (unsigned)p.c.n_pages) {
        if (p.status) p.status[0] = DAISY_EINVAL;
        pg = 0;
      }
      return pg;
    };
    // A tile's rows as lane (g, c) takes them: keys g, g + 8, pieces 32 j + 8 c of the channels; values of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9, channels
    // 8 g .. and 64 + 8 g ...  Rows that nobody sees may hold anything: they count as zeros.
    const int64_t sr = 2 * p.c.p_sr;
    auto seen = [&](int row) { return row >= r.lo && row < r.len; };
    auto whole = [&](int tile) { return tile * PD_TILE >= r.lo && tile * PD_TILE + PD_TILE <= r.len; };
    int q_pos[NT][2];                                                // FEW: positions of this lane's columns
    if constexpr (FEW)
#pragma unroll
      for (int n = 0; n < NT; ++n) { q_pos[n][0] = r.pos0 + query_of(8 * n + 2 * c); q_pos[n][1] = r.pos0 + query_of(8 * n + 2 * c + 1); }
    // the first position that all queries see, and the last
    const int all_lo = FEW && p.window > 0 ? max(r.lo, r.len - p.window) : r.lo, all_hi = FEW ? r.pos0 : r.len - 1;
    auto fetch_k = [&](int tile, int pg, uint4 (&kk)[2][4]) {
      const char* kb = p.c.k + p.c.at(pg, h, tile * PD_TILE) + 16 * c;
      if (whole(tile)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) kk[i][j] = ld_stream16(kb + (g + 8 * i) * sr + 64 * j);
        return;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = seen(tile * PD_TILE + g + 8 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) kk[i][j] = in ? ld_stream16(kb + (g + 8 * i) * sr + 64 * j) : make_uint4(0, 0, 0, 0);
      }
    };
    auto fetch_v = [&](int tile, int pg, uint4 (&vv)[4][2]) {
      const char* vb = p.c.v + p.c.at(pg, h, tile * PD_TILE) + 16 * g;
      if (whole(tile)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) vv[i][j] = ld_stream16(vb + (2 * c + (i & 1) + 8 * (i >> 1)) * sr + 128 * j);
        return;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * c + (i & 1) + 8 * (i >> 1);
        const bool in = seen(tile * PD_TILE + row);
#pragma unroll
        for (int j = 0; j < 2; ++j) vv[i][j] = in ? ld_stream16(vb + row * sr + 128 * j) : make_uint4(0, 0, 0, 0);
      }
    };
    uint4 kk[2][4], vv[4][2];
    int pg = page_of(first + warp), pg_next = page_of(first + warp + PD_WARPS);
    if (first + warp < last) {                                       // on their way under the queries' preparation
      fetch_k(first + warp, pg, kk);
      fetch_v(first + warp, pg, vv);
    }
    // ---------------------------------------------------------------- the queries as B operands: lane (g, c) holds head 8 n + g, channels
    // 32 j + 8 c .. + 7 for j = 0..3; element pair i of piece j goes to k step 2 j + i / 2
    // The second halves of the sums lie in shared memory, a lane's own (16 registers NT that the rows' loads need); the place is the warp's sums',
    // which are left there after the last tile.
    uint32_t qh[NT][4][4];
    uint4* q_low = reinterpret_cast<uint4*>(&sm_acc[warp][0][0]) + lane;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[4][8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (FEW) {                                                   // prepared, in the pages' type
          const uint32_t u[4] = {q_raw[n][j].x, q_raw[n][j].y, q_raw[n][j].z, q_raw[n][j].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) { const float2 f = unpack16<F16>(u[i]); x[j][2 * i] = f.x * p.qscale; x[j][2 * i + 1] = f.y * p.qscale; }
        } else {
          unpack8(q_raw[n][j], x[j]);
        }
      }
      if constexpr (!FEW) {
      float mul = p.qscale;
      if (p.flags & DAISY_NORM_Q) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[j][e], x[j][e], ss);
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        mul *= rsqrtf(ss * (1.0f / DAISY_HEAD_DIM) + p.eps);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float cs[8] = {cs4[j][0].x, cs4[j][0].y, cs4[j][0].z, cs4[j][0].w, cs4[j][1].x, cs4[j][1].y, cs4[j][1].z, cs4[j][1].w};
        const float sn[8] = {sn4[j][0].x, sn4[j][0].y, sn4[j][0].z, sn4[j][0].w, sn4[j][1].x, sn4[j][1].y, sn4[j][1].z, sn4[j][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = x[j][e] * mul, d = x[j + 2][e] * mul;
          x[j][e] = a * cs[e] + d * sn[e];
          x[j + 2][e] = d * cs[e] - a * sn[e];
        }
      }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qh[n][j][i] = pack16<F16>(x[j][2 * i], x[j][2 * i + 1]);
          const float2 back = unpack16<F16>(qh[n][j][i]);
          lo[i] = pack16<F16>(x[j][2 * i] - back.x, x[j][2 * i + 1] - back.y);
        }
        q_low[(n * 4 + j) * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }

    float acc[NT][8][4];                                             // channels 8 g + e (elements 0, 1) and 64 + 8 g + e of heads 2 c, 2 c + 1
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[n][e][0] = acc[n][e][1] = acc[n][e][2] = acc[n][e][3] = 0.f;
      m[n][0] = m[n][1] = PD_NEG;
      l[n][0] = l[n][1] = 0.f;
    }

    for (int tile = first + warp; tile < last; tile += PD_WARPS) {
      const int row0 = tile * PD_TILE, next = tile + PD_WARPS;
      if (tile != first + warp) { fetch_k(tile, pg_next, kk); fetch_v(tile, pg_next, vv); pg_next = page_of(next); }
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 ql[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) ql[n] = q_low[(n * 4 + j) * 32];
        const uint32_t k0[4] = {kk[0][j].x, kk[0][j].y, kk[0][j].z, kk[0][j].w}, k1[4] = {kk[1][j].x, kk[1][j].y, kk[1][j].z, kk[1][j].w};
#pragma unroll
        for (int i = 0; i < 4; i += 2)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816<F16>(s[n], k0[i], k1[i], k0[i + 1], k1[i + 1], qh[n][j][i], qh[n][j][i + 1]);
            mma16816<F16>(s[n], k0[i], k1[i], k0[i + 1], k1[i + 1], i ? ql[n].z : ql[n].x, i ? ql[n].w : ql[n].y);
          }
      }
      if constexpr (FEW) {
        if (row0 < all_lo || row0 + PD_TILE - 1 > all_hi) {
          auto hidden = [&](int key, int pos) { return key > pos || (p.window > 0 && key <= pos - p.window); };
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (hidden(row0 + g + 8 * (i >> 1), q_pos[n][i & 1])) s[n][i] = -INFINITY;
        }
      } else if (!whole(tile)) {
        const bool in0 = seen(row0 + g), in1 = seen(row0 + g + 8);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (!in0) s[n][0] = s[n][1] = -INFINITY;
          if (!in1) s[n][2] = s[n][3] = -INFINITY;
        }
      }
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float t0 = fmaxf(s[n][0], s[n][2]), t1 = fmaxf(s[n][1], s[n][3]);
        // the reference follows the maximum only when that has grown by over 2^8: sums stay far inside their range
        if (__any_sync(0xffffffffu, t0 > m[n][0] + (8.f + WEIGHT_ROOM<F16>) || t1 > m[n][1] + (8.f + WEIGHT_ROOM<F16>))) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
          }
          t0 = fmaxf(t0 - WEIGHT_ROOM<F16>, m[n][0]); t1 = fmaxf(t1 - WEIGHT_ROOM<F16>, m[n][1]);
          const float a0 = fast_exp2(m[n][0] - t0), a1 = fast_exp2(m[n][1] - t1);
          m[n][0] = t0; m[n][1] = t1;
          l[n][0] *= a0; l[n][1] *= a1;
#pragma unroll
          for (int e = 0; e < 8; ++e) { acc[n][e][0] *= a0; acc[n][e][1] *= a1; acc[n][e][2] *= a0; acc[n][e][3] *= a1; }
        }
        const float w0 = fast_exp2(s[n][0] - m[n][0]), w1 = fast_exp2(s[n][1] - m[n][1]);
        const float w2 = fast_exp2(s[n][2] - m[n][0]), w3 = fast_exp2(s[n][3] - m[n][1]);
        l[n][0] += w0 + w2; l[n][1] += w1 + w3;
        const uint32_t h0 = pack16<F16>(w0, w1), h1 = pack16<F16>(w2, w3);
        const float2 b0 = unpack16<F16>(h0), b1 = unpack16<F16>(h1);
        ph[n][0] = transpose8x8(h0); ph[n][1] = transpose8x8(h1);
        pl[n][0] = transpose8x8(pack16<F16>(w0 - b0.x, w1 - b0.y)); pl[n][1] = transpose8x8(pack16<F16>(w2 - b1.x, w3 - b1.y));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t a[4];                                               // channels 8 g + e, 64 + 8 g + e of keys 2 c, 2 c + 1 | 2 c + 8, 2 c + 9
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 lo4 = vv[i & 2][i & 1], hi4 = vv[(i & 2) + 1][i & 1];
          const uint32_t lo = e < 2 ? lo4.x : e < 4 ? lo4.y : e < 6 ? lo4.z : lo4.w, hi = e < 2 ? hi4.x : e < 4 ? hi4.y : e < 6 ? hi4.z : hi4.w;
          a[i] = __byte_perm(lo, hi, (e & 1) ? 0x7632 : 0x5410);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<F16>(acc[n][e], a[0], a[1], a[2], a[3], ph[n][0], ph[n][1]);
          mma16816<F16>(acc[n][e], a[0], a[1], a[2], a[3], pl[n][0], pl[n][1]);
        }
      }
    }

    // ---------------------------------------------------------------- the four warps' sums
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = l[n][i];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int col = 8 * n + 2 * c + i;
        if (col < n_q) {
          if (g == 0) { sm_m[warp][col] = m[n][i]; sm_l[warp][col] = x; }
          float* dst = &sm_acc[warp][col][8 * g];
          *reinterpret_cast<float4*>(dst) = make_float4(acc[n][0][i], acc[n][1][i], acc[n][2][i], acc[n][3][i]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[n][4][i], acc[n][5][i], acc[n][6][i], acc[n][7][i]);
          *reinterpret_cast<float4*>(dst + 64) = make_float4(acc[n][0][2 + i], acc[n][1][2 + i], acc[n][2][2 + i], acc[n][3][2 + i]);
          *reinterpret_cast<float4*>(dst + 68) = make_float4(acc[n][4][2 + i], acc[n][5][2 + i], acc[n][6][2 + i], acc[n][7][2 + i]);
        }
      }
    __syncthreads();
    const bool alone = u_at + PD_HEAD >= deal.t && u_end <= t_end;
    // sums of head `col` over the four warps
    auto mine = [&](int col) {
      Sums x{make_float4(0.f, 0.f, 0.f, 0.f), fmaxf(fmaxf(sm_m[0][col], sm_m[1][col]), fmaxf(sm_m[2][col], sm_m[3][col])), 0.f};
#pragma unroll
      for (int w = 0; w < PD_WARPS; ++w) {
        const float e = fast_exp2(sm_m[w][col] - x.ref);
        const float4 y = *reinterpret_cast<const float4*>(&sm_acc[w][col][4 * lane]);
        x.num.x = fmaf(e, y.x, x.num.x); x.num.y = fmaf(e, y.y, x.num.y); x.num.z = fmaf(e, y.z, x.num.z); x.num.w = fmaf(e, y.w, x.num.w);
        x.den = fmaf(e, sm_l[w][col], x.den);
      }
      return x;
    };
    const int c0 = (u_at + PD_HEAD) / share, c1 = (u_end - 1) / share;            // the CTAs that share this pair
    // Shares are joined by groups of PD_JOIN CTAs, then the groups: the last one of a group to come joins it into the place of the
    // group's first, the last group the pair.
    const int c_grp = c0 + ((int)blockIdx.x - c0) / PD_JOIN * PD_JOIN, n_grps = (c1 - c0) / PD_JOIN + 1;
    auto place = [&](int cta) { return (int64_t)cta * 2 + (cta == c0 ? 1 : 0); };
    if (!alone) {
      float* dst = p.part + place(blockIdx.x) * NQ * PD_PART;
      for (int col = warp; col < n_q; col += PD_WARPS) {
        const Sums x = mine(col);
        __stcg(reinterpret_cast<float4*>(dst + col * PD_PART) + lane, x.num);
        if (lane == 0) __stcg(reinterpret_cast<float2*>(dst + col * PD_PART + 128), make_float2(x.ref, x.den));
      }
      __threadfence();
      __syncthreads();
    }
    // one thread asks whether all other shares are there; under that the other warps prepare the token's own row
    if (threadIdx.x == 0) {
      sm_last = 1;
      if (!alone) {                                                  // of the group's shares, or of the pair's where there is one group
        int* tk = n_grps > 1 ? p.tickets_grp + place(c_grp) : p.tickets + ((int64_t)b * p.c.H * p.n_grp + hh);
        const int of = min(c_grp + PD_JOIN - 1, c1) - c_grp;
        sm_last = atomicAdd(tk, 1) == of;
        if (sm_last) *tk = 0;                                        // every other one has been drawn
      }
    } else if (!FEW && warp > 0 && r.len >= 0) {
      own_row<F16>(p, b, h, q_h0, n_q, r.len, &sm_own, sm_self);
    }
    __syncthreads();
    bool finish = sm_last != 0;
    if (finish && !alone) {
      __threadfence();
      join_shares<NQ>(p.part, &sm_acc[0][0][0], &sm_m[0][0], &sm_l[0][0], n_q, c_grp, min(c_grp + PD_JOIN - 1, c1), 1, c0);
      __syncthreads();
    }
    if (finish && n_grps > 1) {
      float* dst = p.part + place(c_grp) * NQ * PD_PART;
      for (int col = warp; col < n_q; col += PD_WARPS) {
        const Sums x = mine(col);
        __stcg(reinterpret_cast<float4*>(dst + col * PD_PART) + lane, x.num);
        if (lane == 0) __stcg(reinterpret_cast<float2*>(dst + col * PD_PART + 128), make_float2(x.ref, x.den));
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        int* tk = p.tickets + ((int64_t)b * p.c.H * p.n_grp + hh);
        sm_last = atomicAdd(tk, 1) == n_grps - 1;
        if (sm_last) *tk = 0;
      }
      __syncthreads();
      finish = sm_last != 0;
      if (finish) {
        __threadfence();
        join_shares<NQ>(p.part, &sm_acc[0][0][0], &sm_m[0][0], &sm_l[0][0], n_q, c0, c1, PD_JOIN, c0);
        __syncthreads();
      }
    }
    if (finish) {
      if (!FEW && warp == PD_WARPS - 1 && grp == 0 && r.len >= 0) {
        if ((unsigned)sm_own.page < (unsigned)p.c.n_pages) {
          const int64_t at = p.c.at(sm_own.page, h, r.len) + 8 * lane;
          *reinterpret_cast<uint2*>(p.c.k + at) = sm_own.k16[lane];
          *reinterpret_cast<uint2*>(p.c.v + at) = sm_own.v16[lane];
        } else if (p.status && lane == 0) {
          p.status[0] = DAISY_EINVAL;
        }
      }
      for (int col = warp; col < n_q; col += PD_WARPS) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r.len >= 0) {
          const Sums x = mine(col);
          if (FEW) {
            const float inv = 1.0f / x.den;
            y = make_float4(x.num.x * inv, x.num.y * inv, x.num.z * inv, x.num.w * inv);
          } else {
            const float self = sm_self[col], top = fmaxf(x.ref, self), a = fast_exp2(x.ref - top), w = fast_exp2(self - top);
            const float4 v = sm_own.v[lane];
            const float inv = 1.0f / (x.den * a + w), ai = a * inv, wi = w * inv;
            y = make_float4(x.num.x * ai + wi * v.x, x.num.y * ai + wi * v.y, x.num.z * ai + wi * v.z, x.num.w * ai + wi * v.w);
          }
        }
        __nv_bfloat16* dst = p.out + 4 * lane;
        if (FEW) {
          const int i = query_of(col);
          dst += (p.cu ? 0 : b) * p.o_sb + (int64_t)(r.row0 + i) * p.o_st + (h * p.G + grp * NQ + col - i * p.G) * p.o_sh;
        } else {
          dst += b * p.o_sb + (q_h0 + col) * p.o_sh;
        }
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
      }
    }
    t = s_end;
    if (t < t_end) __syncthreads();                                  // shared memory is used again
  }
}

}  // namespace daisy

using namespace daisy;

// query heads a pass: 8, or 16 where a key head has more than 8
static int decode_cols(int G) { return G > 8 ? 16 : 8; }
// Partial sums of either form.  The tickets begin behind them whatever the sizes of a call are: calls of different sizes share a
// workspace, and only tickets are ever written where another call's tickets lie.
static size_t partials_bytes(int sms) {
  constexpr size_t cols = pd_ctas(8) * 8 > pd_ctas(16) * 16 ? pd_ctas(8) * 8 : pd_ctas(16) * 16;
  return (size_t)sms * 2 * cols * PD_PART * sizeof(float);
}
static size_t group_tickets_bytes(int sms) { return (size_t)sms * 2 * pd_ctas(8) * sizeof(int); }

extern "C" size_t daisy_b200_paged_decode_workspace_bytes(int n_seq, int Hq, int H, int D) {
  if (n_seq <= 0 || Hq <= 0 || H <= 0 || D != DAISY_HEAD_DIM || Hq % H) return 0;
  int sms = daisy_host::sm_count_cached();
  if (sms <= 0) sms = daisy_host::MAX_SMS;
  const int nq = decode_cols(Hq / H), n_grp = (Hq / H + nq - 1) / nq;
  return partials_bytes(sms) + group_tickets_bytes(sms) + ((size_t)n_seq * H * n_grp * sizeof(int) + 15) / 16 * 16;
}

extern "C" int daisy_b200_paged_decode_step(const daisy_b200_pages* cache, const void* q_new, const void* k_new, const void* v_new,
                                            int64_t q_sb, int64_t q_sh, int64_t k_sb, int64_t k_sh, int64_t v_sb, int64_t v_sh,
                                            const int32_t* lens, int window, const float* cos, const float* sin, int table_rows,
                                            void* out, int64_t o_sb, int64_t o_sh,
                                            const void* ve, int64_t ve_sb, int64_t ve_sh, const float* ve_gate_logit,
                                            int Hq, int D, float scale, float eps, unsigned flags,
                                            void* workspace, size_t workspace_bytes, int* status_word, void* stream) {
  PagedDecodeParams p = {};
  if (const int rc = daisy_host::paged_cache(cache, D, &p.c); rc != DAISY_OK) return rc;
  if (!q_new || !k_new || !v_new || !lens || !out || !workspace || Hq <= 0 || Hq % cache->H) return DAISY_EINVAL;
  if (flags & ~(DAISY_QKV_DEFAULT | DAISY_CACHE_FP16)) return DAISY_EINVAL;
  if ((flags & DAISY_ROPE) && (!cos || !sin || table_rows <= 0)) return DAISY_EINVAL;
  if (ve && (!ve_gate_logit || !(flags & DAISY_NORM_V))) return DAISY_EINVAL;
  if (!daisy_aligned16(q_new) || !daisy_aligned16(k_new) || !daisy_aligned16(v_new) || !daisy_aligned16(ve) || !daisy_aligned16(workspace) ||
      ((q_sb | q_sh | k_sb | k_sh | v_sb | v_sh) & 7) || (ve && ((ve_sb | ve_sh) & 7)) || (reinterpret_cast<uintptr_t>(lens) & 3) ||
      (reinterpret_cast<uintptr_t>(out) & 7) || ((o_sb | o_sh) & 3))
    return DAISY_EALIGN;
  if ((flags & DAISY_ROPE) && (!daisy_aligned16(cos) || !daisy_aligned16(sin))) return DAISY_EALIGN;
  // rows are written: none may stand for two
  if ((cache->n_seq > 1 && o_sb <= 0) || (Hq > 1 && o_sh <= 0)) return DAISY_EINVAL;
  if (workspace_bytes < daisy_b200_paged_decode_workspace_bytes(cache->n_seq, Hq, cache->H, D)) return DAISY_EWORKSPACE;
  const int sms = daisy_host::sm_count_cached();
  if (sms <= 0) return DAISY_ENODEV;
  p.G = Hq / cache->H; p.Hq = Hq;
  const int nq = decode_cols(p.G);
  p.n_grp = (p.G + nq - 1) / nq;
  // blocks are counted in 32 bits
  const int64_t blocks = (int64_t)cache->width * cache->page / (PD_TILE * PD_WARPS) + 2 + PD_HEAD, pairs = (int64_t)cache->n_seq * cache->H * p.n_grp;
  if (pairs >= (int64_t)1 << 31 || blocks * pairs >= ((int64_t)1 << 31) - 65536) return DAISY_EUNSUPPORTED;
  p.q = (const __nv_bfloat16*)q_new; p.k = (const __nv_bfloat16*)k_new; p.v = (const __nv_bfloat16*)v_new; p.ve = (const __nv_bfloat16*)ve;
  p.q_sb = q_sb; p.q_sh = q_sh; p.k_sb = k_sb; p.k_sh = k_sh; p.v_sb = v_sb; p.v_sh = v_sh; p.ve_sb = ve_sb; p.ve_sh = ve_sh;
  p.o_sb = o_sb; p.o_sh = o_sh;
  p.out = (__nv_bfloat16*)out;
  p.lens = lens; p.cos = cos; p.sin = sin; p.ve_gate = ve_gate_logit;
  p.window = daisy_host::paged_window(cache, window); p.table_rows = table_rows;
  p.qscale = scale * 1.4426950408889634f;
  p.eps = eps; p.flags = flags; p.status = status_word;
  const unsigned grid = (unsigned)(sms * pd_ctas(nq));
  p.part = (float*)workspace;
  p.tickets_grp = (int*)((char*)workspace + partials_bytes(sms));
  p.tickets = (int*)((char*)p.tickets_grp + group_tickets_bytes(sms));
  const bool f16 = (flags & DAISY_CACHE_FP16) != 0;
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto kernel) { return daisy_host::launch_dependent(kernel, dim3(grid), dim3(32 * PD_WARPS), 0, st, p); };
  const cudaError_t e = nq == 8 ? (f16 ? go(paged_decode_kernel<1, true, false>) : go(paged_decode_kernel<1, false, false>))
                                : (f16 ? go(paged_decode_kernel<2, true, false>) : go(paged_decode_kernel<2, false, false>));
  if (e != cudaSuccess) { (void)cudaGetLastError(); return DAISY_ECUDA; }
  DAISY_CHECK_LAUNCH();
  return DAISY_OK;
}

extern "C" int daisy_b200_paged_attend_few_rows(int T, int n_seq, int packed, int Hq, int H) {
  if (T <= 0 || n_seq <= 0 || Hq <= 0 || H <= 0 || Hq % H) return 0;
  const int64_t cols = (int64_t)T * (Hq / H);
  // packed, the lengths are not known here: few tokens, and few a sequence
  return packed ? (cols <= PD_FEW_PACKED && cols <= (int64_t)n_seq * (PD_FEW / 2) ? (int)cols : 0) : (cols <= PD_FEW ? (int)cols : 0);
}

extern "C" size_t daisy_b200_paged_attend_few_workspace_bytes(int n_seq, int H, int D) {
  if (n_seq <= 0 || H <= 0 || D != DAISY_HEAD_DIM) return 0;
  int sms = daisy_host::sm_count_cached();
  if (sms <= 0) sms = daisy_host::MAX_SMS;
  return partials_bytes(sms) + group_tickets_bytes(sms) + ((size_t)n_seq * H * (PD_FEW_PACKED / PD_FEW) * sizeof(int) + 15) / 16 * 16;
}

extern "C" int daisy_b200_paged_attend_few(const daisy_b200_pages* cache, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                           const int32_t* lens, const int32_t* cu, int window,
                                           void* out, int64_t o_sb, int64_t o_st, int64_t o_sh,
                                           int B, int T, int Hq, int D, float scale, unsigned flags,
                                           void* workspace, size_t workspace_bytes, int* status_word, void* stream) {
  PagedDecodeParams p = {};
  if (const int rc = daisy_host::paged_cache(cache, D, &p.c); rc != DAISY_OK) return rc;
  if (!q || !lens || !out || !workspace || B <= 0 || T <= 0 || Hq <= 0 || Hq % cache->H || !(scale > 0.f)) return DAISY_EINVAL;
  if (flags & ~(DAISY_BOUNDED_QK | DAISY_CACHE_FP16)) return DAISY_EINVAL;
  if (B != (cu ? 1 : cache->n_seq)) return DAISY_EINVAL;
  const int cols = daisy_b200_paged_attend_few_rows(T, cache->n_seq, cu != nullptr, Hq, cache->H);
  if (cols == 0) return DAISY_EUNSUPPORTED;
  p.n_grp = (cols + PD_FEW - 1) / PD_FEW;
  // blocks are counted in 32 bits
  const int64_t blocks = (int64_t)cache->width * cache->page / (PD_TILE * PD_WARPS) + 2 + PD_HEAD, pairs = (int64_t)cache->n_seq * cache->H * p.n_grp;
  if (pairs >= (int64_t)1 << 31 || blocks * pairs >= ((int64_t)1 << 31) - 65536) return DAISY_EUNSUPPORTED;
  if (!daisy_aligned16(q) || !daisy_aligned16(workspace) || ((q_sb | q_st | q_sh) & 7) || ((o_sb | o_st | o_sh) & 3) || (reinterpret_cast<uintptr_t>(out) & 7) ||
      (reinterpret_cast<uintptr_t>(lens) & 3) || (reinterpret_cast<uintptr_t>(cu) & 3))
    return DAISY_EALIGN;
  // rows are written: none may stand for two
  if ((T > 1 && o_st <= 0) || (Hq > 1 && o_sh <= 0) || (B > 1 && o_sb <= 0)) return DAISY_EINVAL;
  if (workspace_bytes < daisy_b200_paged_attend_few_workspace_bytes(cache->n_seq, cache->H, D)) return DAISY_EWORKSPACE;
  const int sms = daisy_host::sm_count_cached();
  if (sms <= 0) return DAISY_ENODEV;
  p.G = Hq / cache->H; p.Hq = Hq; p.T = T; p.cu = cu;
  p.q = (const __nv_bfloat16*)q; p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh;
  p.out = (__nv_bfloat16*)out; p.o_sb = o_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.lens = lens; p.window = daisy_host::paged_window(cache, window);
  p.qscale = scale * 1.4426950408889634f;
  p.status = status_word;
  const unsigned grid = (unsigned)(sms * pd_ctas(PD_FEW));
  p.part = (float*)workspace;
  p.tickets_grp = (int*)((char*)workspace + partials_bytes(sms));
  p.tickets = (int*)((char*)p.tickets_grp + group_tickets_bytes(sms));
  const bool f16 = (flags & DAISY_CACHE_FP16) != 0;
  auto go = [&](auto kernel) { return daisy_host::launch_dependent(kernel, dim3(grid), dim3(32 * PD_WARPS), 0, (cudaStream_t)stream, p); };
  const cudaError_t e = f16 ? go(paged_decode_kernel<1, true, true>) : go(paged_decode_kernel<1, false, true>);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return DAISY_ECUDA; }
  DAISY_CHECK_LAUNCH();
  return DAISY_OK;
}
