// Causal attention of a chunk of every sequence over a paged cache, on tcgen05 tensor cores.
//
// Query i of sequence b stands at position lens[b] - n_b + i and sees the nearest `window` keys up to its own, all of them in
// the pages.  A work item is 256 rows (two 128-row streams that share every K/V tile; 128 where few) of `pack` query heads that
// share a key head: row r is query r / pack, head r % pack, so that a few queries of grouped heads fill the rows.  Tiles of 128 keys.
// Long items of a call with few of them are cut along the keys into pieces, whose sums (fp32) a last launch joins in their
// order.  The lengths are on the device, so a first, one-block launch works out the pieces, longest first, and the attention
// kernel's CTAs draw them one by one.  Where nothing would be cut and the sequences have as many queries each, or are few, the items are
// counted off instead, in one launch.
//
// Roles (as in the dense prefill kernel): two softmax warpgroups a stream, 64 key columns each, where the caller bounds the
// logits (no running maximum is needed then), else one a stream with the whole row and a lazily refreshed reference maximum; a
// TMA producer; an MMA issuer.  TMEM: S_0 S_1 O_0 O_1, 128 columns each; P overwrites S.
//
// K/V tiles come page by page (a box of min(page, 128) rows and 64 channels, 128-byte swizzle); pages that nobody sees are not
// touched.  What rows of a tile hold that nobody sees (other sequences' old rows, anything) must not reach an output: their
// scores are replaced, and the issuer clears their V rows in shared memory, since 0 x NaN is NaN in a product.
// All waits are bounded, as in the dense kernel.
#include "paged.cuh"
#include <algorithm>

namespace daisy {

constexpr int PP_BM = 128, PP_BN = 128, PP_NSTAGE = 3, PP_NQBUF = 2, PP_NITEM = 3;
constexpr int PP_TILE = PP_BM * DAISY_HEAD_DIM * 2, PP_HALF = PP_TILE / 2;      // 32 KB; one [128 x 64] swizzled box
constexpr int PP_SMEM_TILES = (2 * PP_NQBUF + PP_NSTAGE) * PP_TILE;
constexpr int PP_BARS = 640;
constexpr int PP_SMEM = 1024 + PP_SMEM_TILES + PP_BARS;
static_assert(PP_SMEM <= 232448, "over the 227 KB a CTA may use");
constexpr float PP_NEG = -1.0e30f;

// A piece: key tiles j0 .. j1 of the item of n queries i0 .. of sequence b, the first at position pos (negative: they see nothing), row row0 of q.
// parts > 1: one of several, at slot + head * parts + part.
struct __align__(16) Piece { int b, i0, j0, j1, slot, part, parts, pos, n, row0, pad[2]; };

struct Cut { int b, i0, slot, parts; };                              // an item in pieces, as Piece has them
struct PlanHead { int n_pieces, queue, n_cuts, pad[5]; };

struct PagedPrefillParams {
  PagedCache c;
  __nv_bfloat16* out;
  int64_t o_sb, o_st, o_sh;
  const int *lens, *cu;
  int T, Hq, G, window, toks;        // toks: queries of an item, 256 or 128 rows / pack
  int lgp, heads;                    // pack = 1 << lgp; heads = Hq / pack
  int counted;                       // > 0: items without a plan, so many a sequence (packed: as the offsets say, up to 32 sequences)
  float scale_log2;
  int* status;
  PlanHead* head;
  Piece* pieces;
  Cut* cuts;
  float* part;                       // [slots][PP_SLOT]
  int slots, max_pieces;             // slots = 0: nothing is cut
};
// a warp's share of a piece's sums: [columns][32 rows], then reference and denominator of the 32 rows
constexpr int PP_SLOT = 2 * 8 * (64 * 32 + 64);                     // floats: 8 warps a stream x 64 columns (or 4 x 128)

// Queries and keys of sequence b: n queries at positions pos .. , n = 0 where there are none; pos < 0: nothing to see (idle, or refused).
struct SeqQueries { int n, row0, pos; bool refused; };
__device__ __forceinline__ SeqQueries seq_queries(const PagedPrefillParams& p, int b) {
  SeqQueries s;
  if (p.cu) {
    const int a = __ldcg(p.cu + b), e = __ldcg(p.cu + b + 1);
    const bool sane = a >= 0 && e >= a && e <= p.T;                  // offsets outside the row: the sequence has no queries
    s.n = sane ? e - a : 0;
    s.row0 = sane ? a : 0;
    s.refused = !sane;
  } else {
    s.n = p.T; s.row0 = 0; s.refused = false;
  }
  const int len = __ldcg(p.lens + b);
  s.pos = len - s.n;
  if (len < 0) s.pos = -1;
  else if (len < s.n || len > p.c.capacity()) { s.pos = -1; s.refused = s.refused || s.n > 0; }
  return s;
}
// key tiles that queries at positions pos .. pos + n - 1 see
__device__ __forceinline__ int first_tile(int pos, int window) { return (window > 0 ? max(0, pos - window + 1) : 0) / PP_BN; }
__device__ __forceinline__ int last_tile(int pos, int n) { return (pos + n - 1) / PP_BN; }

// The pieces of a call, longest first.  One block; a warp a sequence, a lane an item.
// How far items are cut: into pieces of at most L tiles, L from a few candidates by the estimate
// total / CTAs + half a piece such as come last (they go longest first: halfway between the shortest item and the mean), or a longest piece
// where all pieces find a CTA, and PLAN_COST tiles' time for every piece of a cut item
// (its sums are written, and read again by the last: 8192 tokens x 16 heads cut in halves 266 us, whole 233).  Whole items take no less than k of
// the (k - 1) CTAs + 1st longest: of so many, one CTA has k.  The last candidate cuts only
// the shortest items, as many as whole rounds of all CTAs leave over, into as many pieces as find a CTA then (8192 queries x 16 heads over 65536
// keys, 512 items: in turn on one card 3480 us whole, 3175 so; three sequences of up to 1500 queries behind up to 9000, whose items make no rounds: 141 and 152).
constexpr float PLAN_COST = 6.f;
constexpr int PLAN_THREADS = 1024, PLAN_CAND = 6, PLAN_BUCKETS = 1024, PLAN_KEPT = 1024, PLAN_TAIL = 256;
struct PlanItem { int b, i0, j0, j1, pos, n, row0, cut; };          // j1 < j0: queries that see nothing
__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(const PagedPrefillParams p, int ctas) {
  __shared__ PlanItem kept[PLAN_KEPT];
  __shared__ int hist[PLAN_BUCKETS];
  __shared__ unsigned long long sm_total;
  __shared__ int sm_longest, sm_shortest, sm_items, sm_slots, sm_cuts, sm_cut, sm_rounds, sm_full_rounds, sm_pieces[PLAN_CAND], sm_parts[PLAN_CAND], sm_L[PLAN_CAND], sm_tail, sm_tail_parts, warp_sums[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  hist[threadIdx.x] = 0;
  if (threadIdx.x == 0) { sm_total = 0; sm_longest = 0; sm_shortest = 1 << 30; sm_items = 0; sm_slots = 0; sm_cuts = 0; sm_rounds = 0; sm_full_rounds = 0; }
  if (threadIdx.x < PLAN_CAND) { sm_pieces[threadIdx.x] = 0; sm_parts[threadIdx.x] = 0; }
  grid_dep_launch();
  grid_dep_wait();
  __syncthreads();
  // every item, from the lengths: a warp a sequence, a lane an item
  auto count_off = [&](auto f) {
    for (int b = warp; b < p.c.n_seq; b += PLAN_THREADS / 32) {
      const SeqQueries s = seq_queries(p, b);
      if (s.refused && p.status && lane == 0) p.status[0] = DAISY_EINVAL;
      for (int i0 = lane * p.toks; i0 < s.n; i0 += 32 * p.toks) {
        PlanItem it{b, i0, 1, 0, -1, min(p.toks, s.n - i0), s.row0 + i0, 0};
        if (s.pos >= 0) { it.pos = s.pos + i0; it.j0 = first_tile(it.pos, p.window); it.j1 = last_tile(it.pos, it.n); }
        f(it);
      }
    }
  };
  {
    unsigned total = 0;
    int longest = 0, shortest = 1 << 30;
    count_off([&](const PlanItem& it) {
      const int at = atomicAdd(&sm_items, 1), t = it.j1 - it.j0 + 1;
      if (at < PLAN_KEPT) kept[at] = it;
      total += t;
      longest = max(longest, t);
      shortest = min(shortest, t);
    });
    total = __reduce_add_sync(0xffffffffu, total);
    longest = __reduce_max_sync(0xffffffffu, longest);
    shortest = __reduce_min_sync(0xffffffffu, shortest);
    if (lane == 0 && longest > 0) { atomicAdd(&sm_total, (unsigned long long)total); atomicMax(&sm_longest, longest); atomicMin(&sm_shortest, shortest); }
  }
  __syncthreads();
  const int n_items = sm_items;
  auto items = [&](auto f) {                                         // again: a thread an item where they were kept
    if (n_items <= PLAN_KEPT) { if ((int)threadIdx.x < n_items) f(kept[threadIdx.x]); }
    else count_off(f);
  };
  if (threadIdx.x < PLAN_CAND) {
    const int fit = n_items > 0 ? ctas / max(1, n_items * p.heads) : 1;
    const int n = threadIdx.x == 0 ? 1 : threadIdx.x == 1 ? max(1, fit) : threadIdx.x;             // whole; as many as find a CTA; 2, 3, 4; (the tail)
    sm_L[threadIdx.x] = max((sm_longest + n - 1) / n, min(4, max(sm_longest, 1)));
  }
  // Longer items than a kept one's, of equally long ones those in front (by place, not by the order of the list, which no two runs share: a
  // cut item is rounded otherwise than a whole one).
  int in_front = 0;
  if (p.slots > 0 && n_items <= PLAN_TAIL && n_items * p.heads > ctas && (int)threadIdx.x < n_items) {
    const PlanItem it = kept[threadIdx.x];
    for (int i = 0; i < n_items; ++i) {
      const PlanItem& o = kept[i];
      const int d = (o.j1 - o.j0) - (it.j1 - it.j0);
      in_front += d > 0 || (d == 0 && (o.b < it.b || (o.b == it.b && o.i0 < it.i0)));
    }
    for (int k = (in_front * p.heads + ctas - 1) / ctas; k * ctas < (in_front + 1) * p.heads; ++k) {
      atomicMax(&sm_rounds, (k + 1) * (it.j1 - it.j0 + 1));
      if ((k + 1) * ctas <= n_items * p.heads) atomicMax(&sm_full_rounds, (k + 1) * (it.j1 - it.j0 + 1));       // without the tail
    }
  }
  if (p.slots > 0) {
    __syncthreads();
    int pieces[PLAN_CAND] = {}, parts[PLAN_CAND] = {};
    items([&](const PlanItem& it) {
      const unsigned t = max(it.j1 - it.j0 + 1, 1);
#pragma unroll
      for (int k = 0; k < PLAN_CAND; ++k) {
        const int n = (int)((t + sm_L[k] - 1) / (unsigned)sm_L[k]);
        pieces[k] += n;
        if (n > 1) parts[k] += n;
      }
    });
#pragma unroll
    for (int k = 0; k < PLAN_CAND; ++k) {
      const int a = __reduce_add_sync(0xffffffffu, pieces[k]), e = __reduce_add_sync(0xffffffffu, parts[k]);
      if (lane == 0 && a) { atomicAdd(&sm_pieces[k], a); atomicAdd(&sm_parts[k], e); }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float best = 3.0e38f;
    int cut = sm_L[0];
    sm_tail = 0;
    const int whole = n_items * p.heads, over = whole % ctas;        // the host keeps them inside 32 bits
    const float share = (float)sm_total * p.heads / ctas, end = n_items > 0 ? 0.5f * ((float)sm_shortest + (float)sm_total / n_items) : 0.f;
    for (int k = 0; k < PLAN_CAND && p.slots > 0; ++k) {
      if (k == PLAN_CAND - 1) {                                      // the tail
        if (n_items > PLAN_TAIL || whole <= ctas || over == 0 || 2 * over > ctas || sm_longest > 2 * sm_shortest) continue;
        const int tail = (over + p.heads - 1) / p.heads, n = ctas / over;
        const int64_t parts = (int64_t)tail * p.heads * n;
        if (parts > p.slots || n_items + tail * (n - 1) > p.max_pieces) continue;
        const float est = fmaxf(share + 0.5f * end / n, (float)sm_full_rounds) + PLAN_COST * fmaxf(1.f, (float)parts / ctas);
        if (est < best) { best = est; cut = sm_longest; sm_tail = tail; sm_tail_parts = n; }
        continue;
      }
      const int64_t n = (int64_t)sm_pieces[k] * p.heads, parts = (int64_t)sm_parts[k] * p.heads;
      if (k > 0 && (parts > p.slots || sm_pieces[k] > p.max_pieces)) continue;
      const float est = (n <= ctas ? (float)sm_L[k] : fmaxf(share + 0.5f * fminf(end, (float)sm_L[k]), parts > 0 ? 0.f : (float)sm_rounds)) +
                        (parts > 0 ? PLAN_COST * fmaxf(1.f, (float)parts / ctas) : 0.f);
      if (est < best) { best = est; cut = sm_L[k]; }
    }
    sm_cut = max(cut, 1);
  }
  __syncthreads();
  const unsigned L = sm_cut;
  auto bucket = [](int t) { return PLAN_BUCKETS - 1 - min(t, PLAN_BUCKETS - 1); };                  // longest first
  // exclusive prefix sums of the buckets, a thread each -> the sum of all
  auto prefix = [&]() {
    __syncthreads();
    const int own = hist[threadIdx.x];
    int x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    const int sum = warp_sums[lane], before = __reduce_add_sync(0xffffffffu, lane < warp ? sum : 0), all = __reduce_add_sync(0xffffffffu, sum);
    hist[threadIdx.x] = before + x - own;
    __syncthreads();
    return all;
  };
  const int tail = sm_tail;                                          // the shortest items, of equally long ones the last
  if (tail > 0) {
    if ((int)threadIdx.x < n_items) kept[threadIdx.x].cut = in_front >= n_items - tail;
    __syncthreads();
  }
  // an item of t tiles goes in n pieces: t % n of them one tile longer than the others
  auto pieces_of = [&](const PlanItem& it, int t) {
    return tail > 0 ? (it.cut ? max(1, min(sm_tail_parts, t)) : 1) : max(1, (int)((t + L - 1) / L));
  };
  items([&](const PlanItem& it) {
    const int t = it.j1 - it.j0 + 1, n = pieces_of(it, t), rem = t % n;
    if (rem) atomicAdd(&hist[bucket(t / n + 1)], rem);
    atomicAdd(&hist[bucket(t / n)], n - rem);
  });
  const int n_pieces = prefix();
  if (threadIdx.x == 0) { p.head->n_pieces = min(n_pieces, p.max_pieces); p.head->queue = 0; }
  items([&](const PlanItem& it) {
    const int t = it.j1 - it.j0 + 1, n = pieces_of(it, t), rem = t % n, len = t / n;
    int slot = 0;
    if (n > 1) {
      slot = atomicAdd(&sm_slots, n * p.heads);
      p.cuts[atomicAdd(&sm_cuts, 1)] = Cut{it.b, it.i0, slot, n};
    }
    const int at_long = rem ? atomicAdd(&hist[bucket(len + 1)], rem) : 0, at_short = atomicAdd(&hist[bucket(len)], n - rem);
    auto put = [&](int i) {
      const int j = it.j0 + i * len + min(i, rem), at = i < rem ? at_long + i : at_short + i - rem;
      if (at < p.max_pieces) p.pieces[at] = Piece{it.b, it.i0, j, j + len - (i < rem ? 0 : 1), slot, i, n, it.pos, it.n, it.row0, {0, 0}};
    };
    for (int i = 0; i < n; ++i) put(i);
  });
  __syncthreads();
  if (threadIdx.x == 0) p.head->n_cuts = sm_cuts;
}

struct PagedItem {
  int b, h;                          // b < 0: no more; h counts packs of heads
  int q0[2], n[2], jlo_s[2], jhi_s[2];      // of each stream: first position, queries, key tiles
  bool valid[2];                     // has tiles in this piece
  int jlo, jhi;
  int see0, end;                     // keys see0 .. end - 1 are seen by some row of the item
  int row0, bq;                      // first row of stream 0: token and batch row of q and out
  int slot, parts, part;
};

struct PagedBarriers {
  uint64_t q_full[2][PP_NQBUF], q_empty[2][PP_NQBUF];
  uint64_t kv_full[PP_NSTAGE], kv_empty[PP_NSTAGE];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t l_full[2][4];             // the partial row sums of the two warps that share 32 rows of a stream
  uint64_t i_full[PP_NITEM], i_empty[PP_NITEM];
  PagedItem item[PP_NITEM];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(PagedBarriers) <= PP_BARS, "room for the barriers");

// NSPLIT = 2: bounded logits, two warps (64 columns each) for 32 rows; NSPLIT = 1: any logits, one warp.
template <int NSPLIT, bool F16>
__global__ void __launch_bounds__(32 * (8 * NSPLIT + 2), 1)
paged_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, const PagedPrefillParams p) {
  static_assert(!(F16 && NSPLIT == 2), "weights without a reference maximum do not fit float16");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_tiles = smem;
  uint8_t* kv_tiles = smem + 2 * PP_NQBUF * PP_TILE;
  PagedBarriers* bars = reinterpret_cast<PagedBarriers*>(smem + PP_SMEM_TILES);
  volatile int* abort_flag = &bars->abort_flag;
  constexpr int TMA_WARP = 8 * NSPLIT, MMA_WARP = 8 * NSPLIT + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      for (int qb = 0; qb < PP_NQBUF; ++qb) { mbar_init(&bars->q_full[s][qb], 1); mbar_init(&bars->q_empty[s][qb], 4 * NSPLIT); }
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->p_full[s], 128 * NSPLIT);
      mbar_init(&bars->o_full[s], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&bars->l_full[s][i], 2);
    }
    for (int i = 0; i < PP_NSTAGE; ++i) { mbar_init(&bars->kv_full[i], 1); mbar_init(&bars->kv_empty[i], 1); }
    for (int i = 0; i < PP_NITEM; ++i) { mbar_init(&bars->i_full[i], 1); mbar_init(&bars->i_empty[i], 8 * NSPLIT + 1); }
    bars->abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  grid_dep_launch();
  grid_dep_wait();

  auto next_item = [&](int rd) -> const PagedItem* {
    const PagedItem* g = &bars->item[rd % PP_NITEM];
    if (!__all_sync(0xffffffffu, mbar_wait(&bars->i_full[rd % PP_NITEM], (rd / PP_NITEM) & 1, abort_flag, p.status, 13))) return nullptr;
    return g->b >= 0 ? g : nullptr;
  };
  auto item_done = [&](int rd) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->i_empty[rd % PP_NITEM]);
  };

  if (warp == TMA_WARP) {
    // ------------------------------------------------------------------ TMA producer: the warp as one, lane 0 issues
    if (lane == 0) { prefetch_tmap(&tm_q); prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); prefetch_tmap(&tm_o); }
    // the plan's words come from L2: this grid was there before they were written
    int n_work = p.counted * p.c.n_seq * p.heads;                   // with a plan: known with the first piece
    // packed sequences without a plan, a lane each: queries, and items up to it and including it
    SeqQueries mine{0, 0, -1, false};
    int upto = 0;
    if (p.counted > 0 && p.cu) {
      if (lane < p.c.n_seq) mine = seq_queries(p, lane);
      if (mine.refused && p.status) p.status[0] = DAISY_EINVAL;
      upto = (mine.n + p.toks - 1) / p.toks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += y; }
      n_work = __shfl_sync(0xffffffffu, upto, 31) * p.heads;
    }
    const int ts = PP_BM >> p.lgp;                                  // queries of a stream
    const int lgr = min(p.c.lg, 7), boxes = PP_BN >> lgr;           // a tile is `boxes` boxes of 1 << lgr rows
    int n = 0;
    uint32_t qn[2] = {0, 0};
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, where)) != 0;
    };
    auto load_q = [&](const PagedItem& g) {
      for (int s = 0; s < 2 && ok; ++s) {
        if (!g.valid[s]) continue;
        const int qb = qn[s] % PP_NQBUF;
        if (!wait(&bars->q_empty[s][qb], ((qn[s] / PP_NQBUF) & 1) ^ 1, 9)) { ok = false; break; }
        ++qn[s];
        uint8_t* dst = q_tiles + (qb * 2 + s) * PP_TILE;
        if (lane == 0) {
          mbar_expect_tx(&bars->q_full[s][qb], PP_TILE);
          tma_load_4d(dst, &tm_q, &bars->q_full[s][qb], 0, g.h << p.lgp, g.row0 + s * ts, g.bq);
          tma_load_4d(dst + PP_HALF, &tm_q, &bars->q_full[s][qb], 64, g.h << p.lgp, g.row0 + s * ts, g.bq);
        }
      }
    };
    int drawn = blockIdx.x;                                         // the first one is this CTA's own number, later ones are drawn
    int4 px = make_int4(0, 0, 0, 0), py = px, pz = px;              // its piece
    auto fetch_piece = [&]() {
      if (p.counted > 0 || drawn / p.heads >= p.max_pieces) return;
      const int4* src = reinterpret_cast<const int4*>(p.pieces + drawn / p.heads);
      px = __ldcg(src); py = __ldcg(src + 1); pz = __ldcg(src + 2);
    };
    auto draw = [&]() {
      if (p.counted > 0) { drawn += gridDim.x; return; }
      int x = 0;
      if (lane == 0) x = atomicAdd(&p.head->queue, 1);
      drawn = (int)gridDim.x + __shfl_sync(0xffffffffu, x, 0);
      fetch_piece();
    };
    auto publish = [&](int rd, PagedItem& g) {
      const int slot = rd % PP_NITEM;
      g.b = -1;
      Piece pc;
      bool there = false;
      if (p.counted > 0) {                                           // a sequence's last queries first: they see most
        there = drawn < n_work;
        if (there && p.cu) {
          const int at = drawn / p.heads, b = __ffs(__ballot_sync(0xffffffffu, upto > at)) - 1;
          const int n = __shfl_sync(0xffffffffu, mine.n, b), pos = __shfl_sync(0xffffffffu, mine.pos, b), row0 = __shfl_sync(0xffffffffu, mine.row0, b);
          const int i0 = (__shfl_sync(0xffffffffu, upto, b) - 1 - at) * p.toks;
          pc = Piece{b, i0, 0, 1 << 30, 0, 0, 1, pos < 0 ? -1 : pos + i0, min(p.toks, n - i0), row0 + i0, {0, 0}};
        } else if (there) {
          const int at = drawn / p.heads, i = at / p.c.n_seq, i0 = (p.counted - 1 - i) * p.toks, b = at - i * p.c.n_seq;
          const SeqQueries sq = seq_queries(p, b);
          if (sq.refused && p.status && lane == 0) p.status[0] = DAISY_EINVAL;
          pc = Piece{b, i0, 0, 1 << 30, 0, 0, 1, sq.pos < 0 ? -1 : sq.pos + i0, min(p.toks, sq.n - i0), sq.row0 + i0, {0, 0}};
        }
      } else if (drawn / p.heads < p.max_pieces) {
        if (rd == 0) n_work = __ldcg(&p.head->n_pieces) * p.heads;
        there = drawn < n_work;
        pc = Piece{px.x, px.y, px.z, px.w, py.x, py.y, py.z, py.w, pz.x, pz.y, {0, 0}};
      }
      if (there) {
        g.b = pc.b; g.h = drawn % p.heads;
        g.bq = p.cu ? 0 : pc.b;
        g.row0 = pc.row0;
        g.slot = pc.slot + g.h * pc.parts; g.part = pc.part; g.parts = pc.parts;
        const int pos = pc.pos;
        g.jlo = 1 << 30; g.jhi = -1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          g.q0[s] = pos + s * ts;
          g.n[s] = min(max(pc.n - s * ts, 0), ts);
          g.jlo_s[s] = 1; g.jhi_s[s] = 0;
          if (g.n[s] > 0 && pos >= 0) {
            g.jlo_s[s] = max(first_tile(g.q0[s], p.window), pc.j0);
            g.jhi_s[s] = min(last_tile(g.q0[s], g.n[s]), pc.j1);
          }
          g.valid[s] = g.jhi_s[s] >= g.jlo_s[s];
          if (g.valid[s]) { g.jlo = min(g.jlo, g.jlo_s[s]); g.jhi = max(g.jhi, g.jhi_s[s]); }
        }
        g.see0 = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        g.end = pos + g.n[0] + g.n[1];
      }
      if (!wait(&bars->i_empty[slot], ((rd / PP_NITEM) & 1) ^ 1, 14)) { ok = false; return; }
      if (lane == 0) {
        bars->item[slot] = g;
        mbar_arrive(&bars->i_full[slot]);
      }
    };
    PagedItem g, g_next;
    fetch_piece();
    publish(0, g);
    if (ok && g.b >= 0) load_q(g);
    for (int rd = 0; ok && g.b >= 0; ++rd, g = g_next) {
      // the table's entries, a lane each, 32 at a time, the next 32 on their way
      const int* table = p.c.table + g.b * p.c.table_sb;
      const int e_first = g.see0 >> p.c.lg, e_last = (g.end - 1) >> p.c.lg, hk = (g.h << p.lgp) / p.G;
      auto entries = [&](int from) {
        const int i = from + lane;
        return i >= e_first && i <= e_last ? __ldcg(table + i) : 0;
      };
      int from = 0, cur = 0, ahead = 0;
      if (g.jhi >= g.jlo) { from = (g.jlo * PP_BN) >> p.c.lg; cur = entries(from); ahead = entries(from + 32); }
      bool next_out = false;
      // The next item is drawn two tiles before this one's last: what is drawn at the start goes to a CTA that may be the last to come to it (8192
      // queries x 16 heads over 65536 keys, in turn on one card: 3208 us drawn at the start, 3175 so; 32 over 8 heads, 4096 behind 8000: 564, 552)
      if (g.jhi < g.jlo) draw();
      for (int j = g.jlo; j <= g.jhi && ok; ++j) {
        if (j == max(g.jlo, g.jhi - 2)) draw();
        // a lane a box (32 is a multiple of the boxes of a tile); only those that hold a row somebody sees
        const int k0 = j * PP_BN, e_lo = k0 >> p.c.lg;
        if (e_lo >= from + 32) { from += 32; cur = ahead; ahead = entries(from + 32); }
        int pg = __shfl_sync(0xffffffffu, cur, e_lo - from + (lane & (boxes - 1)));
        const int b_first = max(g.see0 - k0, 0) >> lgr, b_last = (min(g.end - k0, PP_BN) - 1) >> lgr;
        const bool issues = lane >= b_first && lane <= b_last;
        if (issues && (unsigned)pg >= (unsigned)p.c.n_pages) {
          if (p.status) p.status[0] = DAISY_EINVAL;
          pg = 0;
        }
        const uint32_t bytes = (uint32_t)(b_last - b_first + 1) << (lgr + 8);
        const int in_page = k0 & ((1 << p.c.lg) - 1);                // of a page longer than a tile
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const int stage = n % PP_NSTAGE;
          if (!wait(&bars->kv_empty[stage], ((n / PP_NSTAGE) & 1) ^ 1, 1)) { ok = false; break; }
          if (lane == 0) mbar_expect_tx(&bars->kv_full[stage], bytes);
          __syncwarp();
          if (issues) {
            uint8_t* dst = kv_tiles + stage * PP_TILE + (lane << (lgr + 7));
            const CUtensorMap* tm = kv ? &tm_v : &tm_k;
            tma_load_4d(dst, tm, &bars->kv_full[stage], 0, in_page, hk, pg);
            tma_load_4d(dst + PP_HALF, tm, &bars->kv_full[stage], 64, in_page, hk, pg);
          }
          __syncwarp();
        }
        if (ok && j == g.jhi) {                                      // the next item's queries, when this one's last tiles are asked for
          publish(rd + 1, g_next);
          if (ok && g_next.b >= 0) load_q(g_next);
          next_out = true;
        }
      }
      if (ok && !next_out) {                                         // an item without tiles
        publish(rd + 1, g_next);
        if (ok && g_next.b >= 0) load_q(g_next);
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------------ MMA issuer.  Per tile: PV_0(j-1) QK_0(j) PV_1(j-1) QK_1(j)
    const uint32_t leader = elect_one() ? 1u : 0u;
    constexpr uint32_t idesc_qk = F16 ? umma_idesc_f16(PP_BM, PP_BN, 0, 0) : umma_idesc_bf16(PP_BM, PP_BN, 0, 0);
    constexpr uint32_t idesc_pv = F16 ? umma_idesc_f16(PP_BM, DAISY_HEAD_DIM, 0, 1) : umma_idesc_bf16(PP_BM, DAISY_HEAD_DIM, 0, 1);
    const uint64_t qd = umma_desc_sw128(smem_u32(q_tiles), 16, 1024);
    const uint64_t kd = umma_desc_sw128(smem_u32(kv_tiles), 16, 1024);
    const uint64_t vd = umma_desc_sw128(smem_u32(kv_tiles), PP_HALF, 1024);
    const uint32_t q_lo0 = (uint32_t)qd, k_lo0 = (uint32_t)kd, qk_hi = (uint32_t)(qd >> 32);
    const uint32_t v_lo0 = (uint32_t)vd, v_hi = (uint32_t)(vd >> 32);
    int n_base = 0;
    uint32_t n_pv[2] = {0, 0}, n_q[2] = {0, 0};
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, where)) != 0;
    };
    const PagedItem* item;
    for (int rd = 0; ok && (item = next_item(rd)); ++rd) {
      const PagedItem g = *item;
      if (g.jhi < g.jlo) { item_done(rd); continue; }
      for (int j = g.jlo; j <= g.jhi + 1 && ok; ++j) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!g.valid[s]) continue;
          const uint32_t s_tmem = tmem_base + s * 128, o_tmem = tmem_base + 256 + s * 128;
          if (j - 1 >= g.jlo_s[s] && j - 1 <= g.jhi_s[s]) {          // O_s += P_s(j-1) V_{j-1}
            const int n = n_base + 2 * (j - 1 - g.jlo) + 1, stage = n % PP_NSTAGE;
            const bool v_seen = s == 1 && g.valid[0] && j - 1 >= g.jlo_s[0] && j - 1 <= g.jhi_s[0];
            if (!v_seen) {                                           // V is there before the weights: what is to be cleared is cleared under the softmax
              if (!wait(&bars->kv_full[stage], (n / PP_NSTAGE) & 1, 3)) { ok = false; break; }
              const int k0 = (j - 1) * PP_BN, lo = max(g.see0 - k0, 0), hi = min(g.end - k0, PP_BN);
              if (lo > 0 || hi < PP_BN) {                            // rows that nobody sees
                uint8_t* tile = kv_tiles + stage * PP_TILE + (lane & 7) * 16;
                auto clear = [&](int r) {
                  *reinterpret_cast<uint4*>(tile + r * 128) = make_uint4(0, 0, 0, 0);
                  *reinterpret_cast<uint4*>(tile + PP_HALF + r * 128) = make_uint4(0, 0, 0, 0);
                };
                for (int r = lane >> 3; r < lo; r += 4) clear(r);
                for (int r = hi + (lane >> 3); r < PP_BN; r += 4) clear(r);
                fence_proxy_async();
                __syncwarp();
              }
            }
            if (!wait(&bars->p_full[s], n_pv[s] & 1, 2)) { ok = false; break; }
            ++n_pv[s];
            tc_fence_after();
            const uint32_t v_lo = v_lo0 + stage * (PP_TILE >> 4);
            umma_ts_lh_p(leader, o_tmem, s_tmem, v_lo, v_hi, idesc_pv, j - 1 == g.jlo_s[s] ? 0u : 1u);
#pragma unroll
            for (int k = 1; k < PP_BN / 16; ++k)
              umma_ts_lh_p(leader, o_tmem, s_tmem + (NSPLIT == 2 ? (k & 3) * 8 + (k >> 2) * 64 : k * 8), v_lo + k * (2048 >> 4), v_hi, idesc_pv, 1u);
            const bool other_uses = s == 0 && g.valid[1] && j - 1 >= g.jlo_s[1] && j - 1 <= g.jhi_s[1];
            if (!other_uses) tc_commit_p(leader, &bars->kv_empty[stage]);
            if (j - 1 == g.jhi_s[s]) tc_commit_p(leader, &bars->o_full[s]);
          }
          if (j >= g.jlo_s[s] && j <= g.jhi_s[s]) {                  // S_s = Q_s K_j^T
            const int n = n_base + 2 * (j - g.jlo), stage = n % PP_NSTAGE;
            if (j == g.jlo_s[s]) {
              const uint32_t qb = n_q[s] % PP_NQBUF;
              if (!wait(&bars->q_full[s][qb], (n_q[s] / PP_NQBUF) & 1, 4)) { ok = false; break; }
              ++n_q[s];
            }
            const bool k_seen = s == 1 && g.valid[0] && j >= g.jlo_s[0] && j <= g.jhi_s[0];
            if (!k_seen && !wait(&bars->kv_full[stage], (n / PP_NSTAGE) & 1, 5)) { ok = false; break; }
            tc_fence_after();
            const uint32_t q_buf = (n_q[s] - 1) % PP_NQBUF;
            const uint32_t q_lo = q_lo0 + (q_buf * 2 + s) * (PP_TILE >> 4), k_lo = k_lo0 + stage * (PP_TILE >> 4);
#pragma unroll
            for (int k = 0; k < DAISY_HEAD_DIM / 16; ++k) {
              const uint32_t off = ((k >> 2) * PP_HALF + (k & 3) * 32) >> 4;
              umma_ss_lh_p(leader, s_tmem, q_lo + off, qk_hi, k_lo + off, qk_hi, idesc_qk, k > 0 ? 1u : 0u);
            }
            tc_commit_p(leader, &bars->s_full[s]);
            const bool other_uses = s == 0 && g.valid[1] && j >= g.jlo_s[1] && j <= g.jhi_s[1];
            if (!other_uses) tc_commit_p(leader, &bars->kv_empty[stage]);
          }
        }
      }
      n_base += 2 * (g.jhi - g.jlo + 1);
      item_done(rd);                                                 // not before what was loaded from it has been used
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    constexpr int COLS = 128 / NSPLIT;                               // of the scores, and of the output in the epilogue
    const int grp = warp >> 2, quarter = warp & 3;
    const int s = NSPLIT == 2 ? grp & 1 : grp, half = NSPLIT == 2 ? grp >> 1 : 0;
    const int row = quarter * 32 + lane, ts = PP_BM >> p.lgp, pack1 = (1 << p.lgp) - 1;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem_base + lane_off + s * 128 + half * 64;
    const uint32_t o_tmem = tmem_base + lane_off + 256 + s * 128 + half * 64;
    const float c2 = p.scale_log2;
    uint32_t n_s = 0, n_o = 0;
    bool ok = true;
    const PagedItem* item;

    auto row_at = [&](const PagedItem* g, int r) {                   // row r of this stream: query r / pack, head r % pack
      return p.out + g->bq * p.o_sb + (int64_t)(g->row0 + s * ts + (r >> p.lgp)) * p.o_st + (int64_t)((g->h << p.lgp) + (r & pack1)) * p.o_sh;
    };
    // rows of this warp to the output, straight from registers
    auto store_row = [&](const PagedItem* g, const float* y) {       // y: COLS values of this lane's row
      if (row >= g->n[s] << p.lgp) return;
      __nv_bfloat16* dst = row_at(g, row) + half * 64;
#pragma unroll
      for (int c = 0; c < COLS; c += 8) *reinterpret_cast<uint4*>(dst + c) = pack8(y + c);
    };
    // this warp's sums of a piece, for the launch that joins them
    auto leave = [&](const PagedItem* g, const uint32_t* o, float m, float l) {
      if (row >= g->n[s] << p.lgp) return;
      float* dst = p.part + (int64_t)(g->slot + g->part) * PP_SLOT + ((s * NSPLIT + half) * 4 + quarter) * (COLS * 32 + 64) + lane;
      if (l != 0.f) {                                                // else the row sees none of the piece
#pragma unroll
        for (int c = 0; c < COLS; ++c) dst[c * 32] = __uint_as_float(o[c]);
      }
      dst[COLS * 32] = m;
      dst[COLS * 32 + 32] = l;
    };
    // rows of an item that this warp's stream has no tiles of
    auto without_tiles = [&](const PagedItem* g) {
      if (g->n[s] == 0) return;
      uint32_t zero[COLS];
      float none[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) { zero[c] = 0; none[c] = 0.f; }
      if (g->parts > 1) leave(g, zero, PP_NEG, 0.f);
      else store_row(g, none);
    };
    // the last step of an item: l, m of this lane's row, sums in O.  They leave through the item's Q buffer, which its last scores have left: a bulk
    // copy of a warp's 32 rows (read back and stored by rows 8192 queries x 16 heads took 233 us, window 512 61; so 227 and 57.5)
    auto finish = [&](const PagedItem* g, float m, float l, uint8_t* box) {
      uint32_t o[COLS];
#pragma unroll
      for (int c = 0; c < COLS; c += 32) tmem_ld32(o_tmem + c, o + c);
      tc_wait_ld();
      if (g->parts > 1) {
        leave(g, o, m, l);
        fence_proxy_async();                                         // the Q buffer, which held the row sums, is next written by a copy
      } else {
        const float inv = 1.0f / l;
        const int n_rows = (g->n[s] << p.lgp) - quarter * 32;
#pragma unroll
        for (int hc = 0; hc < COLS / 64; ++hc) {
          uint8_t* mine = box + hc * PP_HALF;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[hc * 64 + 8 * c + e]) * inv;
            *reinterpret_cast<uint4*>(mine + row * 128 + ((c ^ (row & 7)) << 4)) = pack8(y);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (n_rows >= 32) {
          if (lane == 0) {
#pragma unroll
            for (int hc = 0; hc < COLS / 64; ++hc)
              tma_store_4d(&tm_o, box + hc * PP_HALF + quarter * 4096, half * 64 + hc * 64, g->h << p.lgp, g->row0 + s * ts + quarter * (32 >> p.lgp), g->bq);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {                                                     // the end of a sequence: the rows behind it are another's
#pragma unroll
          for (int hc = 0; hc < COLS / 64; ++hc)
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3);
              if (r >= n_rows) break;
              *reinterpret_cast<uint4*>(row_at(g, quarter * 32 + r) + half * 64 + (lane & 7) * 8 + hc * 64) =
                  *reinterpret_cast<const uint4*>(box + hc * PP_HALF + (quarter * 32 + r) * 128 + (((lane & 7) ^ (r & 7)) << 4));
            }
          fence_proxy_async();                                       // as above
        }
      }
      // the next item's first product into O_s follows this warp's next weights, which follow these loads
      tc_fence_before();
      ++n_o;
    };
    // The item before has left its Q buffer: asked when the next one begins, two items before that buffer is wanted
    auto buffer_free = [&]() {
      __syncwarp();
      if (lane == 0 && n_o > 0) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        mbar_arrive(&bars->q_empty[s][(n_o - 1) % PP_NQBUF]);
      }
    };

    for (int rd = 0; ok && (item = next_item(rd)); item_done(rd), ++rd) {
      const int q0 = item->q0[s], jlo = item->jlo_s[s], jhi = item->jhi_s[s];
      if (jhi < jlo) { without_tiles(item); continue; }
      buffer_free();
      const int q_row = q0 + (row >> p.lgp);
      uint8_t* q_buf = q_tiles + ((n_o % PP_NQBUF) * 2 + s) * PP_TILE;
      auto scores_there = [&]() -> bool {
        const bool there = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[s], n_s & 1, abort_flag, p.status, 6));
        ++n_s;
        tc_fence_after();
        return there;
      };
      auto weights_done = [&]() {
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&bars->p_full[s]);
      };
      // whole tiles: all rows of the stream see all of their keys
      const int f_lo = p.window > 0 ? max(q0 + ts + PP_BN - 1 - p.window, 0) / PP_BN : 0, f_hi = (q0 + 1) / PP_BN - 1;
      if constexpr (NSPLIT == 2) {
        const uint64_t c2p = pack2f(c2, c2);
        uint64_t sum_a = pack2f(0.f, 0.f), sum_b = sum_a;
        auto rebuild = [&](uint32_t (&r)[64], int c) {               // weights of 32 columns and their share of the row sums
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            if (c == 0 && i == 16) tmem_ld32(s_tmem + 32, r + 32);   // the other half of the scores, under this one
            const uint64_t xa = fmul2(pack2f(__uint_as_float(r[32 * c + i]), __uint_as_float(r[32 * c + i + 1])), c2p);
            const uint64_t xb = fmul2(pack2f(__uint_as_float(r[32 * c + i + 2]), __uint_as_float(r[32 * c + i + 3])), c2p);
            float x0, x1, p2, p3;
            unpack2f(xa, x0, x1);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            uint64_t pb;
            if (i & 4) {                                             // one pair in four goes to the FMA pipes
              pb = exp2_poly2(xb);
              unpack2f(pb, p2, p3);
            } else {
              float x2, x3;
              unpack2f(xb, x2, x3);
              p2 = fast_exp2(x2); p3 = fast_exp2(x3);
              pb = pack2f(p2, p3);
            }
            sum_a = fadd2(sum_a, pack2f(p0, p1));
            sum_b = fadd2(sum_b, pb);
            pk[i >> 1] = pack_bf16(p0, p1);
            pk[(i >> 1) + 1] = pack_bf16(p2, p3);
          }
          tmem_st16(s_tmem + 16 * c, pk);
          if (c == 0) tc_wait_ld();
        };
        for (int j = jlo; ok && j <= jhi;) {
          if (j >= f_lo && j <= f_hi) {
            int run = min(f_hi, jhi) + 1 - j;
            j += run;
            for (; run > 0; --run) {
              ok = scores_there();
              if (!ok) break;
              uint32_t r[64];
              tmem_ld32(s_tmem, r);
              tc_wait_ld();
              rebuild(r, 0);
              rebuild(r, 1);
              weights_done();
            }
            if (!ok) break;
          } else {
            ok = scores_there();
            if (!ok) break;
            uint32_t r[64];
            tmem_ld32(s_tmem, r);
            tc_wait_ld();
            const int hi = q_row - (j * PP_BN + half * 64), lo = p.window > 0 ? hi - p.window : -1;      // column i is visible iff lo < i <= hi
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (!__any_sync(0xffffffffu, hi >= 32 * c && lo < 32 * c + 31)) {
                const uint32_t zero[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                if (c == 0) tmem_ld32(s_tmem + 32, r + 32);
                tmem_st16(s_tmem + 16 * c, zero);
                if (c == 0) tc_wait_ld();
                continue;
              }
              if (!__all_sync(0xffffffffu, hi >= 32 * c + 31 && lo < 32 * c)) {
                const int b_lo = min(max(lo + 1 - 32 * c, 0), 32), b_hi = min(max(hi + 1 - 32 * c, 0), 32);
                const uint32_t visible = (uint32_t)(((uint64_t)1 << b_hi) - 1) & ~(uint32_t)(((uint64_t)1 << b_lo) - 1);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!((visible >> i) & 1u)) r[32 * c + i] = 0xff800000u;      // -inf -> weight 0
              }
              rebuild(r, c);
            }
            weights_done();
            ++j;
          }
        }
        if (!ok) break;
        float a0, a1, b0, b1;
        unpack2f(sum_a, a0, a1);
        unpack2f(sum_b, b0, b1);
        float l = (a0 + a1) + (b0 + b1);
        // the two warps that share rows exchange their sums through the item's Q buffer, each into the rows that the other's output will take
        *reinterpret_cast<float*>(q_buf + (1 - half) * PP_HALF + row * 128 + lane * 4) = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->l_full[s][quarter]);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->l_full[s][quarter], n_o & 1, abort_flag, p.status, 15));
        if (!ok) break;
        l += *reinterpret_cast<const float*>(q_buf + half * PP_HALF + row * 128 + lane * 4);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[s], n_o & 1, abort_flag, p.status, 7));
        if (!ok) break;
        tc_fence_after();
        __syncwarp();                                                // all lanes have their sums before the rows are overwritten
        finish(item, 0.f, l, q_buf + half * PP_HALF);
      } else {
        float m_ref = PP_NEG, l = 0.f;
        uint32_t r[128];
        for (int j = jlo; j <= jhi; ++j) {
          ok = scores_there();
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < 128; c += 32) tmem_ld32(s_tmem + c, r + c);
          tc_wait_ld();
          if (j < f_lo || j > f_hi) {
            const int hi = q_row - j * PP_BN, lo = p.window > 0 ? hi - p.window : -1;
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (!(i > lo && i <= hi)) r[i] = 0xff800000u;          // -inf
          }
          // the reference follows the row's maximum only when that has grown by more than 8: weights stay below 2^8 (float16: 2^15, WEIGHT_ROOM)
          float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            m0 = fmax3(m0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            m1 = fmax3(m1, __uint_as_float(r[32 + i]), __uint_as_float(r[33 + i]));
            m2 = fmax3(m2, __uint_as_float(r[64 + i]), __uint_as_float(r[65 + i]));
            m3 = fmax3(m3, __uint_as_float(r[96 + i]), __uint_as_float(r[97 + i]));
          }
          const float m_tgt = fmaxf(m_ref, fmaf(fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), c2, -WEIGHT_ROOM<F16>));
          if (j == jlo) {
            m_ref = m_tgt;
          } else if (__any_sync(0xffffffffu, m_tgt - m_ref > 8.0f)) {
            const float alpha = fast_exp2(m_ref - m_tgt);
            m_ref = m_tgt;
            l *= alpha;
            uint32_t t16[16];
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              tmem_ld16(o_tmem + 16 * c, t16);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) t16[i] = __float_as_uint(__uint_as_float(t16[i]) * alpha);
              tmem_st16(o_tmem + 16 * c, t16);
            }
          }
          const uint64_t c2p = pack2f(c2, c2), nm = pack2f(-m_ref, -m_ref);
          uint64_t sum_a = pack2f(0.f, 0.f), sum_b = sum_a;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float x0, x1, x2, x3;
              unpack2f(ffma2(pack2f(__uint_as_float(r[32 * c + i]), __uint_as_float(r[32 * c + i + 1])), c2p, nm), x0, x1);
              unpack2f(ffma2(pack2f(__uint_as_float(r[32 * c + i + 2]), __uint_as_float(r[32 * c + i + 3])), c2p, nm), x2, x3);
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1), p2 = fast_exp2(x2), p3 = fast_exp2(x3);
              sum_a = fadd2(sum_a, pack2f(p0, p1));
              sum_b = fadd2(sum_b, pack2f(p2, p3));
              pk[i >> 1] = pack16<F16>(p0, p1);
              pk[(i >> 1) + 1] = pack16<F16>(p2, p3);
            }
            tmem_st16(s_tmem + 16 * c, pk);
          }
          float a0, a1, b0, b1;
          unpack2f(sum_a, a0, a1);
          unpack2f(sum_b, b0, b1);
          l += (a0 + a1) + (b0 + b1);
          weights_done();
        }
        if (!ok) break;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_full[s], n_o & 1, abort_flag, p.status, 7));
        if (!ok) break;
        tc_fence_after();
        finish(item, m_ref, l, q_buf);
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// The pieces of cut items joined in their order.  A warp takes 32 rows and 16 of their columns, a lane a row, four pieces' sums in flight.
template <int NSPLIT>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedPrefillParams p) {
  constexpr int COLS = 128 / NSPLIT, SHARE = COLS * 32 + 64, CHUNK = 16;
  const int lane = threadIdx.x & 31;
  grid_dep_launch();
  grid_dep_wait();
  const int ts = PP_BM >> p.lgp;
  const int64_t n_work = (int64_t)__ldcg(&p.head->n_cuts) * p.heads * (8 * NSPLIT) * (COLS / CHUNK);
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < n_work; w += (int64_t)gridDim.x * 8) {
    const int chunk = (int)(w % (COLS / CHUNK)), place = (int)(w / (COLS / CHUNK) % (8 * NSPLIT));
    const int64_t item = w / (COLS / CHUNK) / (8 * NSPLIT);
    const int h = (int)(item % p.heads);
    const int4 c4 = __ldcg(reinterpret_cast<const int4*>(p.cuts + item / p.heads));
    const Cut cut{c4.x, c4.y, c4.z, c4.w};
    const int s = place / (4 * NSPLIT), half = place / 4 % NSPLIT, quarter = place % 4, row = quarter * 32 + lane;
    const SeqQueries sq = seq_queries(p, cut.b);
    const int rows = min(max(min(p.toks, sq.n - cut.i0) - s * ts, 0), ts) << p.lgp;
    if (row >= rows) continue;
    const float* base = p.part + (int64_t)(cut.slot + h * cut.parts) * PP_SLOT + place * SHARE + lane;
    float M = PP_NEG, den = 0.f, y[CHUNK];
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) y[c] = 0.f;
    if (NSPLIT == 1)                                                 // with bounded logits all references are zero
      for (int i = 0; i < cut.parts; ++i)
        if (__ldcg(base + (int64_t)i * PP_SLOT + COLS * 32 + 32) != 0.f) M = fmaxf(M, __ldcg(base + (int64_t)i * PP_SLOT + COLS * 32));
    for (int i0 = 0; i0 < cut.parts; i0 += 4) {
      float x[4][CHUNK], l[4], m[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float* src = base + (int64_t)min(i0 + k, cut.parts - 1) * PP_SLOT;
#pragma unroll
        for (int c = 0; c < CHUNK; ++c) x[k][c] = __ldcg(src + (chunk * CHUNK + c) * 32);
        m[k] = __ldcg(src + COLS * 32);
        l[k] = __ldcg(src + COLS * 32 + 32);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k < cut.parts && l[k] != 0.f) {
          const float e = NSPLIT == 1 ? fast_exp2(m[k] - M) : 1.f;
          den = fmaf(l[k], e, den);
#pragma unroll
          for (int c = 0; c < CHUNK; ++c) y[c] = fmaf(x[k][c], e, y[c]);
        }
    }
    const float inv = 1.0f / den;
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) y[c] *= inv;
    const int bq = p.cu ? 0 : cut.b, tok = sq.row0 + cut.i0 + s * ts + (row >> p.lgp), head = (h << p.lgp) + (row & ((1 << p.lgp) - 1));
    __nv_bfloat16* dst = p.out + bq * p.o_sb + (int64_t)tok * p.o_st + (int64_t)head * p.o_sh + half * 64 + chunk * CHUNK;
    *reinterpret_cast<uint4*>(dst) = pack8(y);
    *reinterpret_cast<uint4*>(dst + 8) = pack8(y + 8);
  }
}

}  // namespace daisy

using namespace daisy;

// Queries [B,T,H,D] as (d, h, t, b) with byte strides: a box of `heads` heads and `queries` queries is 128 rows of 64 channels, heads fastest;
// 128-byte swizzle, zero fill out of bounds.
static int make_tmap_packed_rows(CUtensorMap* m, const void* base, uint64_t D, uint64_t H, uint64_t T, uint64_t B, uint64_t sh, uint64_t st, uint64_t sb,
                                 uint32_t heads, uint32_t queries) {
  daisy_host::EncodeTiledFn enc = daisy_host::get_encode_tiled();
  if (!enc) return DAISY_ECUDA;
  cuuint64_t dims[4] = {D, H, T, B}, strides[3] = {sh, st, sb};
  cuuint32_t box[4] = {64, heads, queries, 1}, estr[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? DAISY_OK : DAISY_ECUDA;
}

static int paged_prefill_smem() {
  static bool done[daisy_host::MAX_DEVICES] = {};             // the attribute is per device
  const int dev = daisy_host::device_slot();
  if (dev < 0) return DAISY_ENODEV;
  if (done[dev]) return DAISY_OK;
  const auto allow = [](auto kernel) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PP_SMEM) == cudaSuccess; };
  if (!allow(paged_prefill_kernel<2, false>) || !allow(paged_prefill_kernel<1, false>) || !allow(paged_prefill_kernel<1, true>)) return DAISY_ECUDA;
  done[dev] = true;
  return DAISY_OK;
}

// Workspace: the plan's head, pieces and sums.
constexpr int PP_SLOTS_PER_SM = 4;
struct PrefillRoom { int slots; int64_t max_pieces; size_t pieces, cuts, part, end; };
static PrefillRoom prefill_room(int sms, int64_t tokens, int n_seq, int toks) {
  PrefillRoom r;
  r.slots = sms * PP_SLOTS_PER_SM;
  // items, and the further pieces of those that are cut
  r.max_pieces = tokens / toks + n_seq + r.slots;
  r.pieces = 256;
  r.cuts = r.pieces + ((size_t)r.max_pieces * sizeof(Piece) + 255) / 256 * 256;
  r.part = r.cuts + ((size_t)r.slots * sizeof(Cut) + 255) / 256 * 256;
  r.end = r.part + (size_t)r.slots * PP_SLOT * sizeof(float);
  return r;
}
// query heads of a key head that lie in one item's rows: the largest power of two, 16 at most, that divides the group
static int prefill_lgp(int G) {
  int l = 0;
  while (l < 4 && G % (2 << l) == 0) ++l;
  return l;
}
// Queries of an item: 256 rows, or 128 where all items of that size find an SM and no item is long (`longest`: key tiles that the table or
// the window leaves).  A tile takes one stream as long as two (1.7 us), so that the second one costs only where it adds tiles: 128 queries of
// 8 heads over one key head and 131000 keys 102 us with items of 128 rows, 69 with 256.
constexpr int64_t PP_SHORT = 16;
static int prefill_toks(int sms, int64_t tokens, int n_seq, int Hq, int lgp, int64_t longest) {
  const int solo = PP_BM >> lgp;
  return longest <= PP_SHORT && (tokens / solo + n_seq) * (Hq >> lgp) <= sms ? solo : 2 * solo;
}

extern "C" size_t daisy_b200_paged_attend_workspace_bytes(int B, int T, int n_seq, int Hq, int H) {
  if (B <= 0 || T <= 0 || n_seq <= 0 || Hq <= 0 || H <= 0 || Hq % H) return 0;
  int sms = daisy_host::sm_count_cached();
  if (sms <= 0) sms = daisy_host::MAX_SMS;
  const int lgp = prefill_lgp(Hq / H);
  return prefill_room(sms, (int64_t)B * T, n_seq, PP_BM >> lgp).end;                       // room for the smaller items
}

extern "C" int daisy_b200_paged_attend(const daisy_b200_pages* cache, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                       const int32_t* lens, const int32_t* cu, int window,
                                       void* out, int64_t o_sb, int64_t o_st, int64_t o_sh,
                                       int B, int T, int Hq, int D, float scale, unsigned flags,
                                       void* workspace, size_t workspace_bytes, int* status_word, void* stream) {
  PagedPrefillParams p = {};
  if (const int rc = daisy_host::paged_cache(cache, D, &p.c); rc != DAISY_OK) return rc;
  if (!q || !lens || !out || !workspace || B <= 0 || T <= 0 || Hq <= 0 || Hq % cache->H || !(scale > 0.f)) return DAISY_EINVAL;
  if (flags & ~(DAISY_BOUNDED_QK | DAISY_CACHE_FP16)) return DAISY_EINVAL;
  if (B != (cu ? 1 : cache->n_seq)) return DAISY_EINVAL;
  if (!daisy_aligned16(q) || !daisy_aligned16(out) || ((q_sb | q_st | q_sh | o_sb | o_st | o_sh) & 7) || (reinterpret_cast<uintptr_t>(lens) & 3) ||
      (reinterpret_cast<uintptr_t>(cu) & 3) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return DAISY_EALIGN;
  // a zero stride on a dimension longer than 1 is a broadcast view, which the tile copies cannot express
  if ((T > 1 && (q_st <= 0 || o_st <= 0)) || (Hq > 1 && (q_sh <= 0 || o_sh <= 0)) || (B > 1 && (q_sb <= 0 || o_sb <= 0))) return DAISY_EINVAL;
  const int sms = daisy_host::sm_count_cached();
  if (sms <= 0) return DAISY_ENODEV;
  const int64_t tokens = (int64_t)B * T;
  p.G = Hq / cache->H;
  p.lgp = prefill_lgp(p.G);
  p.heads = Hq >> p.lgp;
  p.window = daisy_host::paged_window(cache, window);
  int64_t longest = ((int64_t)cache->width * cache->page + PP_BN - 1) / PP_BN;
  if (p.window > 0) longest = std::min<int64_t>(longest, ((int64_t)p.window + (2 * PP_BM >> p.lgp)) / PP_BN + 2);
  p.toks = prefill_toks(sms, tokens, cache->n_seq, Hq, p.lgp, longest);
  const PrefillRoom room = prefill_room(sms, tokens, cache->n_seq, p.toks);
  if (workspace_bytes < room.end) return DAISY_EWORKSPACE;
  if ((room.max_pieces + 1) * Hq >= ((int64_t)1 << 31) - 4096) return DAISY_EUNSUPPORTED;
  if (const int rc = paged_prefill_smem(); rc != DAISY_OK) { (void)cudaGetLastError(); return rc; }
  CUtensorMap tq, tk, tv, to;
  auto sb = [](int64_t s, int64_t n) { return (uint64_t)(n == 1 ? 16 : s * 2); };
  int rc;
  const uint32_t box = (uint32_t)(cache->page < PP_BN ? cache->page : PP_BN);
  if ((rc = make_tmap_packed_rows(&tq, q, D, Hq, T, B, sb(q_sh, Hq), sb(q_st, T), sb(q_sb, B), 1u << p.lgp, (uint32_t)(PP_BM >> p.lgp))) != DAISY_OK) return rc;
  if ((rc = make_tmap_packed_rows(&to, out, D, Hq, T, B, sb(o_sh, Hq), sb(o_st, T), sb(o_sb, B), 1u << p.lgp, 32u >> p.lgp)) != DAISY_OK) return rc;       // a warp's rows
  if ((rc = daisy_host::make_tmap_bf16_dthb(&tk, cache->k, D, cache->page, cache->H, cache->n_pages, cache->p_sr * 2, sb(cache->p_sh, cache->H),
                                            sb(cache->p_sb, cache->n_pages), 64, box)) != DAISY_OK) return rc;
  if ((rc = daisy_host::make_tmap_bf16_dthb(&tv, cache->v, D, cache->page, cache->H, cache->n_pages, cache->p_sr * 2, sb(cache->p_sh, cache->H),
                                            sb(cache->p_sb, cache->n_pages), 64, box)) != DAISY_OK) return rc;
  p.out = (__nv_bfloat16*)out; p.o_sb = o_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.lens = lens; p.cu = cu;
  p.T = T; p.Hq = Hq;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = status_word;
  char* ws = (char*)workspace;
  p.head = (PlanHead*)ws;
  p.pieces = (Piece*)(ws + room.pieces);
  p.cuts = (Cut*)(ws + room.cuts);
  p.part = (float*)(ws + room.part);
  p.slots = room.slots; p.max_pieces = (int)room.max_pieces;
  cudaStream_t st = (cudaStream_t)stream;
  const bool f16 = (flags & DAISY_CACHE_FP16) != 0;
  // weights without a reference maximum reach 2^60, which float16 does not hold
  const bool bounded = (flags & DAISY_BOUNDED_QK) && !f16 && scale * 1.4426950408889634f * (float)D <= 60.f;
  // No plan where tables, or windows, are too short for items of uneven length, and the items can be counted off: as many for every sequence (131
  // tokens x 6 heads 17.5 us with a plan, 9.9 without), or those of up to 32 in at most two items a SM (five of 20 to 200 tokens x 16 heads 18 and
  // 10, of 90 to 900 31 and 21).  With more, the plan's order by length is worth its launch (nine of up to 1800 71 and 94)
  const int64_t per_seq = (T + p.toks - 1) / p.toks, items = (cu ? tokens / p.toks + cache->n_seq : per_seq * cache->n_seq) * p.heads;
  if (longest <= PP_SHORT && (!cu || (cache->n_seq <= 32 && items <= 2 * (int64_t)sms))) p.counted = cu ? 1 : (int)per_seq;
  // Cutting pays where items are fewer than four a SM
  if (tokens / p.toks * p.heads >= 4 * (int64_t)sms) p.slots = 0;
  cudaError_t e = cudaSuccess;
  if (!p.counted) e = daisy_host::launch_dependent(paged_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, p, sms);
  const dim3 grid((unsigned)(p.counted ? std::min<int64_t>(items, sms) : sms));
  if (e == cudaSuccess) {
    if (bounded)  e = daisy_host::launch_dependent(paged_prefill_kernel<2, false>, grid, dim3(576), PP_SMEM, st, tq, tk, tv, to, p);
    else if (f16) e = daisy_host::launch_dependent(paged_prefill_kernel<1, true>, grid, dim3(320), PP_SMEM, st, tq, tk, tv, to, p);
    else          e = daisy_host::launch_dependent(paged_prefill_kernel<1, false>, grid, dim3(320), PP_SMEM, st, tq, tk, tv, to, p);
  }
  if (e == cudaSuccess && !p.counted && p.slots > 0)
    e = bounded ? daisy_host::launch_dependent(paged_join_kernel<2>, dim3(sms * 4), dim3(256), 0, st, p) : daisy_host::launch_dependent(paged_join_kernel<1>, dim3(sms * 4), dim3(256), 0, st, p);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return DAISY_ECUDA; }
  DAISY_CHECK_LAUNCH();
  return DAISY_OK;
}
