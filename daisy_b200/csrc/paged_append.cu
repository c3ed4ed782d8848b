// Keys and values of new tokens into a paged cache, RMS-normalised and rotated on the way; their queries beside them.
//
// A streaming pass: 256 bytes read and 256 written for every row (token, head) of q, k and v, bound by HBM for prompts
// and by the chain start -> position -> page -> row for a few tokens.  A warp takes a token, or a share of one where tokens are few:
// position, page and the lane's piece of the rotation are fetched once and serve all its heads.  Eight lanes a row, 16 bytes of each
// half a lane: the two halves that the rotation pairs lie in one thread.
#include "paged.cuh"

namespace daisy {

struct AppendParams {
  PagedCache c;
  const __nv_bfloat16 *k, *v, *q, *ve;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh, q_sb, q_st, q_sh, ve_sb, ve_st, ve_sh;
  uint4* q_out;
  const int *start, *cu;
  const float *cos, *sin, *ve_gate;
  int table_rows, T, Hq, tokens, split;                             // Hq = 0: no queries; split: warps a token
  float eps;
  unsigned flags;
  int* status;
  bool streams;                      // more is written than L2 keeps
};

// Rows that a group of eight lanes keeps in flight, warps a block, blocks a SM.  8 x 8192 tokens, 48 rows a token: 272-293 us from card to card
// (5.5-5.9 TB/s; 4 rows, blocks of 8 warps, 2 a SM took a tenth more), 3765 packed tokens 22-24.5 us (a quarter more with blocks of 8 warps, 3 a SM: two uneven
// waves), 64 single tokens 2.6 us, launch and the chain of four loads.
constexpr int APPEND_ROWS = 2;
constexpr int APPEND_WARPS = 2;
constexpr int APPEND_BLOCKS = 16;

template <bool F16>
__global__ void __launch_bounds__(32 * APPEND_WARPS, APPEND_BLOCKS) paged_append_kernel(const AppendParams p) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, sub = lane & 7, group = lane >> 3;
  const int w = blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);
  const int tok = w / p.split, part = w - tok * p.split;
  if (tok >= p.tokens) return;
  const int per_tok = p.Hq + 2 * p.c.H, step = 4 * p.split;
  int b, t = tok;                                                    // sequence; the token's place in its row of q, k, v
  int64_t bt = 0, pos;
  if (p.cu) {
    b = find_seq(p.cu, p.c.n_seq, tok, lane);
    if (b < 0 || tok >= __ldcg(p.cu + b + 1)) return;                // in front of the first sequence or behind the last
    pos = (int64_t)tok - __ldcg(p.cu + b);
  } else {
    b = tok / p.T;
    t = tok - b * p.T;
    bt = b;
    pos = t;
  }
  // the first rows are asked for while the position is on its way
  uint4 lo[APPEND_ROWS], hi[APPEND_ROWS];
  auto source = [&](int h) {
    return h < p.Hq ? p.q + bt * p.q_sb + (int64_t)t * p.q_st + h * p.q_sh
         : h < p.Hq + p.c.H ? p.k + bt * p.k_sb + (int64_t)t * p.k_st + (h - p.Hq) * p.k_sh
                            : p.v + bt * p.v_sb + (int64_t)t * p.v_st + (h - p.Hq - p.c.H) * p.v_sh;
  };
  auto fetch = [&](int h0) {
#pragma unroll
    for (int u = 0; u < APPEND_ROWS; ++u) {
      const int h = h0 + u * step;
      if (h >= per_tok) { lo[u] = hi[u] = make_uint4(0, 0, 0, 0); continue; }
      const __nv_bfloat16* src = source(h) + 8 * sub;
      lo[u] = ld_stream16(src);
      hi[u] = ld_stream16(src + 64);
    }
  };
  const int first = __ldcg(p.start + b);
  int h0 = part * 4 + group;
  fetch(h0);
  pos += first;
  if (first < 0) return;                                             // idle
  if (pos < 0 || pos >= p.c.capacity() || ((p.flags & DAISY_ROPE) && pos >= p.table_rows)) {
    if (p.status && lane == 0) p.status[0] = DAISY_EINVAL;
    for (int h = h0; h < p.Hq; h += step) {                          // its queries read as zeros: nothing is left undefined
      uint4* dst = p.q_out + ((int64_t)tok * p.Hq + h) * 16 + sub;
      dst[0] = dst[8] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int pg = __ldcg(p.c.table + b * p.c.table_sb + (pos >> p.c.lg));
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { c[e] = 1.f; s[e] = 0.f; }
  if (p.flags & DAISY_ROPE) {
    const float4* cr = reinterpret_cast<const float4*>(p.cos + pos * 64 + 8 * sub);
    const float4* sr = reinterpret_cast<const float4*>(p.sin + pos * 64 + 8 * sub);
    const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
    c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
    s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
  }
  const bool stored = (unsigned)pg < (unsigned)p.c.n_pages;          // a page outside the pool: the queries alone
  if (!stored && p.status && lane == 0) p.status[0] = DAISY_EINVAL;
  // what does not stay in L2 until it is read shall not drive other lines out (8 x 8192 tokens 293 -> 275 us)
  auto store = [&](uint4* dst, const uint4& y) { if (p.streams) __stcs(dst, y); else *dst = y; };
  const float gate = p.ve ? 1.0f / (1.0f + __expf(-*p.ve_gate)) : 1.f;

  for (int base = part * 4; base < per_tok; base += APPEND_ROWS * step, h0 += APPEND_ROWS * step) {
    if (base != part * 4) fetch(h0);
#pragma unroll
    for (int u = 0; u < APPEND_ROWS; ++u) {
      const int h = h0 + u * step;
      if (base + u * step >= per_tok) break;                         // the whole warp's
      const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.c.H;
      float x1[8], x2[8];
      unpack8(lo[u], x1);
      unpack8(hi[u], x2);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x1[e] * x1[e] + x2[e] * x2[e];
      ss += __shfl_xor_sync(0xffffffffu, ss, 4);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      if (h < per_tok) {
        if (p.flags & (is_q ? DAISY_NORM_Q : is_v ? DAISY_NORM_V : DAISY_NORM_K)) {
          const float r = rsqrtf(ss * (1.0f / DAISY_HEAD_DIM) + p.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) { x1[e] *= r; x2[e] *= r; }
        }
        if (!is_v) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = x1[e], d = x2[e];
            x1[e] = a * c[e] + d * s[e];
            x2[e] = d * c[e] - a * s[e];
          }
        } else if (p.ve) {
          const __nv_bfloat16* m = p.ve + bt * p.ve_sb + (int64_t)t * p.ve_st + (h - p.Hq - p.c.H) * p.ve_sh + 8 * sub;
          float m1[8], m2[8];
          unpack8(ld_stream16(m), m1);
          unpack8(ld_stream16(m + 64), m2);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x1[e] = gate * x1[e] + (1.0f - gate) * m1[e];
            x2[e] = gate * x2[e] + (1.0f - gate) * m2[e];
          }
        }
        const uint4 y1 = pack8_16<F16>(x1), y2 = pack8_16<F16>(x2);
        if (is_q) {
          uint4* dst = p.q_out + ((int64_t)tok * p.Hq + h) * 16 + sub;
          store(dst, y1);
          store(dst + 8, y2);
        } else if (stored) {
          char* dst = (is_v ? p.c.v : p.c.k) + p.c.at(pg, is_v ? h - p.Hq - p.c.H : h - p.Hq, (int)pos) + 16 * sub;
          store(reinterpret_cast<uint4*>(dst), y1);
          store(reinterpret_cast<uint4*>(dst + 128), y2);
        }
      }
    }
  }
}

}  // namespace daisy

using namespace daisy;

extern "C" int daisy_b200_paged_append(const daisy_b200_pages* cache, const void* k, const void* v, const void* q,
                                       int64_t k_sb, int64_t k_st, int64_t k_sh, int64_t v_sb, int64_t v_st, int64_t v_sh,
                                       int64_t q_sb, int64_t q_st, int64_t q_sh, void* q_out,
                                       const int32_t* start, const int32_t* cu, const float* cos, const float* sin, int table_rows,
                                       const void* ve, int64_t ve_sb, int64_t ve_st, int64_t ve_sh, const float* ve_gate_logit,
                                       int B, int T, int Hq, int D, float eps, unsigned flags, int* status_word, void* stream) {
  AppendParams p = {};
  if (const int rc = daisy_host::paged_cache(cache, D, &p.c); rc != DAISY_OK) return rc;
  if (!k || !v || !start || (q != nullptr) != (q_out != nullptr) || B <= 0 || T <= 0 || (q && Hq <= 0)) return DAISY_EINVAL;
  if (flags & ~(DAISY_QKV_DEFAULT | DAISY_CACHE_FP16)) return DAISY_EINVAL;
  if (B != (cu ? 1 : cache->n_seq)) return DAISY_EINVAL;
  if ((flags & DAISY_ROPE) && (!cos || !sin || table_rows <= 0)) return DAISY_EINVAL;
  if (ve && (!ve_gate_logit || !(flags & DAISY_NORM_V))) return DAISY_EINVAL;
  if (!daisy_aligned16(k) || !daisy_aligned16(v) || !daisy_aligned16(q) || !daisy_aligned16(q_out) || !daisy_aligned16(ve) ||
      ((k_sb | k_st | k_sh | v_sb | v_st | v_sh) & 7) || (q && ((q_sb | q_st | q_sh) & 7)) || (ve && ((ve_sb | ve_st | ve_sh) & 7)))
    return DAISY_EALIGN;
  if ((flags & DAISY_ROPE) && (!daisy_aligned16(cos) || !daisy_aligned16(sin))) return DAISY_EALIGN;
  if ((reinterpret_cast<uintptr_t>(start) & 3) || (reinterpret_cast<uintptr_t>(cu) & 3)) return DAISY_EALIGN;
  p.Hq = q ? Hq : 0;
  const int64_t tokens = (int64_t)B * T, per_tok = (int64_t)p.Hq + 2 * (int64_t)cache->H;
  if (tokens * per_tok >= ((int64_t)1 << 31) - 512) return DAISY_EUNSUPPORTED;
  const int sms = daisy_host::sm_count_cached();
  if (sms <= 0) return DAISY_ENODEV;
  // warps a token: as many as come nearest to one wave of the SMs (3765 tokens x 48 rows: one, 0.8 of a wave, takes 5 % less than two), up to
  // a row for every group of eight lanes where tokens are few
  int64_t split = std::max<int64_t>(((int64_t)sms * APPEND_BLOCKS * APPEND_WARPS + tokens / 2) / tokens, 1);
  if (split > (per_tok + 3) / 4) split = (per_tok + 3) / 4;
  p.k = (const __nv_bfloat16*)k; p.v = (const __nv_bfloat16*)v; p.q = (const __nv_bfloat16*)q; p.ve = (const __nv_bfloat16*)ve;
  p.k_sb = k_sb; p.k_st = k_st; p.k_sh = k_sh; p.v_sb = v_sb; p.v_st = v_st; p.v_sh = v_sh;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh; p.ve_sb = ve_sb; p.ve_st = ve_st; p.ve_sh = ve_sh;
  p.q_out = (uint4*)q_out;
  p.start = start; p.cu = cu; p.cos = cos; p.sin = sin; p.ve_gate = ve_gate_logit;
  p.table_rows = table_rows; p.T = T; p.tokens = (int)tokens; p.split = (int)split;
  p.eps = eps; p.flags = flags; p.status = status_word;
  p.streams = tokens * per_tok * 256 > ((int64_t)32 << 20);
  const dim3 grid((unsigned)((tokens * split + APPEND_WARPS - 1) / APPEND_WARPS));
  const cudaError_t e = (flags & DAISY_CACHE_FP16) ? daisy_host::launch_dependent(paged_append_kernel<true>, grid, dim3(32 * APPEND_WARPS), 0, (cudaStream_t)stream, p)
                                                   : daisy_host::launch_dependent(paged_append_kernel<false>, grid, dim3(32 * APPEND_WARPS), 0, (cudaStream_t)stream, p);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return DAISY_ECUDA; }
  DAISY_CHECK_LAUNCH();
  return DAISY_OK;
}
