// Keys and values of new tokens into a paged cache, RMS-normalised and rotated on the way; their queries beside them.
//
// A streaming pass: 256 bytes read and 256 written for every row (token, head) of q, k and v, bound by HBM for prompts
// and by the chain start -> position -> page -> row for a few tokens.  Eight lanes a row, 16 bytes of each half a lane: the two
// halves that the rotation pairs lie in one thread.  Rows are numbered (token, head of q | k | v), so that a warp's four rows of
// one token share its position, page and table row, and consecutive blocks read consecutive memory.
#include "paged.cuh"

namespace daisy {

struct AppendParams {
  PagedCache c;
  const __nv_bfloat16 *k, *v, *q, *ve;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh, q_sb, q_st, q_sh, ve_sb, ve_st, ve_sh;
  uint4* q_out;
  const int *start, *cu;
  const float *cos, *sin, *ve_gate;
  int table_rows, T, Hq, n_rows;     // Hq = 0: no queries; n_rows = tokens x (Hq + 2 H)
  float eps;
  unsigned flags;
  int* status;
};

constexpr int APPEND_ROWS = 2;       // rows a group of eight lanes keeps in flight

template <bool F16>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const uint32_t per_tok = p.Hq + 2 * p.c.H;
  const uint32_t row0 = (blockIdx.x * 256u + threadIdx.x) / 8 * APPEND_ROWS;
  const uint32_t n_rows = p.n_rows;
  // first token of the warp, its sequence, and from there on token by token
  int b = 0, b_end = 0;
  if (p.cu) {
    const uint32_t first = min((row0 & ~(4u * APPEND_ROWS - 1)), n_rows - 1) / per_tok;
    b = find_seq(p.cu, p.c.n_seq, (int)first, lane);
    b_end = b >= 0 ? p.cu[b + 1] : p.cu[0];
  }
  uint4 lo[APPEND_ROWS], hi[APPEND_ROWS], mlo[APPEND_ROWS], mhi[APPEND_ROWS];
  int64_t pos[APPEND_ROWS];
  int seq[APPEND_ROWS], head[APPEND_ROWS];                               // head among q | k | v; -1: nothing to do
#pragma unroll
  for (int u = 0; u < APPEND_ROWS; ++u) {
    const uint32_t row = min(row0 + u, n_rows - 1);
    const uint32_t tok = row / per_tok;
    head[u] = row0 + u < n_rows ? (int)(row - tok * per_tok) : -1;
    int64_t bt, tt;
    if (p.cu) {
      while ((int)tok >= b_end && b + 1 < p.c.n_seq) b_end = p.cu[++b + 1];
      if (b < 0 || (int)tok >= b_end) head[u] = -1;                     // in front of the first sequence or behind the last
      seq[u] = max(b, 0);
      bt = 0; tt = tok;
      pos[u] = (int64_t)tok - p.cu[seq[u]];
    } else {
      seq[u] = tok / (uint32_t)p.T;
      bt = seq[u]; tt = tok - seq[u] * (uint32_t)p.T;
      pos[u] = tt;
    }
    const int h = head[u];
    if (h >= 0) {
      const __nv_bfloat16* src = h < p.Hq ? p.q + bt * p.q_sb + tt * p.q_st + h * p.q_sh
                               : h < p.Hq + p.c.H ? p.k + bt * p.k_sb + tt * p.k_st + (h - p.Hq) * p.k_sh
                                                  : p.v + bt * p.v_sb + tt * p.v_st + (h - p.Hq - p.c.H) * p.v_sh;
      lo[u] = ld_stream16(src + 8 * sub);
      hi[u] = ld_stream16(src + 64 + 8 * sub);
      if (p.ve && h >= p.Hq + p.c.H) {
        const __nv_bfloat16* m = p.ve + bt * p.ve_sb + tt * p.ve_st + (h - p.Hq - p.c.H) * p.ve_sh;
        mlo[u] = ld_stream16(m + 8 * sub);
        mhi[u] = ld_stream16(m + 64 + 8 * sub);
      }
      const int first = p.start[seq[u]];
      if (first < 0) head[u] = -1;
      pos[u] += first;
    } else {
      lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
    }
  }
#pragma unroll
  for (int u = 0; u < APPEND_ROWS; ++u) {
    const int h = head[u];
    const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.c.H;
    bool ok = h >= 0;
    if (ok && (pos[u] < 0 || pos[u] >= p.c.capacity() || ((p.flags & DAISY_ROPE) && pos[u] >= p.table_rows))) {
      if (p.status && sub == 0) p.status[0] = DAISY_EINVAL;
      ok = false;
    }
    float x1[8], x2[8];
    unpack8(lo[u], x1);
    unpack8(hi[u], x2);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x1[e] * x1[e] + x2[e] * x2[e];
    ss += __shfl_xor_sync(0xffffffffu, ss, 4);
    ss += __shfl_xor_sync(0xffffffffu, ss, 2);
    ss += __shfl_xor_sync(0xffffffffu, ss, 1);
    if (!ok) continue;                                              // no shuffles below
    if (p.flags & (is_q ? DAISY_NORM_Q : is_v ? DAISY_NORM_V : DAISY_NORM_K)) {
      const float r = rsqrtf(ss * (1.0f / DAISY_HEAD_DIM) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) { x1[e] *= r; x2[e] *= r; }
    }
    if (!is_v && (p.flags & DAISY_ROPE)) {
      const float4* cr = reinterpret_cast<const float4*>(p.cos + pos[u] * 64 + 8 * sub);
      const float4* sr = reinterpret_cast<const float4*>(p.sin + pos[u] * 64 + 8 * sub);
      const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
      const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x1[e], d = x2[e];
        x1[e] = a * c[e] + d * s[e];
        x2[e] = d * c[e] - a * s[e];
      }
    }
    if (is_v && p.ve) {
      const float g = 1.0f / (1.0f + __expf(-*p.ve_gate));
      float m1[8], m2[8];
      unpack8(mlo[u], m1);
      unpack8(mhi[u], m2);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x1[e] = g * x1[e] + (1.0f - g) * m1[e];
        x2[e] = g * x2[e] + (1.0f - g) * m2[e];
      }
    }
    const uint4 y1 = pack8_16<F16>(x1), y2 = pack8_16<F16>(x2);
    if (is_q) {
      const uint32_t tok = (row0 + u) / per_tok;
      uint4* dst = p.q_out + ((int64_t)tok * p.Hq + h) * 16 + sub;
      dst[0] = y1;
      dst[8] = y2;
    } else {
      const int pg = p.c.table[seq[u] * p.c.table_sb + (pos[u] >> p.c.lg)];
      if ((unsigned)pg >= (unsigned)p.c.n_pages) {
        if (p.status && sub == 0) p.status[0] = DAISY_EINVAL;
        continue;
      }
      char* dst = (is_v ? p.c.v : p.c.k) + p.c.at(pg, is_v ? h - p.Hq - p.c.H : h - p.Hq, (int)pos[u]) + 16 * sub;
      *reinterpret_cast<uint4*>(dst) = y1;
      *reinterpret_cast<uint4*>(dst + 128) = y2;
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
  const int64_t rows = (int64_t)B * T * ((int64_t)p.Hq + 2 * (int64_t)cache->H);
  if (rows >= ((int64_t)1 << 31) - 512) return DAISY_EUNSUPPORTED;
  p.k = (const __nv_bfloat16*)k; p.v = (const __nv_bfloat16*)v; p.q = (const __nv_bfloat16*)q; p.ve = (const __nv_bfloat16*)ve;
  p.k_sb = k_sb; p.k_st = k_st; p.k_sh = k_sh; p.v_sb = v_sb; p.v_st = v_st; p.v_sh = v_sh;
  p.q_sb = q_sb; p.q_st = q_st; p.q_sh = q_sh; p.ve_sb = ve_sb; p.ve_st = ve_st; p.ve_sh = ve_sh;
  p.q_out = (uint4*)q_out;
  p.start = start; p.cu = cu; p.cos = cos; p.sin = sin; p.ve_gate = ve_gate_logit;
  p.table_rows = table_rows; p.T = T; p.n_rows = (int)rows;
  p.eps = eps; p.flags = flags; p.status = status_word;
  constexpr int per_block = 32 * APPEND_ROWS;
  const dim3 grid((unsigned)((rows + per_block - 1) / per_block));
  const cudaError_t e = (flags & DAISY_CACHE_FP16) ? daisy_host::launch_dependent(paged_append_kernel<true>, grid, dim3(256), 0, (cudaStream_t)stream, p)
                                                   : daisy_host::launch_dependent(paged_append_kernel<false>, grid, dim3(256), 0, (cudaStream_t)stream, p);
  if (e != cudaSuccess) { (void)cudaGetLastError(); return DAISY_ECUDA; }
  DAISY_CHECK_LAUNCH();
  return DAISY_OK;
}
