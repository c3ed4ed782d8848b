// A pool of pages and the tables that name them, as the kernels and launchers of the paged cache see them.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace daisy {

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two values to the pages' 16-bit type, and back
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) { return F16 ? pack_half(lo, hi) : pack_bf16(lo, hi); }
template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t u) {
  if (F16) return __half22float2(*reinterpret_cast<const __half2*>(&u));
  return make_float2(bf16_lo(u), bf16_hi(u));
}
template <bool F16>
__device__ __forceinline__ uint4 pack8_16(const float* f) {
  return make_uint4(pack16<F16>(f[0], f[1]), pack16<F16>(f[2], f[3]), pack16<F16>(f[4], f[5]), pack16<F16>(f[6], f[7]));
}

// Softmax weights are powers of two over a reference that lies this far under the row's maximum: float16 has a floor of 2^-25 and room up to 2^15,
// bf16 neither.  With the references' lag of up to 2^8 a float16 weight reaches 2^15, and is off by at most 2^-32 of the largest one
// beside its rounding (with a reference at the maximum 2^-25: 4096 rows at 2^-25.3 behind one at 1 were not seen at all).
template <bool F16>
constexpr float WEIGHT_ROOM = F16 ? 7.f : 0.f;

struct PagedCache {
  char *k, *v;                       // pages [n_pages, H, page, 128] of 16-bit values
  int64_t p_sb, p_sh, p_sr;          // element strides of page, head, row
  const int* table;
  int64_t table_sb;
  int n_pages, H, lg, width, n_seq;  // page = 1 << lg
  int cap;                           // positions that the table has, or the caller grants
  __device__ __forceinline__ int64_t capacity() const { return cap; }
  // byte offset of row `pos` of head h in page `pg`
  __device__ __forceinline__ int64_t at(int pg, int h, int pos) const {
    return 2 * (pg * p_sb + h * p_sh + (pos & ((1 << lg) - 1)) * p_sr);
  }
};

// The sequence that token `tok` of a packed row belongs to: the last b with cu[b] <= tok, by the warp's 32 lanes at once; -1 in front
// of cu[0].  Whatever cu holds the result is below n_seq.
__device__ __forceinline__ int find_seq(const int* cu, int n_seq, int tok, int lane) {
  int lo = 0, len = n_seq;
  while (len > 0) {
    const int step = (len + 31) / 32, i = lo + lane * step;
    const bool le = lane * step < len && cu[i] <= tok;
    const int n = __popc(__ballot_sync(0xffffffffu, le));
    if (n == 0) return lo - 1;                                     // only in front of cu[0], where lo is 0, or in an unsorted cu
    if (step == 1) return lo + n - 1;
    lo += (n - 1) * step;
    len = min(step, n_seq - lo);
  }
  return -1;
}

}  // namespace daisy

namespace daisy_host {

// The cache as the kernels take it, or a status.
static inline int paged_cache(const daisy_b200_pages* c, int D, daisy::PagedCache* out) {
  if (!c || !c->k || !c->v || !c->table || c->n_pages <= 0 || c->H <= 0 || c->width <= 0 || c->n_seq <= 0 || c->table_sb < 0 || c->max_len < 0) return DAISY_EINVAL;
  if (D != DAISY_HEAD_DIM) return DAISY_EUNSUPPORTED;
  int lg = 4;
  while (lg < 8 && (1 << lg) != c->page) ++lg;
  if ((1 << lg) != c->page) return DAISY_EUNSUPPORTED;
  if (((int64_t)c->width << lg) >= ((int64_t)1 << 31) - 256) return DAISY_EUNSUPPORTED;          // positions are 32-bit
  if (!daisy_aligned16(c->k) || !daisy_aligned16(c->v) || ((c->p_sb | c->p_sh | c->p_sr) & 7) || (reinterpret_cast<uintptr_t>(c->table) & 3)) return DAISY_EALIGN;
  // rows are written: none may stand for two
  if (c->p_sr < D || (c->H > 1 && c->p_sh < D) || (c->n_pages > 1 && c->p_sb < D)) return DAISY_EINVAL;
  *out = daisy::PagedCache{(char*)c->k, (char*)c->v, c->p_sb, c->p_sh, c->p_sr, c->table, c->table_sb, c->n_pages, c->H, lg, c->width, c->n_seq, c->width << lg};
  if (c->max_len > 0 && c->max_len < out->cap) out->cap = c->max_len;
  return DAISY_OK;
}

// A window that holds every position that the table can is none: differences of positions and windows stay inside 32 bits.
static inline int paged_window(const daisy_b200_pages* c, int window) { return window > 0 && window < (int64_t)c->width * c->page ? window : 0; }

}  // namespace daisy_host
