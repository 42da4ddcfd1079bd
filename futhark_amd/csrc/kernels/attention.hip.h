// What the attention kernels (attention.hip, attention_grad.hip, kv_append.hip)
// share: argument checks on the host, 16-bit element types, arrays of heads and
// the walk over segments on the device.
#pragma once
#include "dispatch.hip.h"

namespace fa {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// 16-bit element types.  `store` rounds to nearest even.
struct ElemF16 {
  static __device__ __forceinline__ float load(uint16_t b) { return (float)bit_cast<_Float16>(b); }
  static __device__ __forceinline__ uint16_t store(float f) { return bit_cast<uint16_t>((_Float16)f); }
};
struct ElemBF16 {
  static __device__ __forceinline__ float load(uint16_t b) { return bit_cast<float>((uint32_t)b << 16); }
  static __device__ __forceinline__ uint16_t store(float f) { return bit_cast<uint16_t>((__bf16)f); }
};

// fa_heads as the kernels take it.
struct Heads {
  uint16_t *data;
  int64_t row_stride, head_stride;
  __device__ __forceinline__ uint16_t *at(int64_t row, int64_t head) const {
    return data + row * row_stride + head * head_stride;
  }
};

// A paged cache and its table (fa_kv_append, fa_attention_paged).
struct Pages {
  uint16_t *k, *v;
  int64_t n_pages;
  int page_shift;  // page_size is a power of two
  const int32_t *table;
  int64_t cols;
  const int64_t *past_lens;
  __device__ __forceinline__ int64_t capacity() const { return cols << page_shift; }
  // Elements before head `head` of page `page`, in rows of head_dim.
  __device__ __forceinline__ int64_t row_of(int64_t page, int64_t head, int64_t kv_heads) const {
    return (page * kv_heads + head) << page_shift;
  }
};

// ------------------------------------------------------------------ segments
// Segment i as the rules of fa_segred_irregular read it: inside [0, n), not
// before the end of its predecessor.
__device__ __forceinline__ bool segment_ok(const int64_t *offsets, const int64_t *lens, int64_t i,
                                           int64_t n, int64_t &first, int64_t &len) {
  first = offsets[i];
  len = lens[i];
  bool ok = first >= 0 && len >= 0 && first <= n && len <= n - first;
  if (i > 0) {
    const int64_t before = offsets[i - 1];
    ok = ok && before >= 0 && before <= first && lens[i - 1] <= first - before;
  }
  return ok;
}

// The segment that holds `row`, or -1; the same for the whole wave, which looks
// at 64 segments at a time.
__device__ __forceinline__ int64_t segment_of_row(const int64_t *offsets, const int64_t *lens, int64_t m,
                                                  int64_t n, int64_t row, int64_t &first, int64_t &len) {
  for (int64_t base = 0; base < m; base += WAVE) {
    const int64_t i = base + lane_id();
    int64_t f = 0, l = 0;
    const bool here = i < m && segment_ok(offsets, lens, i, n, f, l) && row >= f && row < f + l;
    const uint64_t found = __ballot(here);
    if (found != 0) {
      const int at = __builtin_ctzll(found);
      first = read_lane(f, at);
      len = read_lane(l, at);
      return base + at;
    }
  }
  return -1;
}

// Reports broken segments; every thread of the calling block takes part.
__device__ __forceinline__ void report_segments(const int64_t *offsets, const int64_t *lens, int64_t m,
                                                int64_t n, int32_t *failure, int32_t code) {
  if (failure == nullptr) return;
  for (int64_t i = threadIdx.x; i < m; i += blockDim.x) {
    int64_t first, len;
    if (!segment_ok(offsets, lens, i, n, first, len)) *failure = code;
  }
}

// ------------------------------------------------------------- host side checks
inline bool heads_span_ok(int64_t rows, int64_t heads, int64_t dim, const fa_heads *x) {
  const __int128 last = (__int128)(rows > 0 ? rows - 1 : 0) * x->row_stride +
                        (__int128)(heads > 0 ? heads - 1 : 0) * x->head_stride + dim;
  return last < ((__int128)1 << 61);
}

inline int check_heads(const fa_heads *x, int64_t rows, int64_t heads, int64_t dim, bool written) {
  if (x == nullptr || (x->data == nullptr && rows > 0)) return FA_EINVAL;
  if (x->row_stride < 0 || x->head_stride < 0) return FA_EINVAL;
  if (!is_aligned(x->data, 16) || x->row_stride % 8 != 0 || x->head_stride % 8 != 0) return FA_EALIGN;
  if (!heads_span_ok(rows, heads, dim, x)) return FA_EINVAL;
  if (written) {
    // One of the two dimensions lies inside a step of the other.
    const __int128 r = x->row_stride, h = x->head_stride;
    const bool rows_outer = (heads <= 1 || h >= dim) && (rows <= 1 || r >= (heads - 1) * h + dim);
    const bool heads_outer = (rows <= 1 || r >= dim) && (heads <= 1 || h >= (rows - 1) * r + dim);
    if (!rows_outer && !heads_outer) return FA_EINVAL;
  }
  return 0;
}

inline int check_shape(fa_dtype t, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  if (heads <= 0 || kv_heads <= 0 || head_dim <= 0 || heads % kv_heads != 0) return FA_EINVAL;
  if (t != FA_F16 && t != FA_BF16) return FA_ENOTSUP;
  if (head_dim % 8 != 0 || head_dim > 128 || heads / kv_heads > 128 || heads > 65535) return FA_ENOTSUP;
  return 0;
}

inline int check_segments(const int64_t *offsets, const int64_t *lens, int64_t m, int64_t n) {
  if (m < 0 || n < 0) return FA_EINVAL;
  if (m > INT32_MAX || n > INT32_MAX) return FA_ENOTSUP;
  if (m > 0 && (offsets == nullptr || lens == nullptr)) return FA_EINVAL;
  if (!is_aligned(offsets, 8) || !is_aligned(lens, 8)) return FA_EALIGN;
  return 0;
}

inline int check_pages(const void *k_pages, const void *v_pages, int64_t n_pages, int64_t page_size,
                       const int32_t *table, int64_t cols, const int64_t *past_lens, int64_t kv_heads,
                       int64_t head_dim) {
  if (n_pages < 0 || page_size <= 0 || cols < 0) return FA_EINVAL;
  if ((page_size & (page_size - 1)) != 0 || n_pages > INT32_MAX) return FA_ENOTSUP;
  if ((__int128)cols * page_size > INT32_MAX) return FA_ENOTSUP;
  if ((__int128)n_pages * page_size * kv_heads * head_dim >= ((__int128)1 << 61)) return FA_EINVAL;
  if (past_lens == nullptr || (table == nullptr && cols > 0)) return FA_EINVAL;
  if ((k_pages == nullptr || v_pages == nullptr) && n_pages > 0) return FA_EINVAL;
  if (!is_aligned(k_pages, 16) || !is_aligned(v_pages, 16) || !is_aligned(past_lens, 8) || !is_aligned(table, 4))
    return FA_EALIGN;
  return 0;
}

inline Heads to_heads(const fa_heads *x) {
  return Heads{(uint16_t *)x->data, x->row_stride, x->head_stride};
}

inline Pages to_pages(const void *k_pages, const void *v_pages, int64_t n_pages, int64_t page_size,
                      const int32_t *table, int64_t cols, const int64_t *past_lens) {
  return Pages{(uint16_t *)k_pages, (uint16_t *)v_pages, n_pages, __builtin_ctzll((uint64_t)page_size),
               table, cols, past_lens};
}

}  // namespace fa
