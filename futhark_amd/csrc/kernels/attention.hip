// Attention over packed sequences and over a paged cache: forward.
#include "attention.hip.h"

namespace fa {

static __device__ uint4 g_zero_row[16];  // a key or value of zeros: 128 components

// A wave per query row and head: lane l holds components l and l + 64, walks
// the visible keys one by one and keeps the running maximum and sum of the
// softmax in f32.
struct Row {
  float q[2], o[2] = {0.0f, 0.0f};
  float top = -INFINITY, sum = 0.0f;
};
template <class E>
__device__ __forceinline__ void row_see(Row &r, const uint16_t *k, const uint16_t *v, int dim, float scale) {
  const int lane = lane_id();
  float s = 0.0f, vv[2];
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const int d = lane + 64 * c;
    s += d < dim ? r.q[c] * E::load(k[d]) : 0.0f;
    vv[c] = d < dim ? E::load(v[d]) : 0.0f;
  }
  for (int step = 1; step < WAVE; step *= 2) s += __shfl_xor(s, step);
  s *= scale;
  const float top = fmaxf(r.top, s);
  if (top == -INFINITY) return;
  const float old = __expf(r.top - top), p = __expf(s - top);
  r.sum = r.sum * old + p;
#pragma unroll
  for (int c = 0; c < 2; c++) r.o[c] = r.o[c] * old + p * vv[c];
  r.top = top;
}
template <class E> __device__ __forceinline__ void row_load(Row &r, const uint16_t *q, int dim) {
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const int d = lane_id() + 64 * c;
    r.q[c] = d < dim ? E::load(q[d]) : 0.0f;
  }
}
template <class E> __device__ __forceinline__ void row_store(const Row &r, uint16_t *out, float *lse, int dim) {
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const int d = lane_id() + 64 * c;
    if (d < dim) out[d] = E::store(r.top == -INFINITY ? 0.0f : r.o[c] / r.sum);
  }
  if (lse != nullptr && lane_id() == 0) *lse = r.top == -INFINITY ? -INFINITY : r.top + __logf(r.sum);
}

template <class E>
__global__ __launch_bounds__(256) void attention_kernel(
    Heads q, Heads k, Heads v, Heads out, float *lse, int64_t q_rows, int64_t k_rows, int heads, int group,
    int dim, const int64_t *q_offsets, const int64_t *q_lens, const int64_t *k_offsets,
    const int64_t *k_lens, int64_t m, float scale, int causal, int32_t *failure, int32_t code) {
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    report_segments(q_offsets, q_lens, m, q_rows, failure, code);
    report_segments(k_offsets, k_lens, m, k_rows, failure, code);
  }
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
  const int h = blockIdx.y;
  if (row >= q_rows) return;
  int64_t q_first, q_len, k_first, k_len;
  const int64_t seg = segment_of_row(q_offsets, q_lens, m, q_rows, row, q_first, q_len);
  if (seg < 0 || !segment_ok(k_offsets, k_lens, seg, k_rows, k_first, k_len)) return;
  int64_t keys = causal ? row - q_first + (k_len - q_len) + 1 : k_len;
  Row r;
  row_load<E>(r, q.at(row, h), dim);
  for (int64_t j = 0; j < keys; j++)
    row_see<E>(r, k.at(k_first + j, h / group), v.at(k_first + j, h / group), dim, scale);
  row_store<E>(r, out.at(row, h), lse == nullptr ? nullptr : lse + row * heads + h, dim);
}

template <class E>
__global__ __launch_bounds__(256) void attention_paged_kernel(
    Heads q, Heads out, float *lse, int64_t n, int heads, int group, int dim, const int64_t *offsets,
    const int64_t *lens, int64_t m, float scale, Pages pages, int32_t *failure, int32_t code) {
  if (blockIdx.x == 0 && blockIdx.y == 0) report_segments(offsets, lens, m, n, failure, code);
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
  const int h = blockIdx.y;
  if (row >= n) return;
  int64_t first, len;
  const int64_t seg = segment_of_row(offsets, lens, m, n, row, first, len);
  if (seg < 0) return;
  const int64_t past = pages.past_lens[seg];
  if (past < 0 || past > pages.capacity() || len > pages.capacity() - past) {
    if (failure != nullptr) *failure = code;
    return;
  }
  Row r;
  row_load<E>(r, q.at(row, h), dim);
  for (int64_t j = 0; j <= past + (row - first); j++) {
    const int64_t page = pages.table[seg * pages.cols + (j >> pages.page_shift)];
    const int64_t slot = j & (((int64_t)1 << pages.page_shift) - 1);
    const uint16_t *kp = (const uint16_t *)g_zero_row, *vp = kp;
    if (page >= 0 && page < pages.n_pages) {
      const int64_t at = (pages.row_of(page, h / group, heads / group) + slot) * dim;
      kp = pages.k + at;
      vp = pages.v + at;
    } else if (failure != nullptr) {
      *failure = code;
    }
    row_see<E>(r, kp, vp, dim, scale);
  }
  row_store<E>(r, out.at(row, h), lse == nullptr ? nullptr : lse + row * heads + h, dim);
}

}  // namespace fa

extern "C" int fa_attention(fa_stream_t stream, fa_dtype t, const fa_heads *q, int64_t q_rows,
                            const fa_heads *k, const fa_heads *v, int64_t k_rows, int64_t heads,
                            int64_t kv_heads, int64_t head_dim, const int64_t *q_offsets,
                            const int64_t *q_lens, const int64_t *k_offsets, const int64_t *k_lens,
                            int64_t m, float scale, int causal, const fa_heads *out, float *lse,
                            int32_t *failure, int32_t code) {
  int rc = check_shape(t, heads, kv_heads, head_dim);
  if (rc == 0) rc = check_segments(q_offsets, q_lens, m, q_rows);
  if (rc == 0) rc = check_segments(k_offsets, k_lens, m, k_rows);
  if (rc != 0) return rc;
  if (!(scale > 0.0f) || !(scale <= FLT_MAX)) return FA_EINVAL;
  if (q_rows == 0 || m == 0) return 0;
  rc = check_heads(q, q_rows, heads, head_dim, false);
  if (rc == 0) rc = check_heads(k, k_rows, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(v, k_rows, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(out, q_rows, heads, head_dim, true);
  if (rc == 0 && !is_aligned(lse, 4)) rc = FA_EALIGN;
  if (rc != 0) return rc;
  const auto kernel = t == FA_F16 ? attention_kernel<ElemF16> : attention_kernel<ElemBF16>;
  kernel<<<dim3((unsigned)ceil_div(q_rows, 4), (unsigned)heads), dim3(256), 0, (hipStream_t)stream>>>(
      to_heads(q), to_heads(k), to_heads(v), to_heads(out), lse, q_rows, k_rows, (int)heads,
      (int)(heads / kv_heads), (int)head_dim, q_offsets, q_lens, k_offsets, k_lens, m, scale, causal, failure,
      code);
  return launch_status();
}

extern "C" size_t fa_attention_paged_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                                                     int64_t) {
  return 0;
}

extern "C" int fa_attention_paged(fa_stream_t stream, fa_dtype t, const fa_heads *q, int64_t n,
                                  int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  const int64_t *offsets, const int64_t *lens, int64_t m,
                                  const int64_t *past_lens, float scale, const void *k_pages,
                                  const void *v_pages, int64_t n_pages, int64_t page_size,
                                  const int32_t *page_table, int64_t table_cols, const fa_heads *out,
                                  float *lse, void *workspace, size_t workspace_bytes, int32_t *failure,
                                  int32_t code) {
  int rc = check_shape(t, heads, kv_heads, head_dim);
  if (rc == 0) rc = check_segments(offsets, lens, m, n);
  if (rc != 0) return rc;
  if (!(scale > 0.0f) || !(scale <= FLT_MAX)) return FA_EINVAL;
  if (n == 0 || m == 0) return 0;
  rc = check_heads(q, n, heads, head_dim, false);
  if (rc == 0) rc = check_heads(out, n, heads, head_dim, true);
  if (rc == 0) rc = check_pages(k_pages, v_pages, n_pages, page_size, page_table, table_cols, past_lens, kv_heads, head_dim);
  if (rc == 0 && !is_aligned(lse, 4)) rc = FA_EALIGN;
  if (rc != 0) return rc;
  const size_t need = fa_attention_paged_workspace_bytes(n, heads, kv_heads, head_dim, m, page_size, table_cols);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FA_ESCRATCH;
  const Pages pages = to_pages(k_pages, v_pages, n_pages, page_size, page_table, table_cols, past_lens);
  const auto kernel = t == FA_F16 ? attention_paged_kernel<ElemF16> : attention_paged_kernel<ElemBF16>;
  kernel<<<dim3((unsigned)ceil_div(n, 4), (unsigned)heads), dim3(256), 0, (hipStream_t)stream>>>(
      to_heads(q), to_heads(out), lse, n, (int)heads, (int)(heads / kv_heads), (int)head_dim, offsets, lens, m,
      scale, pages, failure, code);
  return launch_status();
}
