// Appending new keys and values to a paged cache, with the position rotation of
// keys and queries applied on the way.  Pure traffic: every row is read once
// and written once.
#include "attention.hip.h"

namespace fa {

// A wave per token and slice of its heads; lanes walk the (head, component)
// pairs.  The angle is position * frequency in f64, reduced there, because a
// far position times a frequency near 1 leaves few bits of the angle in f32.
template <class E>
__global__ __launch_bounds__(256) void kv_append_kernel(Heads q, Heads q_out, Heads k, Heads v, int64_t n,
                                                        int heads, int kv_heads, int dim,
                                                        const int64_t *__restrict__ offsets,
                                                        const int64_t *__restrict__ lens, int64_t m,
                                                        const float *__restrict__ freqs, int rot,
                                                        int interleaved, Pages pages, int32_t *failure,
                                                        int32_t code) {
  if (blockIdx.x == 0) report_segments(offsets, lens, m, n, failure, code);
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
  if (row >= n) return;
  int64_t first, len;
  const int64_t seg = segment_of_row(offsets, lens, m, n, row, first, len);
  if (seg < 0) return;
  const int64_t past = pages.past_lens[seg];
  if (past < 0 || past > pages.capacity() || len > pages.capacity() - past) {
    if (failure != nullptr) *failure = code;
    return;
  }
  const int64_t pos = past + (row - first);
  const int64_t page = pages.table[seg * pages.cols + (pos >> pages.page_shift)];
  const int64_t slot = pos & (((int64_t)1 << pages.page_shift) - 1);
  const bool stored = page >= 0 && page < pages.n_pages;
  if (!stored && failure != nullptr) *failure = code;
  const int half = rot / 2, units = dim - half;  // a pair or a lone component
  const int q_heads = q.data != nullptr ? heads : 0;
  for (int i = lane_id(); i < (q_heads + 2 * kv_heads) * units; i += WAVE) {
    const int h = i / units, u = i % units;
    const uint16_t *src;
    uint16_t *dst;
    bool turn = true;
    if (h < q_heads) {
      src = q.at(row, h);
      dst = q_out.at(row, h);
    } else {
      if (!stored) continue;
      const bool is_v = h >= q_heads + kv_heads;
      const int kh = h - q_heads - (is_v ? kv_heads : 0);
      src = is_v ? v.at(row, kh) : k.at(row, kh);
      dst = (is_v ? pages.v : pages.k) + (pages.row_of(page, kh, kv_heads) + slot) * dim;
      turn = !is_v;
    }
    if (u < half) {
      const int a = interleaved ? 2 * u : u, b = interleaved ? 2 * u + 1 : u + half;
      if (turn) {
        double s, c;
        sincos((double)pos * (double)freqs[u], &s, &c);
        const float x = E::load(src[a]), y = E::load(src[b]), cf = (float)c, sf = (float)s;
        dst[a] = E::store(x * cf - y * sf);
        dst[b] = E::store(y * cf + x * sf);
      } else {
        dst[a] = src[a];
        dst[b] = src[b];
      }
    } else {
      dst[u + half] = src[u + half];
    }
  }
}

}  // namespace fa

extern "C" int fa_kv_append(fa_stream_t stream, fa_dtype t, const fa_heads *q, const fa_heads *q_out,
                            const fa_heads *k, const fa_heads *v, int64_t n, int64_t heads,
                            int64_t kv_heads, int64_t head_dim, const int64_t *offsets,
                            const int64_t *lens, int64_t m, const int64_t *past_lens, const float *freqs,
                            int64_t rot_dim, int interleaved, void *k_pages, void *v_pages,
                            int64_t n_pages, int64_t page_size, const int32_t *page_table,
                            int64_t table_cols, int32_t *failure, int32_t code) {
  int rc = check_shape(t, heads, kv_heads, head_dim);
  if (rc == 0) rc = check_segments(offsets, lens, m, n);
  if (rc != 0) return rc;
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0) return FA_EINVAL;
  if (n == 0 || m == 0) return 0;
  if (rot_dim > 0 && freqs == nullptr) return FA_EINVAL;
  if (!is_aligned(freqs, 4)) return FA_EALIGN;
  if (q != nullptr) {
    rc = check_heads(q, n, heads, head_dim, false);
    if (rc == 0) rc = check_heads(q_out, n, heads, head_dim, true);
    if (rc != 0) return rc;
  }
  rc = check_heads(k, n, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(v, n, kv_heads, head_dim, false);
  if (rc == 0) rc = check_pages(k_pages, v_pages, n_pages, page_size, page_table, table_cols, past_lens, kv_heads, head_dim);
  if (rc != 0) return rc;
  const fa_heads none = {nullptr, 0, 0};
  const Heads qh = to_heads(q != nullptr ? q : &none), qo = to_heads(q != nullptr ? q_out : &none);
  const Pages pages = to_pages(k_pages, v_pages, n_pages, page_size, page_table, table_cols, past_lens);
  const auto kernel = t == FA_F16 ? kv_append_kernel<ElemF16> : kv_append_kernel<ElemBF16>;
  kernel<<<dim3((unsigned)ceil_div(n, 4)), dim3(256), 0, (hipStream_t)stream>>>(
      qh, qo, to_heads(k), to_heads(v), n, (int)heads, (int)kv_heads, (int)head_dim, offsets, lens, m, freqs,
      (int)rot_dim, interleaved, pages, failure, code);
  return launch_status();
}
