// Gradients of attention over packed sequences.
#include "attention.hip.h"

namespace fa {

struct GradArgs {
  Heads q, k, v, out, dout, dq, dk, dv;
  const float *lse;
  float *delta;  // [q_rows][heads]: dout . out
  int64_t q_rows, k_rows;
  int heads, kv_heads, group, dim;
  const int64_t *q_offsets, *q_lens, *k_offsets, *k_lens;
  int64_t m;
  float scale;
  int causal;
  int32_t *failure, code;
};

// Two components a lane, as in the forward kernel.
template <class E> __device__ __forceinline__ void load2(float (&x)[2], const uint16_t *p, int dim) {
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const int d = lane_id() + 64 * c;
    x[c] = d < dim ? E::load(p[d]) : 0.0f;
  }
}
template <class E> __device__ __forceinline__ void store2(const float (&x)[2], uint16_t *p, int dim) {
#pragma unroll
  for (int c = 0; c < 2; c++) {
    const int d = lane_id() + 64 * c;
    if (d < dim) p[d] = E::store(x[c]);
  }
}
__device__ __forceinline__ float dot2(const float (&a)[2], const float (&b)[2]) {
  float s = a[0] * b[0] + a[1] * b[1];
  for (int step = 1; step < WAVE; step *= 2) s += __shfl_xor(s, step);
  return s;
}

// A wave per query row and head: delta, then dq over the keys the row sees.
template <class E> __global__ __launch_bounds__(256) void attention_dq_kernel(GradArgs a) {
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    report_segments(a.q_offsets, a.q_lens, a.m, a.q_rows, a.failure, a.code);
    report_segments(a.k_offsets, a.k_lens, a.m, a.k_rows, a.failure, a.code);
  }
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
  const int h = blockIdx.y;
  if (row >= a.q_rows) return;
  int64_t q_first, q_len, k_first, k_len;
  const int64_t seg = segment_of_row(a.q_offsets, a.q_lens, a.m, a.q_rows, row, q_first, q_len);
  if (seg < 0 || !segment_ok(a.k_offsets, a.k_lens, seg, a.k_rows, k_first, k_len)) return;
  float q[2], o[2], g[2], dq[2] = {0.0f, 0.0f};
  load2<E>(q, a.q.at(row, h), a.dim);
  load2<E>(o, a.out.at(row, h), a.dim);
  load2<E>(g, a.dout.at(row, h), a.dim);
  const float delta = dot2(o, g), lse = a.lse[row * a.heads + h];
  if (lane_id() == 0) a.delta[row * a.heads + h] = delta;
  const int64_t keys = a.causal ? row - q_first + (k_len - q_len) + 1 : k_len;
  for (int64_t j = 0; j < keys; j++) {
    float k[2], v[2];
    load2<E>(k, a.k.at(k_first + j, h / a.group), a.dim);
    load2<E>(v, a.v.at(k_first + j, h / a.group), a.dim);
    const float p = lse == -INFINITY ? 0.0f : __expf(dot2(q, k) * a.scale - lse);
    const float ds = p * (dot2(g, v) - delta) * a.scale;
    dq[0] += ds * k[0];
    dq[1] += ds * k[1];
  }
  store2<E>(dq, a.dq.at(row, h), a.dim);
}

// A wave per key row and key head: dk and dv over the query rows that see it,
// of all the query heads of the group.
template <class E> __global__ __launch_bounds__(256) void attention_dkv_kernel(GradArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
  const int h = blockIdx.y;
  if (row >= a.k_rows) return;
  int64_t q_first, q_len, k_first, k_len;
  const int64_t seg = segment_of_row(a.k_offsets, a.k_lens, a.m, a.k_rows, row, k_first, k_len);
  if (seg < 0 || !segment_ok(a.q_offsets, a.q_lens, seg, a.q_rows, q_first, q_len)) return;
  float k[2], v[2], dk[2] = {0.0f, 0.0f}, dv[2] = {0.0f, 0.0f};
  load2<E>(k, a.k.at(row, h), a.dim);
  load2<E>(v, a.v.at(row, h), a.dim);
  int64_t from = a.causal ? row - k_first - (k_len - q_len) : 0;
  if (from < 0) from = 0;
  for (int qh = h * a.group; qh < (h + 1) * a.group; qh++)
    for (int64_t i = from; i < q_len; i++) {
      float q[2], g[2];
      load2<E>(q, a.q.at(q_first + i, qh), a.dim);
      load2<E>(g, a.dout.at(q_first + i, qh), a.dim);
      const float lse = a.lse[(q_first + i) * a.heads + qh], delta = a.delta[(q_first + i) * a.heads + qh];
      const float p = lse == -INFINITY ? 0.0f : __expf(dot2(q, k) * a.scale - lse);
      const float ds = p * (dot2(g, v) - delta) * a.scale;
#pragma unroll
      for (int c = 0; c < 2; c++) {
        dk[c] += ds * q[c];
        dv[c] += p * g[c];
      }
    }
  store2<E>(dk, a.dk.at(row, h), a.dim);
  store2<E>(dv, a.dv.at(row, h), a.dim);
}

}  // namespace fa

extern "C" size_t fa_attention_grad_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t heads,
                                                    int64_t kv_heads, int64_t head_dim, int64_t m) {
  (void)k_rows, (void)kv_heads, (void)head_dim, (void)m;
  return q_rows > 0 && heads > 0 ? (size_t)q_rows * heads * sizeof(float) : 0;
}

extern "C" int fa_attention_grad(fa_stream_t stream, fa_dtype t, const fa_heads *q, int64_t q_rows,
                                 const fa_heads *k, const fa_heads *v, int64_t k_rows, int64_t heads,
                                 int64_t kv_heads, int64_t head_dim, const int64_t *q_offsets,
                                 const int64_t *q_lens, const int64_t *k_offsets, const int64_t *k_lens,
                                 int64_t m, float scale, int causal, const fa_heads *out,
                                 const float *lse, const fa_heads *dout, const fa_heads *dq,
                                 const fa_heads *dk, const fa_heads *dv, void *workspace,
                                 size_t workspace_bytes, int32_t *failure, int32_t code) {
  int rc = check_shape(t, heads, kv_heads, head_dim);
  if (rc == 0) rc = check_segments(q_offsets, q_lens, m, q_rows);
  if (rc == 0) rc = check_segments(k_offsets, k_lens, m, k_rows);
  if (rc != 0) return rc;
  if (!(scale > 0.0f) || !(scale <= FLT_MAX)) return FA_EINVAL;
  if (m == 0 || (q_rows == 0 && k_rows == 0)) return 0;
  rc = check_heads(q, q_rows, heads, head_dim, false);
  if (rc == 0) rc = check_heads(k, k_rows, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(v, k_rows, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(out, q_rows, heads, head_dim, false);
  if (rc == 0) rc = check_heads(dout, q_rows, heads, head_dim, false);
  if (rc == 0) rc = check_heads(dq, q_rows, heads, head_dim, true);
  if (rc == 0) rc = check_heads(dk, k_rows, kv_heads, head_dim, true);
  if (rc == 0) rc = check_heads(dv, k_rows, kv_heads, head_dim, true);
  if (rc == 0 && lse == nullptr && q_rows > 0) rc = FA_EINVAL;
  if (rc == 0 && !is_aligned(lse, 4)) rc = FA_EALIGN;
  if (rc != 0) return rc;
  const size_t need = fa_attention_grad_workspace_bytes(q_rows, k_rows, heads, kv_heads, head_dim, m);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FA_ESCRATCH;
  if (!is_aligned(workspace, 16)) return FA_EALIGN;
  const GradArgs a = {to_heads(q), to_heads(k), to_heads(v), to_heads(out), to_heads(dout), to_heads(dq),
                      to_heads(dk), to_heads(dv), lse, (float *)workspace, q_rows, k_rows, (int)heads,
                      (int)kv_heads, (int)(heads / kv_heads), (int)head_dim, q_offsets, q_lens, k_offsets,
                      k_lens, m, scale, causal, failure, code};
  if (q_rows > 0) {
    const auto kernel = t == FA_F16 ? attention_dq_kernel<ElemF16> : attention_dq_kernel<ElemBF16>;
    kernel<<<dim3((unsigned)ceil_div(q_rows, 4), (unsigned)heads), dim3(256), 0, (hipStream_t)stream>>>(a);
    rc = launch_status();
    if (rc != 0) return rc;
  }
  if (k_rows > 0) {
    const auto kernel = t == FA_F16 ? attention_dkv_kernel<ElemF16> : attention_dkv_kernel<ElemBF16>;
    kernel<<<dim3((unsigned)ceil_div(k_rows, 4), (unsigned)kv_heads), dim3(256), 0, (hipStream_t)stream>>>(a);
    rc = launch_status();
  }
  return rc;
}
