// Appending new keys and values to a paged cache, with the position rotation of
// keys and queries applied on the way.  Pure traffic: every row is read once and
// written once, 16 bytes a thread.
//
// A block takes some heads of one token.  Their rows go through LDS, because a
// component's partner in the rotation may lie anywhere in its row; the sines and
// cosines of the token's position are computed once for all of them.  Loads return
// in the order they were asked for: the segments come first, the rows behind them,
// and the page number past both by the scalar cache, so that looking up the place
// and computing the angles hide behind the rows (14555 tokens of 32 + 8 heads of
// 128: 79 -> 58 us a call, 6.1 TB/s).  Loads and stores are non-temporal: nothing is
// used twice (88 -> 78 us before that).  32 tokens: 4.5 us, launch and the chain.
#include "attention.hip.h"

namespace fa {

constexpr int KA_THREADS = 256;
constexpr int KA_MOST_DIM = 128;
constexpr int KA_UNITS = 3;      // 16-byte units a thread
constexpr int KA_SEGMENTS = 4;   // segments a lane looks at at a time

// The sequence of a row with its first row and cached tokens; the same for the
// whole wave.  A lane looks at N segments from `base` on.
template <int N> struct Look {
  int64_t first[N], len[N], past[N];
  bool ok[N];
  __device__ __forceinline__ void load(const int64_t *offsets, const int64_t *lens, const int64_t *past_lens, int64_t m,
                                       int64_t n, int64_t base) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int64_t i = base + j * WAVE + lane_id(), at = i < m ? i : m - 1;
      past[j] = past_lens[at];
      ok[j] = segment_ok(offsets, lens, at, n, first[j], len[j]) & (i < m);
    }
  }
  // The number of the row's segment from `base` on, or -1.
  __device__ __forceinline__ int find(int64_t row, const int64_t *offsets, const int64_t *lens, int64_t m, int64_t n, int64_t base,
                                      SegChain &chain, int64_t &f, int64_t &l, int64_t &p) const {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const bool kept = chain.keep(ok[j], first[j], len[j], offsets, lens, m, n, base + j * WAVE);
      const uint64_t found = __ballot(kept && row >= first[j] && row < first[j] + len[j]);
      if (found != 0) {
        const int at = __builtin_ctzll(found);
        f = read_lane(first[j], at);
        l = read_lane(len[j], at);
        p = read_lane(past[j], at);
        return j * WAVE + at;
      }
    }
    return -1;
  }
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
  Heads q, q_out, k, v;
  int64_t n;
  int q_heads, kv_heads, dim, block_heads;
  const int64_t *offsets, *lens;
  int64_t m;
  const float *freqs;
  int rot, interleaved;
  Pages pages;
  int32_t *failure, code;
};

// From an address that is the same for the wave, through the scalar cache.
__device__ __forceinline__ int32_t scalar_load(const int32_t *p) {
  return *(const int32_t __attribute__((address_space(4))) *)wave_address(p);
}

template <class E> __global__ __launch_bounds__(KA_THREADS) void kv_append_kernel(AppendArgs a) {
  __shared__ uint4 rows[KA_THREADS * KA_UNITS];
  __shared__ float cosine[KA_MOST_DIM / 2], sine[KA_MOST_DIM / 2];
  const int64_t row = blockIdx.x;
  const int per_row = a.dim / 8, heads = a.q_heads + 2 * a.kv_heads;
  const int head0 = blockIdx.y * a.block_heads;
  const int units = (heads - head0 < a.block_heads ? heads - head0 : a.block_heads) * per_row;
  // The first segments and this thread's frequency before the rows.
  Look<1> nearest;
  nearest.load(a.offsets, a.lens, a.pages.past_lens, a.m, a.n, 0);
  const int half = a.rot / 2;
  const float *freqs = half > 0 ? a.freqs : reinterpret_cast<const float *>(a.lens);  // (something to load)
  const float freq = freqs[(int)threadIdx.x < half ? threadIdx.x : 0];
  // Heads are numbered: queries, keys, values.
  uint4 mine[KA_UNITS];
  const uint16_t *q_row = a.q.at(row, 0), *k_row = a.k.at(row, 0), *v_row = a.v.at(row, 0);
#pragma unroll
  for (int j = 0; j < KA_UNITS; j++) {
    // (no branches: loads under a condition would be waited for one by one)
    const int i = j * KA_THREADS + threadIdx.x < units ? j * KA_THREADS + threadIdx.x : units - 1;
    const int h = head0 + i / per_row, kh = h - a.q_heads, vh = kh - a.kv_heads;
    const uint16_t *q = q_row + h * a.q.head_stride, *k = k_row + kh * a.k.head_stride, *v = v_row + vh * a.v.head_stride;
    const uint16_t *src = kh < 0 ? q : vh < 0 ? k : v;
    mine[j] = bit_cast<uint4>(__builtin_nontemporal_load(reinterpret_cast<const i32x4 *>(src + i % per_row * 8)));
  }
  int64_t first, len, past;
  SegChain chain;
  int64_t seg = nearest.find(row, a.offsets, a.lens, a.m, a.n, 0, chain, first, len, past);
  for (int64_t base = WAVE; seg < 0 && base < a.m; base += WAVE * KA_SEGMENTS) {
    Look<KA_SEGMENTS> more;
    more.load(a.offsets, a.lens, a.pages.past_lens, a.m, a.n, base);
    const int at = more.find(row, a.offsets, a.lens, a.m, a.n, base, chain, first, len, past);
    if (at >= 0) seg = base + at;
  }
  if (blockIdx.x == 0 && blockIdx.y == 0) report_segments(a.offsets, a.lens, a.m, a.n, a.failure, a.code);
  if (seg < 0) return;
  const int64_t room = a.pages.capacity();
  if (past < 0 || past > room || len > room - past) {
    if (a.failure != nullptr) *a.failure = a.code;
    return;
  }
  const int64_t pos = past + (row - first);
  const int64_t page = scalar_load(a.pages.table + seg * a.pages.cols + (pos >> a.pages.page_shift));
  if ((int)threadIdx.x < half) {
    // The angle in turns, reduced in f64: a far position times a frequency near 1
    // leaves few bits of the angle in f32.  What remains is at most half a turn and
    // is rounded to f32 (an error of at most 2^-25 turns of its size).
    const double turns = (double)pos * (double)freq * 0.15915494309189533577;
    const float part = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * part, &s, &c);
    cosine[threadIdx.x] = c;
    sine[threadIdx.x] = s;
  }
#pragma unroll
  for (int j = 0; j < KA_UNITS; j++) rows[j * KA_THREADS + threadIdx.x] = mine[j];
  __syncthreads();
  const int64_t slot = pos & (((int64_t)1 << a.pages.page_shift) - 1);
  const bool stored = page >= 0 && page < a.pages.n_pages;
  if (!stored && a.failure != nullptr) *a.failure = a.code;
#pragma unroll
  for (int j = 0; j < KA_UNITS; j++) {
    const int i = j * KA_THREADS + threadIdx.x;
    if (i >= units) break;
    const int h = head0 + i / per_row, kh = h - a.q_heads, c0 = i % per_row * 8;
    uint4 x = mine[j];
    if (kh < a.kv_heads && c0 < a.rot) {
      uint16_t in[8], out[8];
      *reinterpret_cast<uint4 *>(in) = x;
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const bool turned = c0 + e < a.rot;
          const float u = E::load(in[e]), v = E::load(in[e + 1]);
          const float c = turned ? cosine[(c0 + e) / 2] : 1.0f, s = turned ? sine[(c0 + e) / 2] : 0.0f;
          out[e] = turned ? E::store(u * c - v * s) : in[e];
          out[e + 1] = turned ? E::store(v * c + u * s) : in[e + 1];
        }
      } else {
        const uint16_t *whole = reinterpret_cast<const uint16_t *>(rows + (i - i % per_row));
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int at = c0 + e;
          const bool turned = at < a.rot, upper = at >= half;
          const int pair = turned ? (upper ? at - half : at) : 0;
          const float u = E::load(in[e]), v = E::load(whole[turned ? (upper ? at - half : at + half) : 0]);
          out[e] = turned ? E::store(upper ? u * cosine[pair] + v * sine[pair] : u * cosine[pair] - v * sine[pair]) : in[e];
        }
      }
      x = *reinterpret_cast<const uint4 *>(out);
    }
    if (kh < 0) {
      __builtin_nontemporal_store(bit_cast<i32x4>(x), reinterpret_cast<i32x4 *>(a.q_out.at(row, h) + c0));
    } else if (stored) {
      const bool is_v = kh >= a.kv_heads;
      uint16_t *pages = is_v ? a.pages.v : a.pages.k;
      __builtin_nontemporal_store(bit_cast<i32x4>(x), reinterpret_cast<i32x4 *>(
          pages + (a.pages.row_of(page, is_v ? kh - a.kv_heads : kh, a.kv_heads) + slot) * a.dim + c0));
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
  if (n > AT_MOST_BLOCKS) return FA_ENOTSUP;  // a row of blocks a token
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
  AppendArgs a = {to_heads(q != nullptr ? q : &none), to_heads(q != nullptr ? q_out : &none), to_heads(k),
                  to_heads(v), n, q != nullptr ? (int)heads : 0, (int)kv_heads, (int)head_dim, 0, offsets, lens, m,
                  freqs, (int)rot_dim, interleaved, to_pages(k_pages, v_pages, n_pages, page_size, page_table,
                  table_cols, past_lens), failure, code};
  // Heads a block takes: as many as its threads hold, fewer while there are few
  // tokens (two blocks a CU).
  const int64_t all = a.q_heads + 2 * a.kv_heads, most = KA_THREADS * KA_UNITS / (head_dim / 8);
  int64_t block_heads = ceil_div(all * n, 2 * NUM_CUS_HINT);
  if (block_heads < ceil_div(all, 65535)) block_heads = ceil_div(all, 65535);
  if (block_heads > most) block_heads = most;
  a.block_heads = (int)block_heads;
  const dim3 grid((unsigned)n, (unsigned)ceil_div(all, block_heads));
  if (t == FA_F16) kv_append_kernel<ElemF16><<<grid, KA_THREADS, 0, (hipStream_t)stream>>>(a);
  else kv_append_kernel<ElemBF16><<<grid, KA_THREADS, 0, (hipStream_t)stream>>>(a);
  return launch_status();
}
