// Attention over packed sequences and over a paged cache: forward.
//
// A block takes 128 query rows of one key head: the query heads of the group
// side by side for each of 128 / group tokens, so that keys and values are
// fetched once for the group.  A wave owns 32 of the rows and walks the keys 64
// at a time with the running maximum and sum of the softmax:
//   S^T = K Q^T      keys are rows, query rows are columns: a lane holds 32 of the
//                    64 scores of ONE query row, its partner in the other half of
//                    the wave the rest, and maximum, sum and weights need no
//                    exchange but one with that partner;
//   O^T += V^T P^T   the weights are the right operand as they stand in their
//                    registers (TileReads::columns reads V in the matching key order),
//                    and a lane's column of O^T is its query row again, so that
//                    rescaling is a multiplication by the lane's own factor.
// Keys and values go from memory straight into LDS, double buffered, one
// barrier per 64 keys.  Weights are rounded to the element type for the second
// product (the matrix units take nothing wider at this rate); sums stay f32.
//
// Bound by the matrix units at the clock that the card's power allows: nine prompts
// of up to 8192 tokens, 32 + 8 heads of 128, 1.6 ms or 0.98 PFLOP/s, the units busy
// half of the time at 1.9 GHz (a product of two 8192 x 8192 matrices: 1.38).  Two
// blocks a CU hide each other's softmax; one with 64 rows a wave, half the LDS reads
// and products and weights issued in turn by hand ran at 2.3 GHz and took 1.84 ms.
// Calls of few tiles are bound by the chain segments, rows, keys, steps, output:
// forty prompts of up to 333 tokens, 12 heads of 64, 13 us.
#include "attention.hip.h"

namespace fa {

constexpr int AT_WAVES = 4, AT_THREADS = AT_WAVES * WAVE;
constexpr int AT_ROWS = 32 * AT_WAVES;  // query rows a block
constexpr int AT_KEYS = 64;             // keys a step

// Keys, values and query rows a block works on.
struct Unit {
  int64_t seg, q_first, k_first;
  int tokens, t0, q_len, k_len;  // tokens of the tile, its first one, lengths
  int kv_head;
};

template <bool PAGED>
__device__ __forceinline__ bool find_unit(const AttentionArgs &a, int64_t number, int per_tile, Unit &u) {
  SegTile t;
  if (a.by_keys) {
    const int64_t i = lane_id() < a.m ? lane_id() : a.m - 1;
    int64_t first, len, first2 = 0, len2;
    bool ok = segment_ok(a.q_offsets, a.q_lens, i, a.q_rows, first, len) & (lane_id() < a.m), found;
    if constexpr (PAGED) {
      const int64_t past = a.pages.past_lens[i], room = a.pages.capacity();
      const bool fits = past >= 0 && past <= room && len <= room - past;
      ok = SegChain().keep(ok, first, len, a.q_offsets, a.q_lens, a.m, a.q_rows, 0);
      if (number == 0 && ok && len > 0 && !fits && a.failure != nullptr) *a.failure = a.code;
      ok = ok & fits;
      len2 = past + len;
    } else {
      const bool ok2 = segment_ok(a.k_offsets, a.k_lens, i, a.k_rows, first2, len2);
      ok = SegChain().keep(ok, first, len, a.q_offsets, a.q_lens, a.m, a.q_rows, 0) &
           SegChain().keep(ok2, first2, len2, a.k_offsets, a.k_lens, a.m, a.k_rows, 0);
    }
    find_tile_by_keys(ok, first, len, first2, len2, len2, per_tile, a.causal, number / a.kv_heads, t, found);
    if (!found) return false;
  } else if (!find_tile(a.q_offsets, a.q_lens, a.q_rows, PAGED ? nullptr : a.k_offsets, a.k_lens, a.k_rows, a.m,
                        per_tile, number / a.kv_heads, t)) {
    return false;
  }
  u.kv_head = (int)(number % a.kv_heads);
  u.seg = t.seg;
  u.q_first = t.first;
  u.q_len = (int)t.len;
  u.k_first = t.first2;
  u.k_len = (int)t.len2;
  if constexpr (PAGED) {
    const int64_t past = a.pages.past_lens[t.seg], room = a.pages.capacity();
    if (past < 0 || past > room || t.len > room - past) {
      if (a.failure != nullptr) *a.failure = a.code;
      return false;
    }
    u.k_len = (int)(past + t.len);
  }
  u.t0 = (int)(t.tiles - 1 - t.tile) * per_tile;  // the last tokens see most: they start first
  u.tokens = u.q_len - u.t0 < per_tile ? u.q_len - u.t0 : per_tile;
  return true;
}

// What splits of a unit leave for the kernel that joins them: maximum and sum of
// every row, and the output so far, of which four components of every thread stand
// side by side as they do in the registers.
__device__ __forceinline__ float *part_ml(const AttentionArgs &a, int64_t unit, int split, int row) {
  return a.part_ml + 2 * ((unit * a.splits + split) * AT_ROWS + row);
}
template <int D> __device__ __forceinline__ f32x4 *part_o(const AttentionArgs &a, int64_t unit, int split, int four) {
  return reinterpret_cast<f32x4 *>(a.part_o + (unit * a.splits + split) * (AT_ROWS * D)) + four * AT_THREADS + threadIdx.x;
}

template <class E, int D, bool PAGED>
__global__ __launch_bounds__(AT_THREADS, 2) void attention_kernel(AttentionArgs a) {
  constexpr int TILE = TileLoads<D, AT_THREADS>::BYTES;   // 64 keys (or values)
  constexpr int LOADS = TileLoads<D, AT_THREADS>::COUNT;  // 16-byte loads a thread and tile
  extern __shared__ __align__(16) unsigned char lds[];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int half = lane >> 5;
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    report_segments(a.q_offsets, a.q_lens, a.m, a.q_rows, a.failure, a.code);
    if constexpr (!PAGED) report_segments(a.k_offsets, a.k_lens, a.m, a.k_rows, a.failure, a.code);
  }
  const int per_tile = AT_ROWS / a.group;
  Unit u;
  if (!find_unit<PAGED>(a, blockIdx.x, per_tile, u)) return;

  // This lane's query row, and the last key it, its wave and its block see.
  const int behind = a.causal ? u.k_len - u.q_len : 0;
  const auto last_key = [&](int token) { return a.causal ? u.t0 + token + behind : u.k_len - 1; };
  const int rows = u.tokens * a.group;
  const int row = wave * 32 + (lane & 31);
  const int my_row = row < rows ? row : rows - 1;
  const int token = my_row / a.group, head = u.kv_head * a.group + my_row % a.group;
  const int limit = last_key(token);
  const bool wave_works = wave * 32 < rows;
  const int wave_last = __builtin_amdgcn_readfirstlane(
      last_key(((wave + 1) * 32 < rows ? (wave + 1) * 32 - 1 : rows - 1) / a.group));
  const int wave_first = __builtin_amdgcn_readfirstlane(last_key(wave_works ? wave * 32 / a.group : 0));
  const int block_first = last_key(0), block_last = last_key(u.tokens - 1);
  const int keys = block_last + 1;  // all the block's rows see together
  int from = 0, to = keys;
  if constexpr (PAGED) {
    from = blockIdx.y * a.chunk;
    to = keys - from < a.chunk ? keys : from + a.chunk;
    if (from >= keys && blockIdx.y > 0) return;
  }

  const TileLoads<D, AT_THREADS> loads(a.dim);
  const TileReads<D> reads;
  const uint32_t lds_base = lds_address(lds);
  clear_unloaded<D>(lds, 4 * TILE, a.dim);
  int page = 0;  // paged: this lane's one of the page numbers of the tile fetched next
  const auto fetch_pages = [&](int key0) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      const int key = key0 + lane < to ? key0 + lane : to - 1;
      page = a.pages.table[u.seg * a.pages.cols + (key >> a.pages.page_shift)];
    }
  };
  const int64_t k_stride = PAGED ? a.dim : a.k.row_stride, v_stride = PAGED ? a.dim : a.v.row_stride;
  const uint32_t k_offset = loads.offset(k_stride), v_offset = loads.offset(v_stride);
  const int slot_mask = PAGED ? (1 << a.pages.page_shift) - 1 : 0;
  // The keys (values) from key0 on to the tile at LDS address `tile`.
  const auto fetch_one = [&](int key0, uint32_t tile, const uint16_t *pages, const Heads &x, int64_t stride,
                             uint32_t offset) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      const bool there = key0 + lane < to, named = page >= 0 && page < a.pages.n_pages;
      // Rows of a load in one page: its address is the same for all lanes.
      if (slot_mask >= loads.ROWS - 1 && __all(there && named)) {
        if (loads.live) {
#pragma unroll
          for (int i = 0; i < LOADS; i++) {
            const int r = loads.first_row + i * loads.STEP;
            const int64_t id = __builtin_amdgcn_readlane(page, r);
            load_to_lds(pages + (a.pages.row_of(id, u.kv_head, a.kv_heads) + ((key0 + r) & slot_mask)) * a.dim, offset,
                        loads.place(tile, i));
          }
        }
        return;
      }
      if (there && !named && a.failure != nullptr) *a.failure = a.code;
      const int safe = there && named ? page : -1;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const int id = __shfl(safe, loads.row(i));
        if (loads.live)
          loads.load(pages + (a.pages.row_of(id, u.kv_head, a.kv_heads) + ((key0 + loads.row(i)) & slot_mask)) * a.dim,
                     id >= 0, tile, i);
      }
    } else {
      const uint16_t *first = x.at(u.k_first + key0, u.kv_head);
      if (key0 + AT_KEYS <= to) loads.load(first, stride, offset, tile);
      else loads.load(first, stride, to - key0, tile);
    }
  };
  const auto fetch = [&](int key0, int stage) __attribute__((always_inline)) {
    const uint32_t tile = lds_base + stage * (2 * TILE);
    fetch_one(key0, tile, a.pages.k, a.k, k_stride, k_offset);
    fetch_one(key0, tile + TILE, a.pages.v, a.v, v_stride, v_offset);
  };
  // The tile at key0 has arrived in `stage`, the one behind it is on its way.
  const auto arrive_and_fetch = [&](int key0, int stage) __attribute__((always_inline)) {
    wait_loads();
    block_barrier();
    if (key0 + AT_KEYS < to) {
      fetch(key0 + AT_KEYS, stage ^ 1);
      fetch_pages(key0 + 2 * AT_KEYS);
    }
  };

  uint4 q[D / 16];
  {
    const uint16_t *src = a.q.at(u.q_first + u.t0 + token, head);
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) q[ks] = load_unit(src, ks * 16 + half * 8, a.dim);
  }
  f32x16 o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[dt][i] = 0.0f;
  float top = -INFINITY, sum = 0.0f;  // top: of scores times log2(e); sum: this lane's half

  // Scores of 32 keys, their maximum, their weights, and the weights' products
  // with the values.
  const auto scores = [&](const unsigned char *kt, int b) __attribute__((always_inline)) {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) s = E::mfma(reads.rows(kt, b * 32, ks), q[ks], s);
    return s;
  };
  const auto maximum = [&](const f32x16 &s) __attribute__((always_inline)) {
    float high = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) high = fmaxf(high, s[i]);
    return fold_halves(high, FMax()) * a.scale_log2;
  };
  const auto raise = [&](float high) __attribute__((always_inline)) {
    if (__any(high > top + AT_RESCALE)) {
      // (each row by its own scores alone: what other rows see changes no bit of it)
      const float now = high > top + AT_RESCALE ? high : top;
      const float factor = now == top ? 1.0f : exp2f(top - now);
      top = now;
      sum *= factor;
#pragma unroll
      for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] *= factor;
    }
  };
  const auto weigh = [&](const f32x16 &s, uint4 (&p)[2]) __attribute__((always_inline)) {
    const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int c = 0; c < 2; c++) {
      f32x8 w;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        w[i] = __builtin_amdgcn_exp2f(fmaf(s[c * 8 + i], a.scale_log2, -shift));
        sum += w[i];
      }
      p[c] = E::pack(w);
    }
  };
  const auto values = [&](const unsigned char *vt, int b, const uint4 (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
      for (int dt = 0; dt < D / 32; dt++) o[dt] = E::mfma(reads.columns(vt, b * 32 + c * 16, dt), p[c], o[dt]);
  };

  // A tile of which rows of the block see different keys, or that is not full.
  const auto border = [&](int key0, int stage) __attribute__((always_inline)) {
    arrive_and_fetch(key0, stage);
    unsigned char *kt = lds + stage * (2 * TILE), *vt = kt + TILE;
    // A value that a row does not see must not reach it, and 0 * NaN would.
    bool unsafe = false;
    if (block_first < block_last) {
      bool found = false;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const uint4 x = *reinterpret_cast<const uint4 *>(vt + (i * AT_THREADS + threadIdx.x) * 16);
        for (uint32_t w : {x.x, x.y, x.z, x.w})
          found = found || (w & E::exponent) == E::exponent || (w >> 16 & E::exponent) == E::exponent;
      }
      unsafe = __syncthreads_or(found);
    }
    const bool active = wave_works && key0 <= wave_last;
    uint4 p[2][2];
    if (active) {
      f32x16 s[2];
#pragma unroll
      for (int b = 0; b < 2; b++) s[b] = scores(kt, b);
      if (key0 + AT_KEYS - 1 > wave_first) {
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (key0 + b * 32 + 8 * (i >> 2) + 4 * half + (i & 3) > limit) s[b][i] = -INFINITY;
      }
      raise(fmaxf(maximum(s[0]), maximum(s[1])));
#pragma unroll
      for (int b = 0; b < 2; b++) weigh(s[b], p[b]);
    }
    if (unsafe) {
      // Add what the rows see of the values that are not finite, one by one, and
      // take them out of the tile.
      if (active) {
        for (int j = 0; j < AT_KEYS && key0 + j < to; j++) {
#pragma unroll
          for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int d = dt * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
              const uint16_t bits = *reinterpret_cast<const uint16_t *>(vt + tile_offset<D>(j, d >> 3) + (d & 7) * 2);
              if ((bits & E::exponent) == E::exponent && key0 + j <= limit) o[dt][i] += E::load(bits);
            }
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < LOADS * 8; i++) {
        uint16_t *x = reinterpret_cast<uint16_t *>(vt) + (i / 8 * AT_THREADS + threadIdx.x) * 8 + i % 8;
        if ((*x & E::exponent) == E::exponent) *x = 0;
      }
      __syncthreads();
    }
    if (active) {
#pragma unroll
      for (int b = 0; b < 2; b++) values(vt, b, p[b]);
    }
  };

  // A tile that is full and that all rows of the block see.
  const auto inner = [&](int key0, int stage) __attribute__((always_inline)) {
    arrive_and_fetch(key0, stage);
    const unsigned char *kt = lds + stage * (2 * TILE), *vt = kt + TILE;
    if (wave_works) {
      f32x16 s[2];
#pragma unroll
      for (int b = 0; b < 2; b++) s[b] = scores(kt, b);
      raise(fmaxf(maximum(s[0]), maximum(s[1])));
      uint4 p[2][2];
#pragma unroll
      for (int b = 0; b < 2; b++) weigh(s[b], p[b]);
#pragma unroll
      for (int b = 0; b < 2; b++) values(vt, b, p[b]);
    }
  };
  const int full = block_first + 1 < to ? block_first + 1 : to;  // keys before it are seen by all rows
  const int tiles = full > from ? (full - from) / AT_KEYS : 0;
  arrived(q);
  fetch_pages(from);
  if (from < to) fetch(from, 0);
  fetch_pages(from + AT_KEYS);
  int t = 0;
  for (; t < tiles; t++) inner(from + t * AT_KEYS, t & 1);
  for (; from + t * AT_KEYS < to; t++) border(from + t * AT_KEYS, t & 1);

  sum = fold_halves(sum, FAdd());
  const bool there = row < rows;
  if (PAGED && keys > a.chunk) {
    if (!there) return;
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *part_o<D>(a, blockIdx.x, blockIdx.y, dt * 4 + i / 4) = f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
    if (half == 0) *reinterpret_cast<f32x2 *>(part_ml(a, blockIdx.x, blockIdx.y, row)) = f32x2{top, sum};
    return;
  }
  const int64_t out_row = u.q_first + u.t0 + token;
  const bool empty = sum == 0.0f;  // saw nothing, or only scores of -inf (and no NaN)
  const float inverse = empty ? 0.0f : 1.0f / sum;
  store_column<E, D>(o, inverse, a.out.at(out_row, head), a.dim, there, empty);
  if (a.lse != nullptr && half == 0 && there)
    a.lse[out_row * a.heads + head] = empty ? -INFINITY : (top + log2f(sum)) * LN2;
}

// Joins the parts of the units whose keys were split: a block a unit and 32
// components, laid out as the block that left them.
template <class E, int D> __global__ __launch_bounds__(AT_THREADS) void attention_join_kernel(AttentionArgs a) {
  const int per_tile = AT_ROWS / a.group;
  Unit u;
  if (!find_unit<true>(a, blockIdx.x, per_tile, u)) return;
  const int keys = u.t0 + u.tokens + u.k_len - u.q_len, dt = blockIdx.y;
  if (keys <= a.chunk || dt * 32 >= a.dim) return;
  const int row = threadIdx.x / WAVE * 32 + (lane_id() & 31), rows = u.tokens * a.group;
  const int splits = (keys - 1) / a.chunk + 1;  // (the sum of the two may pass 2^31)
  float top = -INFINITY;
  for (int s = 0; s < splits; s++) top = fmaxf(top, part_ml(a, blockIdx.x, s, row)[0]);
  const float shift = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  f32x16 o[1];
#pragma unroll
  for (int i = 0; i < 16; i++) o[0][i] = 0.0f;
  for (int s = 0; s < splits; s++) {
    const f32x2 ml = *reinterpret_cast<const f32x2 *>(part_ml(a, blockIdx.x, s, row));
    const float f = exp2f(ml[0] - shift);
    sum += f * ml[1];
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const f32x4 x = *part_o<D>(a, blockIdx.x, s, dt * 4 + i / 4);
#pragma unroll
      for (int j = 0; j < 4; j++) o[0][i + j] += f * x[j];
    }
  }
  const bool there = row < rows, empty = sum == 0.0f;
  const int my_row = there ? row : 0, head = u.kv_head * a.group + my_row % a.group;
  const int64_t out_row = u.q_first + u.t0 + my_row / a.group;
  store_column<E, 32>(o, 1.0f / sum, a.out.at(out_row, head) + dt * 32, a.dim - dt * 32, there, empty);
  if (a.lse != nullptr && dt == 0 && there && lane_id() < 32)
    a.lse[out_row * a.heads + head] = empty ? -INFINITY : (top + log2f(sum)) * LN2;
}

// How a cache's keys are split over blocks.  Lengths are not known here.  One
// sequence is taken to be as long as the table allows: as many blocks as run at a
// time (two a CU).  Several are ragged: twice as many, at least 256 keys to a block.
// (Twenty chunks of up to 300 tokens behind up to 4096 105 -> 74 us, two of 32 heads
// without groups 184 -> 117; six of up to 1024 behind up to 8192, which fill the chip
// unsplit, 266 -> 280.  Three times as many: 93, 127, 279.)  A table much wider than
// its sequences are long is split too coarsely: 100 tokens behind 8092 take 42 us with
// a table of their length and 203 with one of 131072 positions.
struct SplitPlan {
  int64_t units;
  int chunk, splits;
};
static SplitPlan split_plan(int64_t n, int64_t heads, int64_t kv_heads, int64_t m, int64_t capacity) {
  SplitPlan p;
  p.units = most_tiles(n, m, AT_ROWS / (heads / kv_heads)) * kv_heads;
  const int64_t blocks = (m > 1 ? 4 : 2) * NUM_CUS_HINT;
  const int64_t even = p.units < blocks ? ceil_div(capacity * p.units, blocks) : capacity;
  const int64_t chunk = ceil_div(even < 256 ? 256 : even, AT_KEYS) * AT_KEYS;
  p.chunk = (int)(chunk < capacity ? chunk : (capacity > 0 ? capacity : 1));
  p.splits = (int)(capacity > 0 ? ceil_div(capacity, p.chunk) : 1);
  return p;
}

template <bool PAGED> static int launch_attention(hipStream_t stream, fa_dtype t, const AttentionArgs &a, int64_t units) {
  if (units > AT_MOST_BLOCKS) return FA_ENOTSUP;
  const dim3 grid((unsigned)units, (unsigned)a.splits);
  const bool narrow = a.dim <= 64;
  const size_t lds = 4 * AT_KEYS * (narrow ? 64 : 128) * 2;
  if (t == FA_F16) {
    if (narrow) attention_kernel<ElemF16, 64, PAGED><<<grid, AT_THREADS, lds, stream>>>(a);
    else attention_kernel<ElemF16, 128, PAGED><<<grid, AT_THREADS, lds, stream>>>(a);
  } else {
    if (narrow) attention_kernel<ElemBF16, 64, PAGED><<<grid, AT_THREADS, lds, stream>>>(a);
    else attention_kernel<ElemBF16, 128, PAGED><<<grid, AT_THREADS, lds, stream>>>(a);
  }
  return launch_status();
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
  if ((rc = check_scale(scale)) != 0) return rc;
  if (q_rows == 0 || m == 0) return 0;
  rc = check_heads(q, q_rows, heads, head_dim, false);
  if (rc == 0) rc = check_heads(k, k_rows, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(v, k_rows, kv_heads, head_dim, false);
  if (rc == 0) rc = check_heads(out, q_rows, heads, head_dim, true);
  if (rc == 0 && !is_aligned(lse, 4)) rc = FA_EALIGN;
  if (rc != 0) return rc;
  AttentionArgs a = {};
  a.q = to_heads(q), a.k = to_heads(k), a.v = to_heads(v), a.out = to_heads(out);
  a.lse = lse;
  a.q_rows = q_rows, a.k_rows = k_rows;
  a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.group = (int)(heads / kv_heads), a.dim = (int)head_dim;
  a.q_offsets = q_offsets, a.q_lens = q_lens, a.k_offsets = k_offsets, a.k_lens = k_lens;
  a.m = m;
  a.scale_log2 = scale * LOG2E;
  a.causal = causal != 0;
  a.failure = failure, a.code = code;
  a.splits = 1;
  const int64_t units = most_tiles(q_rows, m, AT_ROWS / a.group) * kv_heads;
  a.by_keys = takes_by_keys(units, m, head_dim);
  return launch_attention<false>((hipStream_t)stream, t, a, units);
}

extern "C" size_t fa_attention_paged_workspace_bytes(int64_t n, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                     int64_t m, int64_t page_size, int64_t table_cols) {
  if (n <= 0 || m <= 0 || n > AT_MOST_ROWS || m > AT_MOST_ROWS || page_size <= 0 || table_cols < 0 ||
      (__int128)page_size * table_cols > AT_MOST_ROWS || check_shape(FA_F16, heads, kv_heads, head_dim) != 0)
    return 0;
  const int few = few_rows(n, heads, kv_heads, m);
  if (few > 0) return few_workspace(few, n, heads, kv_heads, head_dim, m, page_size * table_cols);
  const SplitPlan p = split_plan(n, heads, kv_heads, m, page_size * table_cols);
  if (p.splits == 1 || p.units > AT_MOST_BLOCKS) return 0;  // (more is refused)
  return (size_t)p.units * p.splits * AT_ROWS * ((head_dim <= 64 ? 64 : 128) + 2) * sizeof(float);
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
  if ((rc = check_scale(scale)) != 0) return rc;
  if (n == 0 || m == 0) return 0;
  rc = check_heads(q, n, heads, head_dim, false);
  if (rc == 0) rc = check_heads(out, n, heads, head_dim, true);
  if (rc == 0) rc = check_pages(k_pages, v_pages, n_pages, page_size, page_table, table_cols, past_lens, kv_heads, head_dim);
  if (rc == 0 && !is_aligned(lse, 4)) rc = FA_EALIGN;
  if (rc != 0) return rc;
  const size_t need = fa_attention_paged_workspace_bytes(n, heads, kv_heads, head_dim, m, page_size, table_cols);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need) return FA_ESCRATCH;
    if (!is_aligned(workspace, 16)) return FA_EALIGN;
  }
  const int few = few_rows(n, heads, kv_heads, m);
  AttentionArgs a = {};
  a.q = to_heads(q), a.out = to_heads(out);
  a.lse = lse;
  a.q_rows = n;
  a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.group = (int)(heads / kv_heads), a.dim = (int)head_dim;
  a.q_offsets = offsets, a.q_lens = lens;
  a.m = m;
  a.scale_log2 = scale * LOG2E;
  a.causal = 1;
  a.failure = failure, a.code = code;
  a.pages = to_pages(k_pages, v_pages, n_pages, page_size, page_table, table_cols, past_lens);
  if (few > 0) return launch_few((hipStream_t)stream, t, few, a, workspace);
  const SplitPlan p = split_plan(n, heads, kv_heads, m, page_size * table_cols);
  a.chunk = p.chunk, a.splits = p.splits;
  a.by_keys = takes_by_keys(p.units, m, head_dim);
  if (p.splits > 1) {
    const int64_t parts = p.units * p.splits * AT_ROWS;
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o + parts * (head_dim <= 64 ? 64 : 128);
  }
  rc = launch_attention<true>((hipStream_t)stream, t, a, p.units);
  if (rc != 0 || p.splits == 1) return rc;
  const dim3 grid((unsigned)p.units, head_dim <= 64 ? 2 : 4);
  if (t == FA_F16) {
    if (head_dim <= 64) attention_join_kernel<ElemF16, 64><<<grid, AT_THREADS, 0, (hipStream_t)stream>>>(a);
    else attention_join_kernel<ElemF16, 128><<<grid, AT_THREADS, 0, (hipStream_t)stream>>>(a);
  } else {
    if (head_dim <= 64) attention_join_kernel<ElemBF16, 64><<<grid, AT_THREADS, 0, (hipStream_t)stream>>>(a);
    else attention_join_kernel<ElemBF16, 128><<<grid, AT_THREADS, 0, (hipStream_t)stream>>>(a);
  }
  return launch_status();
}
