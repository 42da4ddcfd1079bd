// Gradients of attention over packed sequences, in two passes without atomics: one
// owns query rows (dq), one owns keys (dk and dv); each computes the scores again.
// Both are bound by the matrix units at the clock that power allows, on long
// sequences 1.2 and 1.08 PFLOP/s of the products they compute (one of 8192 tokens,
// not causal, 32 + 8 heads of 128: 1.36 and 2.04 ms).  On ragged ones (five of up
// to 4096: 271 and 430 us on average under the profiler, 261 and 394 at best, the
// units busy 55 and 43 % of the time) about 13 us of a key tile are its beginning and
// end.  Weights and derivatives of scores are rounded to the element type once, for
// the products that they enter; sums, shifts and D are f32.
#include "attention.hip.h"

namespace fa {

constexpr int AG_WAVES = 4, AG_THREADS = AG_WAVES * WAVE;
constexpr int AG_ROWS = 32 * AG_WAVES;  // query rows a block of the first kernel owns
constexpr int AG_STEP = 64;             // keys (query rows) a step
// A row of few keys has an output as large as its values, and D taken from the
// rounded output is then off by as much as a rounding of the scores' derivative;
// rows with fewer keys than this take D from the weights instead.
constexpr int AG_EXACT_KEYS = 64;
// A key tile's rows are split into up to AG_MOST_PARTS parts.
constexpr int AG_MOST_PARTS = 8;
// Steps that are worth a part of their own, by the rounds that AG_MOST_PARTS of every
// tile would take: the fewer there are, the longer the chip would wait for the
// longest tile.  (32 steps, against 4: one sequence of 512, 32 + 8 heads of 128,
// forward and backward 109 and 70 us, four of up to 700, 8 + 2 heads, 114 and 76;
// against 8: three of up to 700, 32 + 8 heads, 118 and 89, one of 1024 140 and 127.)
constexpr int part_steps_for(int64_t rounds) { return rounds <= 1 ? 4 : rounds <= 4 ? 8 : 32; }

struct GradArgs {
  Heads q, k, v, out, dout, dq, dk, dv;
  const float *lse;
  float *shift, *delta;  // [q_rows][heads]: lse times log2(e), infinite for a row that sees nothing; D
  float *part;   // sums of the parts of split key tiles
  int64_t q_rows, k_rows;
  int heads, kv_heads, group, dim;
  const int64_t *q_offsets, *q_lens, *k_offsets, *k_lens;
  int64_t m;
  float scale;
  int causal, parts, part_steps;
  bool by_keys, by_rows;  // the order of dq's tiles, and of dk's and dv's
  int32_t *failure, code;
};

template <int D> __device__ __forceinline__ void load_operand(uint4 (&x)[D / 16], const uint16_t *src, int dim) {
#pragma unroll
  for (int s = 0; s < D / 16; s++) x[s] = load_unit(src, s * 16 + (lane_id() >> 5) * 8, dim);
}
template <int D> __device__ __forceinline__ void clear(f32x16 (&x)[D / 32]) {
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) x[t][i] = 0.0f;
}
// dq and D.  Laid out as the forward kernel: 128 query rows of a key head, a wave
// owns 32 of them, 64 keys a step;
//   S^T = K Q^T, dP^T = V dO^T, dS^T = P^T (dP^T - D), dQ^T += K^T dS^T,
// where K is read from one tile both by rows and by columns.
template <class E, int D> __global__ __launch_bounds__(AG_THREADS, 2) void attention_dq_kernel(GradArgs a) {
  constexpr int TILE = TileLoads<D, AG_THREADS>::BYTES;
  extern __shared__ __align__(16) unsigned char lds[];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = lane >> 5;
  if (blockIdx.x == 0) {
    report_segments(a.q_offsets, a.q_lens, a.m, a.q_rows, a.failure, a.code);
    report_segments(a.k_offsets, a.k_lens, a.m, a.k_rows, a.failure, a.code);
  }
  const int per_tile = AG_ROWS / a.group, kv_head = blockIdx.x % a.kv_heads;
  SegTile t;
  if (a.by_keys) {
    const int64_t i = lane_id() < a.m ? lane_id() : a.m - 1;
    int64_t first, len, first2, len2;
    bool ok = segment_ok(a.q_offsets, a.q_lens, i, a.q_rows, first, len) & (lane_id() < a.m), found;
    const bool ok2 = segment_ok(a.k_offsets, a.k_lens, i, a.k_rows, first2, len2);
    ok = SegChain().keep(ok, first, len, a.q_offsets, a.q_lens, a.m, a.q_rows, 0) &
         SegChain().keep(ok2, first2, len2, a.k_offsets, a.k_lens, a.m, a.k_rows, 0);
    find_tile_by_keys(ok, first, len, first2, len2, len2, per_tile, a.causal, blockIdx.x / a.kv_heads, t, found);
    if (!found) return;
  } else if (!find_tile(a.q_offsets, a.q_lens, a.q_rows, a.k_offsets, a.k_lens, a.k_rows, a.m, per_tile,
                        blockIdx.x / a.kv_heads, t)) {
    return;
  }
  const int q_len = (int)t.len, k_len = (int)t.len2;
  const int t0 = (int)(t.tiles - 1 - t.tile) * per_tile;  // the last tokens see most: they start first
  const int tokens = q_len - t0 < per_tile ? q_len - t0 : per_tile;
  const int behind = k_len - q_len;
  const auto last_key = [&](int token) { return a.causal ? t0 + token + behind : k_len - 1; };
  const int rows = tokens * a.group, row = wave * 32 + (lane & 31);
  const int my_row = row < rows ? row : rows - 1;
  const int token = my_row / a.group, head = kv_head * a.group + my_row % a.group;
  const int limit = last_key(token);
  const bool wave_works = wave * 32 < rows;
  const int wave_last = __builtin_amdgcn_readfirstlane(
      last_key(((wave + 1) * 32 < rows ? (wave + 1) * 32 - 1 : rows - 1) / a.group));
  const int wave_first = __builtin_amdgcn_readfirstlane(last_key(wave_works ? wave * 32 / a.group : 0));
  const int keys = last_key(tokens - 1) + 1;

  const TileLoads<D, AG_THREADS> loads(a.dim);
  const TileReads<D> reads;
  const uint32_t lds_base = lds_address(lds);
  clear_unloaded<D>(lds, 4 * TILE, a.dim);
  const uint32_t k_offset = loads.offset(a.k.row_stride), v_offset = loads.offset(a.v.row_stride);
  const auto fetch = [&](int key0, int stage) __attribute__((always_inline)) {
    const uint16_t *k = a.k.at(t.first2 + key0, kv_head), *v = a.v.at(t.first2 + key0, kv_head);
    const uint32_t k_tile = lds_base + stage * (2 * TILE), v_tile = k_tile + TILE;
    if (key0 + AG_STEP <= keys) {
      loads.load(k, a.k.row_stride, k_offset, k_tile);
      loads.load(v, a.v.row_stride, v_offset, v_tile);
    } else {
      loads.load(k, a.k.row_stride, keys - key0, k_tile);
      loads.load(v, a.v.row_stride, keys - key0, v_tile);
    }
  };

  const int64_t at = t.first + t0 + token;
  uint4 q[D / 16], g[D / 16];
  load_operand<D>(q, a.q.at(at, head), a.dim);
  load_operand<D>(g, a.dout.at(at, head), a.dim);
  float delta = 0.0f;
  {
    uint4 o[D / 16];
    load_operand<D>(o, a.out.at(at, head), a.dim);
#pragma unroll
    for (int s = 0; s < D / 16; s++)
      for (int w = 0; w < 4; w++) {
        const uint32_t x = (&o[s].x)[w], y = (&g[s].x)[w];
        delta += E::load((uint16_t)x) * E::load((uint16_t)y) + E::load((uint16_t)(x >> 16)) * E::load((uint16_t)(y >> 16));
      }
    delta = fold_halves(delta, FAdd());
  }
  // A row that sees nothing has lse = -inf; its weights must come out as zero.
  const float lse = a.lse[at * a.heads + head];
  const float shift = lse == -INFINITY ? INFINITY : lse * LOG2E, scale_log2 = a.scale * LOG2E;
  arrived(q);
  arrived(g);
  f32x16 dq[D / 32];
  clear<D>(dq);

  // Weights and derivatives of their scores' products for keys b .. b+31 of the tile.
  const auto weights = [&](const unsigned char *kt, int key0, int b, f32x16 &p, f32x16 &dp) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; i++) p[i] = dp[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
      p = E::mfma(reads.rows(kt, b, s), q[s], p);
      dp = E::mfma(reads.rows(kt + TILE, b, s), g[s], dp);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], scale_log2, -shift));
    if (key0 + b + 31 > wave_first) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (key0 + b + 8 * (i >> 2) + 4 * half + (i & 3) > limit) p[i] = 0.0f;
    }
  };
  // All keys, `step` for each 64 of them.
  const auto walk = [&](auto step) __attribute__((always_inline)) {
    if (keys > 0) fetch(0, 0);
    int stage = 0;
    for (int key0 = 0; key0 < keys; key0 += AG_STEP, stage ^= 1) {
      wait_loads();
      __syncthreads();
      if (key0 + AG_STEP < keys) fetch(key0 + AG_STEP, stage ^ 1);
      if (wave_works && key0 <= wave_last) step(lds + stage * (2 * TILE), key0);
    }
  };
  if (last_key(0) < AG_EXACT_KEYS) {
    // A row of one key has the weight 1, whatever lse's rounding makes of it: its D is
    // dP itself, so that dP - D is zero here and, with the same products, for dk.
    float d = 0.0f, only = 0.0f;
    walk([&](const unsigned char *kt, int key0) __attribute__((always_inline)) {
      for (int b = 0; b < AG_STEP; b += 32) {
        f32x16 p, dp;
        weights(kt, key0, b, p, dp);
        if (key0 + b == 0 && half == 0) only = dp[0];
#pragma unroll
        for (int i = 0; i < 16; i++) d += p[i] * dp[i];
      }
    });
    delta = fold_halves(limit == 0 ? only : d, FAdd());
    __syncthreads();  // the tiles are read again from the start
  }
  if (row < rows && half == 0) {
    a.shift[at * a.heads + head] = shift;
    a.delta[at * a.heads + head] = delta;
  }
  walk([&](const unsigned char *kt, int key0) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < AG_STEP; b += 32) {
      f32x16 p, dp;
      weights(kt, key0, b, p, dp);
#pragma unroll
      for (int c = 0; c < 2; c++) {
        f32x8 w;
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = p[c * 8 + i] * (dp[c * 8 + i] - delta);
        const uint4 ds = E::pack(w);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
          dq[dt] = E::mfma(reads.columns(kt, b + c * 16, dt), ds, dq[dt]);
      }
    }
  });
  store_column<E, D>(dq, a.scale, a.dq.at(at, head), a.dim, row < rows);
}

// The query rows of a key tile, in steps of AG_STEP: `heads` query heads side by
// side (all of the group up to 64 of them, else in `chunks` rounds) for `tokens`
// tokens.
struct RowSteps {
  int heads, chunks, tokens, first, per_chunk;  // first token, steps of a chunk
  __device__ __forceinline__ RowSteps(int group, int q_len, int from) {
    heads = group < AG_STEP ? group : AG_STEP;
    chunks = (group + heads - 1) / heads;
    tokens = AG_STEP / heads;
    first = from;
    per_chunk = from < q_len ? (q_len - from + tokens - 1) / tokens : 0;
  }
  __device__ __forceinline__ int64_t count() const { return (int64_t)chunks * per_chunk; }
};
// A step: its first token and the first of its heads in the group.
struct StepAt {
  int token, head;
  __device__ __forceinline__ StepAt(const RowSteps &r, int64_t step) {
    const int chunk = r.chunks == 1 ? 0 : (int)(step / r.per_chunk);
    token = r.first + (int)(step - (int64_t)chunk * r.per_chunk) * r.tokens;
    head = chunk * r.heads;
  }
  __device__ __forceinline__ void advance(const RowSteps &r, int q_len) {
    token += r.tokens;
    if (token >= q_len) {
      token = r.first;
      head += r.heads;
    }
  }
};
__device__ __forceinline__ int parts_of(int64_t steps, int most, int part_steps) {
  const int64_t worth = (steps + part_steps - 1) / part_steps;
  return worth < 1 ? 1 : (worth < most ? (int)worth : most);
}
// First token that sees a key of the tile from key0 on.
__device__ __forceinline__ int first_token(const GradArgs &a, int key0, int q_len, int k_len) {
  const int from = a.causal ? key0 - (k_len - q_len) : 0;
  return from > 0 ? from : 0;
}
constexpr int AG_KEYS = 32 * AG_WAVES;  // keys a block of the second kernel owns
// Where part `part` of a key tile leaves its sums: dk then dv, and of each four
// components of every thread side by side, as they stand in the registers.
template <int D> __device__ __forceinline__ float *part_sums(const GradArgs &a, int64_t tile, int part) {
  return a.part + (tile * a.parts + part) * (2 * AG_KEYS * D);
}
// The key tile of this block, the one that most tokens see first if by_rows.
__device__ __forceinline__ bool find_key_tile(const GradArgs &a, SegTile &t) {
  const int64_t number = blockIdx.x / a.kv_heads;
  if (!a.by_rows)
    return find_tile(a.k_offsets, a.k_lens, a.k_rows, a.q_offsets, a.q_lens, a.q_rows, a.m, AG_KEYS, number, t);
  const int64_t i = lane_id() < a.m ? lane_id() : a.m - 1;
  int64_t first, len, first2, len2;
  bool ok = segment_ok(a.k_offsets, a.k_lens, i, a.k_rows, first, len) & (lane_id() < a.m), found;
  const bool ok2 = segment_ok(a.q_offsets, a.q_lens, i, a.q_rows, first2, len2);
  ok = SegChain().keep(ok, first, len, a.k_offsets, a.k_lens, a.m, a.k_rows, 0) &
       SegChain().keep(ok2, first2, len2, a.q_offsets, a.q_lens, a.m, a.q_rows, 0);
  find_tile_by_keys(ok, first, len, first2, len2, a.causal ? len : len2, AG_KEYS, a.causal, number, t, found);
  return found;
}

// Stages of 64 query rows in LDS: Q, dO, and of every row its shift and D; so many
// that rows have two steps to arrive.  Behind them, of every row of a step, which
// of the step's tokens it belongs to.
template <int D> struct GradStage {
  static constexpr int TILE = TileLoads<D, AG_THREADS>::BYTES, BYTES = 2 * TILE + 2 * AG_STEP * 4, COUNT = 4;
  static constexpr int TOKENS = COUNT * BYTES, LDS = TOKENS + AG_STEP * 4;
};
static __device__ const float g_infinity = INFINITY;  // the shift of a row that is not there (its D is 0)

// dk and dv.  A block owns 128 keys of a key head, a wave 32 of them with K and V
// as right operands in registers, and walks the query rows that see them, all
// heads of the group, 64 a step and 32 at a time:
//   S = Q K^T, dP = dO V^T, dS = P (dP - D), dV^T += dO^T P, dK^T += Q^T dS,
// with Q and dO read from one tile each by rows and by columns.  The products S
// and dP of the next 32 rows are issued in turn with the weights of the last, as
// the order in the source fixes.  (All four waves read the same rows of LDS; 64 keys
// a wave would halve those reads, but its sums, operands and products need more than
// the 512 registers of a lane, and the spills took 2.4 times as long.  From the last
// step to the first, so that blocks side by side read the same rows: the same time,
// D = 64 3 % more.)  The keys at the start of a long sequence are
// seen by all its rows: their rows are split over `parts` blocks, whose sums a
// second kernel adds in order.
template <class E, int D> __global__ __launch_bounds__(AG_THREADS, D == 128 ? 1 : 2) void attention_dkv_kernel(GradArgs a) {
  using L = GradStage<D>;
  constexpr int TILE = L::TILE, PRODUCTS = D / 8;  // of S and dP together, and of dV and dK
  constexpr int AHEAD = D == 128 ? 3 : 2;          // operands read before their product (as registers allow)
  extern __shared__ __align__(16) unsigned char lds[];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = lane >> 5;
  const int kv_head = blockIdx.x % a.kv_heads;
  if (a.q_rows == 0 && blockIdx.x == 0 && blockIdx.y == 0) {  // (without query rows the dq kernel is not launched)
    report_segments(a.q_offsets, a.q_lens, a.m, a.q_rows, a.failure, a.code);
    report_segments(a.k_offsets, a.k_lens, a.m, a.k_rows, a.failure, a.code);
  }
  const int part = gridDim.y - 1 - blockIdx.y;  // tiles of many parts, the long ones, start first
  SegTile t;
  if (!find_key_tile(a, t)) return;
  const int k_len = (int)t.len, q_len = (int)t.len2, key0 = (int)t.tile * AG_KEYS, behind = k_len - q_len;
  const RowSteps steps(a.group, q_len, first_token(a, key0, q_len, k_len));
  const int parts = parts_of(steps.count(), a.parts, a.part_steps);
  if (part >= parts) return;
  const int64_t from = steps.count() * part / parts, to = steps.count() * (part + 1) / parts;

  const int key = key0 + wave * 32 + (lane & 31);
  uint4 k[D / 16], v[D / 16];
  {
    const int64_t at = t.first + (key < k_len ? key : k_len - 1);
    load_operand<D>(k, a.k.at(at, kv_head), a.dim);
    load_operand<D>(v, a.v.at(at, kv_head), a.dim);
  }
  arrived(k);
  arrived(v);
  f32x16 dk[D / 32], dv[D / 32];
  clear<D>(dk);
  clear<D>(dv);

  const TileLoads<D, AG_THREADS> loads(a.dim);
  const TileReads<D> reads;
  const uint32_t lds_base = lds_address(lds);
  clear_unloaded<D>(lds, L::TOKENS, a.dim);
  int *tokens_of = reinterpret_cast<int *>(lds + L::TOKENS);
  if (wave < 2) tokens_of[lane] = lane / steps.heads;  // (both, for their own loads below)
  // Row r of a step is token r / heads, head r % heads of the step's.  The usual
  // case: all rows of a step used, and within 32-bit offsets of its first.
  const bool near = steps.tokens * steps.heads == AG_STEP &&
                    ((int64_t)AG_STEP * (a.q.row_stride + a.dout.row_stride) +
                     steps.heads * (a.q.head_stride + a.dout.head_stride)) < (1 << 30);
  uint32_t q_at[loads.COUNT], g_at[loads.COUNT];
#pragma unroll
  for (int i = 0; i < loads.COUNT; i++) {
    const int r = loads.row(i);
    q_at[i] = (uint32_t)(r / steps.heads * a.q.row_stride + r % steps.heads * a.q.head_stride + loads.unit * 8) * 2;
    g_at[i] = (uint32_t)(r / steps.heads * a.dout.row_stride + r % steps.heads * a.dout.head_stride + loads.unit * 8) * 2;
  }
  // Loads of a step: FETCHES of every wave, and one more of the first two.
  constexpr int FETCHES = 2 * TileLoads<D, AG_THREADS>::COUNT;
  const auto fetch = [&](const StepAt &s, int stage) __attribute__((always_inline)) {
    const uint32_t q_tile = lds_base + stage * L::BYTES, g_tile = q_tile + TILE;
    const int head = kv_head * a.group + s.head;
    if (near && s.token + steps.tokens <= q_len && s.head + steps.heads <= a.group) {
      const uint16_t *q0 = a.q.at(t.first2 + s.token, head), *g0 = a.dout.at(t.first2 + s.token, head);
      if (loads.live) {
#pragma unroll
        for (int i = 0; i < loads.COUNT; i++) {
          load_to_lds(q0, q_at[i], loads.place(q_tile, i));
          load_to_lds(g0, g_at[i], loads.place(g_tile, i));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < loads.COUNT; i++) {
        const int token = loads.row(i) / steps.heads, h = loads.row(i) % steps.heads;
        const bool there = token < steps.tokens && s.token + token < q_len && s.head + h < a.group;
        if (loads.live) {
          loads.load(a.q.at(t.first2 + s.token + token, head + h), there, q_tile, i);
          loads.load(a.dout.at(t.first2 + s.token + token, head + h), there, g_tile, i);
        }
      }
    }
    if (wave < 2) {
      const int my_token = tokens_of[lane], my_head = lane - my_token * steps.heads;
      const bool there = my_token < steps.tokens && s.token + my_token < q_len && s.head + my_head < a.group;
      const float *src = (wave == 0 ? a.shift : a.delta) + (t.first2 + s.token + my_token) * a.heads + head + my_head;
      const void *none = wave == 0 ? (const void *)&g_infinity : (const void *)&g_zeros;
      load_word_to_lds(there ? (const void *)src : none, g_tile + TILE + wave * (AG_STEP * 4));
    }
  };
  // All loads but those of the youngest step have arrived.
  const auto wait_for_older = [&]() {
    if (wave < 2) wait_but<FETCHES + 1>();
    else wait_but<FETCHES>();
  };
  const float scale_log2 = a.scale * LOG2E;

  // Operand `i` of the products S and dP (in turn) of 32 rows, and of dV and dK.
  const auto by_rows = [&](const unsigned char *tile, int b, auto i) __attribute__((always_inline)) {
    return reads.rows(tile + (i % 2 ? TILE : 0), b, i / 2);
  };
  const auto by_columns = [&](const unsigned char *tile, int b, auto i) __attribute__((always_inline)) {
    constexpr int c = i / (D / 16), dt = i % (D / 16) / 2;
    return reads.columns(tile + (i % 2 ? 0 : TILE), b + 16 * c, dt);
  };
  const auto products = [&](const unsigned char *tile, int b, f32x16 &s, f32x16 &dp) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = dp[i] = 0.0f;
    static_for<PRODUCTS>([&](auto i) __attribute__((always_inline)) {
      if constexpr (i % 2 == 0) s = E::mfma(by_rows(tile, b, i), k[i / 2], s);
      else dp = E::mfma(by_rows(tile, b, i), v[i / 2], dp);
    });
  };
  // 32 rows (`tile`, from b on) whose products are s and dp; and the products of
  // the next 32 (`next_tile`, from next_b on).  If masked, the step's tokens from
  // first_seen on see this lane's key.
  const auto half_step = [&](const unsigned char *tile, int b, f32x16 &s, f32x16 &dp, const unsigned char *next_tile,
                             int next_b, f32x16 &next_s, f32x16 &next_dp, int first_seen, auto masked)
      __attribute__((always_inline)) {
    const float *shifts = reinterpret_cast<const float *>(tile + 2 * TILE) + b + 4 * half, *deltas = shifts + AG_STEP;
    uint4 x[AHEAD];
    uint32_t pw[8], pds[8];
    f32x4 shift[4], delta[4];
    int4 token[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      shift[j] = *reinterpret_cast<const f32x4 *>(shifts + 8 * j);
      delta[j] = *reinterpret_cast<const f32x4 *>(deltas + 8 * j);
      if constexpr (decltype(masked)::value) token[j] = *reinterpret_cast<const int4 *>(tokens_of + b + 4 * half + 8 * j);
    }
    static_for<AHEAD>([&](auto i) __attribute__((always_inline)) { x[i] = by_rows(next_tile, next_b, i); });
#pragma unroll
    for (int i = 0; i < 16; i++) next_s[i] = next_dp[i] = 0.0f;
    __builtin_amdgcn_sched_barrier(0);
    static_for<PRODUCTS>([&](auto i) __attribute__((always_inline)) {
      const uint4 now = x[i % AHEAD];
      if constexpr (i + AHEAD < PRODUCTS) x[i % AHEAD] = by_rows(next_tile, next_b, std::integral_constant<int, i + AHEAD>());
      else x[i % AHEAD] = by_columns(tile, b, std::integral_constant<int, i + AHEAD - PRODUCTS>());
      if constexpr (i % 2 == 0) next_s = E::mfma(now, k[i / 2], next_s);
      else next_dp = E::mfma(now, v[i / 2], next_dp);
      constexpr int SHARE = 16 / PRODUCTS;
      static_for<SHARE>([&](auto j) __attribute__((always_inline)) {
        constexpr int e = i * SHARE + j;
        float p = __builtin_amdgcn_exp2f(fmaf(s[e], scale_log2, -shift[e / 4][e % 4]));
        if constexpr (decltype(masked)::value) {
          const int4 &four = token[e / 4];
          p = (e % 4 == 0 ? four.x : e % 4 == 1 ? four.y : e % 4 == 2 ? four.z : four.w) < first_seen ? 0.0f : p;
        }
        s[e] = p;
        dp[e] = p * (dp[e] - delta[e / 4][e % 4]);
        if constexpr (e % 2 == 1) {
          pw[e / 2] = E::pack(s[e - 1], s[e]);
          pds[e / 2] = E::pack(dp[e - 1], dp[e]);
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    static_for<PRODUCTS>([&](auto i) __attribute__((always_inline)) {
      constexpr int c = i / (D / 16), dt = i % (D / 16) / 2, at = (i + PRODUCTS) % AHEAD;
      const uint4 now = x[at];
      if constexpr (i + AHEAD < PRODUCTS) x[at] = by_columns(tile, b, std::integral_constant<int, i + AHEAD>());
      if constexpr (i % 2 == 0) dv[dt] = E::mfma(now, uint4{pw[4 * c], pw[4 * c + 1], pw[4 * c + 2], pw[4 * c + 3]}, dv[dt]);
      else dk[dt] = E::mfma(now, uint4{pds[4 * c], pds[4 * c + 1], pds[4 * c + 2], pds[4 * c + 3]}, dk[dt]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  // While a step is worked on, its successor's rows are in LDS from the middle of
  // the step on, and those of the two behind that on their way.
  StepAt now(steps, from), ahead = now;
  int stage = 0;  // of the step
  const auto stage_after = [&](int n) { return (stage + n) % L::COUNT; };
  if (from < to) {
    for (int i = 0; i < 3 && from + i < to; i++, ahead.advance(steps, q_len)) {
      fetch(ahead, i);
      if (i == 0) wait_loads();
    }
    block_barrier();
    f32x16 s0, dp0, s1, dp1;
    products(lds, 0, s0, dp0);
    const auto whole_step = [&](int64_t step, auto masked) __attribute__((always_inline)) {
      const unsigned char *tile = lds + stage * L::BYTES, *next = lds + stage_after(1) * L::BYTES;
      const int first_seen = key - behind - now.token;
      half_step(tile, 0, s0, dp0, tile, 32, s1, dp1, first_seen, masked);
      if (step + 2 < to) wait_for_older();
      else wait_loads();
      block_barrier();
      if (step + 3 < to) {
        fetch(ahead, stage_after(3));
        ahead.advance(steps, q_len);
      }
      // (after the last step these products are of what the stage holds, unused)
      half_step(tile, 32, s1, dp1, next, 0, s0, dp0, first_seen, masked);
      stage = stage_after(1);
      now.advance(steps, q_len);
    };
    // The first steps of a causal tile see only some of its keys.
    const int64_t border =
        !a.causal ? 0 : steps.chunks > 1 ? steps.count() : (key0 + AG_KEYS - 1 - behind - steps.first + steps.tokens - 1) / steps.tokens;
    int64_t step = from;
    for (; step < to && step < border; step++) whole_step(step, std::true_type());
    for (; step < to; step++) whole_step(step, std::false_type());
  }
  if (parts > 1) {
    f32x4 *dst = reinterpret_cast<f32x4 *>(part_sums<D>(a, blockIdx.x, part)) + threadIdx.x;
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        dst[(dt * 4 + i / 4) * AG_THREADS] = f32x4{dk[dt][i], dk[dt][i + 1], dk[dt][i + 2], dk[dt][i + 3]};
        dst[(D / 8 + dt * 4 + i / 4) * AG_THREADS] = f32x4{dv[dt][i], dv[dt][i + 1], dv[dt][i + 2], dv[dt][i + 3]};
      }
  } else {
    store_column<E, D>(dk, a.scale, a.dk.at(t.first + key, kv_head), a.dim, key < k_len);
    store_column<E, D>(dv, 1.0f, a.dv.at(t.first + key, kv_head), a.dim, key < k_len);
  }
}

// Adds the parts of the split key tiles, gridDim.y blocks a tile, laid out as the
// blocks that left them.  (The last block of a tile to finish could add them instead, but
// making its sums visible to the other XCDs costs more: 490 + 41 us became 735 us.)
template <class E, int D> __global__ __launch_bounds__(AG_THREADS) void attention_dkv_join_kernel(GradArgs a) {
  const int kv_head = blockIdx.x % a.kv_heads;
  SegTile t;
  if (!find_key_tile(a, t)) return;
  const int k_len = (int)t.len, q_len = (int)t.len2, key0 = (int)t.tile * AG_KEYS;
  const int parts = parts_of(RowSteps(a.group, q_len, first_token(a, key0, q_len, k_len)).count(), a.parts, a.part_steps);
  if (parts == 1) return;
  const int row = threadIdx.x / WAVE * 32 + (lane_id() & 31);
  const bool there = key0 + row < k_len;
  const int64_t at = t.first + key0 + (there ? row : 0);
  // 32 components of dk or of dv at a time, two parts at a time.
  for (int c = blockIdx.y; c < D / 16; c += gridDim.y) {
    const bool is_v = c >= D / 32;
    const int dt = c % (D / 32);
    const auto load = [&](int part, f32x4 (&x)[4]) __attribute__((always_inline)) {
      const f32x4 *src = reinterpret_cast<const f32x4 *>(part_sums<D>(a, blockIdx.x, part)) + 4 * c * AG_THREADS + threadIdx.x;
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = src[i * AG_THREADS];
    };
    f32x16 sum[1];
#pragma unroll
    for (int i = 0; i < 16; i++) sum[0][i] = 0.0f;
    for (int p = 0; p < parts; p += 2) {
      f32x4 x[4], y[4];
      load(p, x);
      load(p + 1 < parts ? p + 1 : p, y);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        sum[0][i] += x[i / 4][i % 4];
        if (p + 1 < parts) sum[0][i] += y[i / 4][i % 4];
      }
    }
    store_column<E, 32>(sum, is_v ? 1.0f : a.scale, (is_v ? a.dv : a.dk).at(at, kv_head) + dt * 32, a.dim - dt * 32, there);
  }
}

// Workspace: the shift and D of every row and head, then the parts.  Key tiles are
// split so that there are about three blocks for every place on the chip (one a
// CU, two for D = 64); lengths are not known here, and a sequence is expected to be
// at most eight times as long as the average (a longer one has fewer parts).  What
// that balances against is the parts' traffic and the second launch: five sequences
// of up to 4096 tokens, 32 + 8 heads of 128, all kernels 947 us with eight blocks a
// place and 16 steps a part, 895 with three and 32; thirty of up to 512, 16 heads of
// 64, 71 us with parts and 62 without.
struct GradPlan {
  int64_t tiles;
  int parts, part_steps;
  size_t row_bytes, part_bytes;
};
static GradPlan grad_plan(int64_t q_rows, int64_t k_rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t m) {
  GradPlan p;
  p.tiles = most_tiles(k_rows, m, AG_KEYS) * kv_heads;
  const int64_t places = NUM_CUS_HINT * (head_dim <= 64 ? 2 : 1);
  const int64_t wanted = p.tiles > 0 ? ceil_div(3 * places, p.tiles) : 1;
  p.parts = (int)(wanted < AG_MOST_PARTS ? wanted : AG_MOST_PARTS);
  p.part_steps = part_steps_for(ceil_div(p.tiles * AG_MOST_PARTS, places));
  // no tile has more steps than the rows of one head group make
  const int64_t group = heads / kv_heads, lanes = group < AG_STEP ? group : AG_STEP;
  const int64_t longest = m > 0 && q_rows / m < q_rows / 8 ? 8 * (q_rows / m + 1) : q_rows;
  const int64_t steps = ceil_div(group, lanes) * ceil_div(longest, AG_STEP / lanes);
  if (p.parts > ceil_div(steps, p.part_steps)) p.parts = (int)ceil_div(steps, p.part_steps);
  if (p.parts < 1) p.parts = 1;
  p.row_bytes = (size_t)ceil_div(q_rows * heads, 4) * 16;
  p.part_bytes = p.parts > 1 ? (size_t)p.tiles * p.parts * 2 * AG_KEYS * (head_dim <= 64 ? 64 : 128) * sizeof(float) : 0;
  return p;
}

template <class E, int D> static int launch_grad(hipStream_t stream, GradArgs a, const GradPlan &p) {
  const int64_t units = most_tiles(a.q_rows, a.m, AG_ROWS / a.group) * a.kv_heads;
  if (units > AT_MOST_BLOCKS || p.tiles > AT_MOST_BLOCKS) return FA_ENOTSUP;
  constexpr int TILE = TileLoads<D, AG_THREADS>::BYTES, LDS = GradStage<D>::LDS;
  const auto dkv = attention_dkv_kernel<E, D>;
  static const hipError_t raised =
      hipFuncSetAttribute((const void *)dkv, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (raised != hipSuccess) return (int)raised;
  a.by_keys = takes_by_keys(units, a.m, a.dim);
  a.by_rows = a.m <= WAVE && p.tiles <= 2 * NUM_CUS_HINT * (a.dim <= 64 ? 2 : 1);
  if (units > 0) {
    attention_dq_kernel<E, D><<<dim3((unsigned)units), AG_THREADS, 4 * TILE, stream>>>(a);
    const int rc = launch_status();
    if (rc != 0) return rc;
  }
  if (p.tiles == 0) return 0;
  dkv<<<dim3((unsigned)p.tiles, (unsigned)p.parts), AG_THREADS, LDS, stream>>>(a);
  const int rc = launch_status();
  if (rc != 0 || p.parts == 1) return rc;
  // About as many blocks as run at a time: tiles that were not split end at once.
  int64_t blocks = 16 * NUM_CUS_HINT / p.tiles;
  blocks = blocks < 1 ? 1 : blocks > 8 ? 8 : blocks;
  attention_dkv_join_kernel<E, D><<<dim3((unsigned)p.tiles, (unsigned)blocks), AG_THREADS, 0, stream>>>(a);
  return launch_status();
}

}  // namespace fa

extern "C" size_t fa_attention_grad_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t heads,
                                                    int64_t kv_heads, int64_t head_dim, int64_t m) {
  if (q_rows < 0 || k_rows < 0 || m <= 0 || q_rows > AT_MOST_ROWS || k_rows > AT_MOST_ROWS || m > AT_MOST_ROWS ||
      check_shape(FA_F16, heads, kv_heads, head_dim) != 0)
    return 0;
  const GradPlan p = grad_plan(q_rows, k_rows, heads, kv_heads, head_dim, m);
  return 2 * p.row_bytes + p.part_bytes;
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
  if ((rc = check_scale(scale)) != 0) return rc;
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
  const GradPlan p = grad_plan(q_rows, k_rows, heads, kv_heads, head_dim, m);
  const GradArgs a = {to_heads(q), to_heads(k), to_heads(v), to_heads(out), to_heads(dout), to_heads(dq),
                      to_heads(dk), to_heads(dv), lse, (float *)workspace, (float *)((char *)workspace + p.row_bytes),
                      (float *)((char *)workspace + 2 * p.row_bytes), q_rows, k_rows, (int)heads, (int)kv_heads,
                      (int)(heads / kv_heads), (int)head_dim, q_offsets, q_lens, k_offsets, k_lens, m, scale,
                      causal != 0, p.parts, p.part_steps, false, false, failure, code};
  const hipStream_t s = (hipStream_t)stream;
  if (t == FA_F16) return head_dim <= 64 ? launch_grad<ElemF16, 64>(s, a, p) : launch_grad<ElemF16, 128>(s, a, p);
  return head_dim <= 64 ? launch_grad<ElemBF16, 64>(s, a, p) : launch_grad<ElemBF16, 128>(s, a, p);
}
