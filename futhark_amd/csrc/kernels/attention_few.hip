// Attention over a paged cache for few query rows a sequence (one new token, or
// a handful): bound by reading the cache once.
//
// A unit of work is a key head of a sequence with up to ROWS query rows (the
// query heads of the group for ROWS / group tokens), and its keys in tiles of
// 32.  All tiles of all units form one line that is cut into equal pieces, one
// for each wave the chip runs: how long the sequences are is read on the device,
// so that ragged lengths, and lengths that change between replays of a captured
// launch, always spread evenly, and the workspace does not grow with the cache.
// A wave works alone (no barriers): it streams its tiles through two stages of
// its own LDS, the loads of the next tile in flight while one is multiplied.
// Where a piece begins or ends inside a unit the wave leaves its part (output
// so far, maximum, sum) in the workspace, and a second kernel joins the parts.
//
// The products are 16 x 16 x 32: S^T = K Q^T with 16 query rows as columns, and
// O^T += V^T P^T with the weights as right operand in the registers they are
// computed in.  They are rounded to the element type once, for that product, which
// takes nothing wider; sums and statistics are f32.
//
// 64 sequences of up to 8192 keys, 8 key heads of 128: 518 MB in 88 us, 5.9 TB/s
// (reading alone reaches 6.1 to 6.9), and 5 us for the second kernel; one of 131072:
// 89 + 9 us.  Tens of microseconds and less are the chain lengths, page numbers,
// keys, weights: four of up to 500 keys 7.8 us.
#include "attention.hip.h"

namespace fa {

constexpr int FEW_KEYS = 32;        // keys of a tile
// What beginning a unit costs a wave, in tiles: on a long line every unit is that
// much longer, or waves that meet many short sequences end last (64 ragged
// sequences: the last wave at 121 us with the mean at 86 us).
constexpr int FEW_START = 2;
// On a short line, where a wave need not begin more than one unit, pieces end with
// their units and have at least few_least() tiles (32 KiB of keys and values: fewer
// leave more parts to join, 17 sequences of up to nine tokens, heads of 64, with two
// tiles 18.6 us and with four 15.7).  Short: up to FEW_SHORT of them; with more,
// waves that end with a unit lose more than beginning another costs (64 sequences of
// up to 2048 keys, heads of 128: up to 16 of them 41.5 us, four 31.9).
constexpr int FEW_SHORT = 4;
template <int D> constexpr int few_least() { return D == 128 ? 2 : 4; }
constexpr int FEW_THREADS = 256, FEW_WAVES = FEW_THREADS / WAVE;

// Waves a launch has: what fits the LDS of the chip (four waves of 33 KiB a CU,
// twice as many for D = 64).
template <int D> constexpr int few_waves() { return NUM_CUS_HINT * FEW_WAVES * (D == 128 ? 1 : 2); }
static_assert((NUM_CUS_HINT & (NUM_CUS_HINT - 1)) == 0, "a power of two");

// LDS of a wave: two stages of K and V, four slots of page numbers.
template <int D> struct FewLds {
  static constexpr int HALF = FEW_KEYS * D * 2, STAGE = 2 * HALF, IDS = 2 * STAGE, BYTES = IDS + 4 * WAVE * 4;
};

// A sequence: each of its row tiles and key heads is a unit of key_tiles() tiles.
struct FewSeq {
  int first, past, len, row_tiles;
  __device__ __forceinline__ int key_tiles() const { return (int)(((int64_t)past + len + FEW_KEYS - 1) / FEW_KEYS); }
  __device__ __forceinline__ int64_t units(int kv_heads) const { return (int64_t)row_tiles * kv_heads; }
};
// Segment i as the arrays have it.
struct FewSegment {
  int64_t first, len, past;
  bool ok;  // by segment_ok
  __device__ __forceinline__ FewSegment(const AttentionArgs &a, int64_t i) {
    past = a.pages.past_lens[i];
    ok = segment_ok(a.q_offsets, a.q_lens, i, a.q_rows, first, len);
  }
  __device__ __forceinline__ int end(const AttentionArgs &a) const { return segment_end(first, len, a.q_rows); }
  // The sequence, of no tokens unless `kept` and its cached ones fit the table.
  __device__ __forceinline__ FewSeq seq(const AttentionArgs &a, int per_tile, bool kept, bool report) const {
    FewSeq s = {0, 0, 0, 0};
    const int64_t room = a.pages.capacity();
    if (kept && (len == 0 || (past >= 0 && past <= room && len <= room - past))) {
      s.first = (int)first;
      s.past = len > 0 ? (int)past : 0;
      s.len = (int)len;
      s.row_tiles = (int)(((uint32_t)len + (uint32_t)per_tile - 1) / (uint32_t)per_tile);
    } else if (report && a.failure != nullptr) {
      *a.failure = a.code;
    }
    return s;
  }
};

// What a block knows of the line.  Thread t counts the sequences t * each ..
// (t + 1) * each - 1.  Up to FEW_THREADS sequences are kept.
struct FewTable {
  int64_t tiles[FEW_WAVES], units[FEW_WAVES], places[FEW_WAVES];  // a wave's threads count
  int ends[FEW_WAVES];  // the largest end of their segments
  // Where the pieces of the block's waves begin: the thread that counts the
  // place, the places and units before those it counts, and, if any segment is
  // broken, the largest end of the segments before them (else -1).
  int thread[FEW_WAVES], reach[FEW_WAVES];
  int64_t before[FEW_WAVES], units_before[FEW_WAVES];
  FewSeq seq[FEW_THREADS];
};
struct FewLine {
  int64_t each;
  int64_t total, piece;  // places in all and of a wave
  int64_t units;         // units in all
  int start;             // places of a unit before its tiles
  bool is_short;
  const FewTable *table;
  // A sequence, `reach` being that of the segments before it.
  __device__ __forceinline__ FewSeq seq(const AttentionArgs &a, int per_tile, int64_t i, const int &reach) const {
    if (each == 1) return table->seq[i];
    const FewSegment g(a, i);
    return g.seq(a, per_tile, g.ok && g.first >= reach, false);
  }
  // Takes `reach` behind sequence i.
  __device__ __forceinline__ void pass(const AttentionArgs &a, int64_t i, int &reach) const {
    if (each > 1 && reach >= 0) reach = OpMax<int>::apply(reach, FewSegment(a, i).end(a));
  }
  // Places of a unit; a short line pads it to whole pieces.
  __device__ __forceinline__ int unit(const FewSeq &s) const {
    const int tiles = s.key_tiles();
    return is_short ? (int)(((uint32_t)tiles + (uint32_t)piece - 1) / (uint32_t)piece * (uint32_t)piece) : tiles + start;
  }
};
__device__ __forceinline__ int64_t few_sum(const int64_t (&x)[FEW_WAVES], int to) {
  int64_t sum = 0;
#pragma unroll
  for (int w = 0; w < FEW_WAVES; w++) sum += w < to ? x[w] : 0;
  return sum;
}
// Lays out the line, and finds for each wave of the block the thread that counts
// the place where the wave's piece begins, with the places and units before that.
template <int D> __device__ __forceinline__ FewLine few_line(const AttentionArgs &a, int per_tile, FewTable &table) {
  const int waves = gridDim.x * FEW_WAVES;
  FewLine line;
  line.each = (a.m + FEW_THREADS - 1) / FEW_THREADS;
  line.table = &table;
  const int64_t i0 = threadIdx.x * line.each, i1 = i0 + line.each < a.m ? i0 + line.each : a.m;
  const int wave = threadIdx.x / WAVE;
  FewSeq s = {0, 0, 0, 0};
  int64_t tiles, units, units_upto, tiles_upto;
  int reach = -1;
  for (;;) {
    bool whole = true;
    int end = reach;
    tiles = units = 0;
    for (int64_t i = i0; i < i1; i++) {
      const FewSegment g(a, i);
      s = g.seq(a, per_tile, g.ok && (reach < 0 || g.first >= end), blockIdx.x == 0);
      units += s.units(a.kv_heads);
      tiles += s.units(a.kv_heads) * s.key_tiles();
      whole = whole && g.ok;
      end = OpMax<int>::apply(end, g.end(a));
    }
    table.seq[threadIdx.x] = s;
    units_upto = wave_incl_scan<int64_t, OpAdd<int64_t>>(units);
    tiles_upto = wave_incl_scan<int64_t, OpAdd<int64_t>>(tiles);
    if (reach < 0 && !__all(whole)) tiles_upto = -1;  // (of segments that do not count)
    if (lane_id() == WAVE - 1) table.tiles[wave] = tiles_upto, table.units[wave] = units_upto;
    __syncthreads();
    int64_t least = 0;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; w++) least = OpMin<int64_t>::apply(least, table.tiles[w]);
    if (least == 0) break;  // (the same for the whole block)
    // Once more, with where the segments before end.
    const int ends = wave_incl_scan<int, OpMax<int>>(end);
    if (lane_id() == WAVE - 1) table.ends[wave] = ends;
    __syncthreads();
    reach = OpMax<int>::apply(0, wave_shift_up1<int, OpMax<int>>(ends));
#pragma unroll
    for (int w = 0; w < FEW_WAVES; w++) reach = w < wave ? OpMax<int>::apply(reach, table.ends[w]) : reach;
  }
  const int64_t all_units = few_sum(table.units, FEW_WAVES), all_tiles = few_sum(table.tiles, FEW_WAVES);
  // Pieces of this many tiles are at most as many as there are waves: every unit
  // has at most one that is not full.
  line.units = all_units;
  const int64_t spare = waves - all_units;
  line.is_short = spare > 0 && all_tiles <= spare * FEW_SHORT;
  int64_t places = tiles + units * FEW_START;
  line.start = FEW_START;
  if (line.is_short) {
    const uint32_t even = ((uint32_t)all_tiles + (uint32_t)spare - 1) / (uint32_t)spare;
    line.piece = even < few_least<D>() ? few_least<D>() : even;
    line.start = 0;
    places = 0;
    int before = reach;
    for (int64_t i = i0; i < i1; i++) {
      if (line.each > 1) s = line.seq(a, per_tile, i, before);
      line.pass(a, i, before);
      places += s.units(a.kv_heads) * line.unit(s);
    }
  }
  const int64_t places_upto = wave_incl_scan<int64_t, OpAdd<int64_t>>(places);
  if (lane_id() == WAVE - 1) table.places[wave] = places_upto;
  __syncthreads();
  line.total = few_sum(table.places, FEW_WAVES);
  if (!line.is_short) line.piece = (line.total + waves - 1) >> __builtin_ctz(waves);  // a power of two
  const int64_t before = few_sum(table.places, wave) + places_upto - places;
  const int64_t units_here = few_sum(table.units, wave) + units_upto - units;
#pragma unroll
  for (int w = 0; w < FEW_WAVES; w++) {
    const int64_t at = ((int64_t)blockIdx.x * FEW_WAVES + w) * line.piece;
    if (at >= before && at < before + places) {
      table.thread[w] = threadIdx.x;
      table.reach[w] = reach;
      table.before[w] = before;
      table.units_before[w] = units_here;
    }
  }
  __syncthreads();
  return line;
}

// x / y where the quotient fits 32 bits; mostly both do.
__device__ __forceinline__ uint32_t few_divide(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? (uint32_t)x / (uint32_t)y : (uint32_t)(x / y);
}
// The workspace: where a wave leaves the part of the unit its piece begins in
// (slot 0) or ends in (slot 1), [rows][D] sums and [rows][2] maximum and sum; then
// the number of units, and of each what the second kernel needs to join it.
struct FewUnit {
  int64_t row;  // of its first token
  int w0, w1;   // the first and last wave that had a part (w0 == w1: nothing to join)
  int rows, head, unused[2];
};
__host__ __device__ constexpr int64_t few_part_floats(int waves, int rows, int d) {
  return (int64_t)2 * waves * rows * (d + 2);
}
__device__ __forceinline__ int64_t few_slot(int64_t wave, int slot, int rows) { return (2 * wave + slot) * rows; }
__device__ __forceinline__ int64_t *few_units(const AttentionArgs &a, int rows, int d) {
  return (int64_t *)(a.part_o + few_part_floats(d == 128 ? few_waves<128>() : few_waves<64>(), rows, d));
}
__device__ __forceinline__ FewUnit *few_unit(const AttentionArgs &a, int rows, int d) {
  return (FewUnit *)(few_units(a, rows, d) + 2);
}

// A wave's work on a unit: tiles from .. to - 1 of a sequence's keys for some of
// its tokens and one key head.
struct FewRun {
  int64_t seq, row;  // the row of the first token
  int head, tokens, rows;
  int first_limit, keys;  // last key the first token sees, keys the last one sees
  int from, to;
  __device__ __forceinline__ FewRun(const AttentionArgs &a, int per_tile, const FewSeq &s, int64_t seq, uint32_t unit,
                                    int from, int to)
      : seq(seq), from(from), to(to) {
    head = (int)(unit % (uint32_t)a.kv_heads);
    const int t0 = (int)(unit / (uint32_t)a.kv_heads) * per_tile;
    row = (int64_t)s.first + t0;
    tokens = s.len - t0 < per_tile ? s.len - t0 : per_tile;
    rows = tokens * a.group;
    first_limit = s.past + t0;
    keys = first_limit + tokens;
  }
};
// What comes of it, by query rows (columns) ct * 16 + lane % 16: components
// dt * 16 + 4 (lane / 16) + i of the sums, maxima of scores times log2(e), and
// this lane's share of the sum of weights.
template <int D, int ROWS> struct FewResult {
  f32x4 o[ROWS / 16][D / 16];
  float top[ROWS / 16], sum[ROWS / 16];
};

// Clears a wave's tiles where units past dim stay as they are.
template <int D> __device__ __forceinline__ void few_clear(unsigned char *mine, int dim) {
  if (dim == D) return;
  for (int i = lane_id() * 16; i < 2 * FewLds<D>::STAGE; i += WAVE * 16) *reinterpret_cast<uint4 *>(mine + i) = uint4{0, 0, 0, 0};
  wait_loads();
}

template <class E, int D, int ROWS>
__device__ __forceinline__ void few_attend(const AttentionArgs &a, unsigned char *mine, const FewRun &u,
                                           FewResult<D, ROWS> &r) {
  using L = FewLds<D>;
  constexpr int CT = ROWS / 16;                 // column tiles of 16 query rows
  constexpr int LOADS = L::HALF / (WAVE * 16);  // loads a lane and operand
  constexpr int LOAD_ROWS = FEW_KEYS / LOADS;
  const int lane = lane_id(), quarter = lane >> 4, col = lane & 15;
  const int32_t *table = a.pages.table + u.seq * a.pages.cols;
  const uint32_t lds_base = lds_address(mine);
  int *ids = reinterpret_cast<int *>(mine + L::IDS);
  const int load_row = lane / (D / 8), load_slot = lane % (D / 8);
  const int64_t row_bytes = a.dim * 2, head_bytes = row_bytes << a.pages.page_shift;
  const int slot_mask = (1 << a.pages.page_shift) - 1;
  // The usual case: pages of at least the rows a load covers.  lane_at: this lane's
  // place among them (the swizzle repeats every 16 rows), and whether its unit lies
  // below dim; those that do not were cleared beforehand.
  const bool plain = ((LOAD_ROWS - 1) & ~slot_mask) == 0;
  uint32_t lane_at[4];
  bool lane_live[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int unit = load_slot ^ tile_swizzle<D>(load_row + i * LOAD_ROWS);
    lane_at[i] = load_row * (uint32_t)row_bytes + unit * 16;
    lane_live[i] = unit * 8 < a.dim;
  }

  // Operand places inside a tile.  Row m of a product's 16 keys is key
  // 4 s(m / 4) + m % 4 of them, s = 0 2 1 3: with that order the rows that two
  // neighbouring quarters of a wave read of V together fall into different banks.
  const int sigma = (quarter >> 1) | ((quarter & 1) << 1);
  const int k_row = 4 * (((col >> 2) >> 1) | (((col >> 2) & 1) << 1)) + (col & 3);
  int k_at[D / 32], v_at[D / 16][2];
#pragma unroll
  for (int s = 0; s < D / 32; s++) k_at[s] = tile_offset<D>(k_row, 4 * s + quarter);
#pragma unroll
  for (int dt = 0; dt < D / 16; dt++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int c = dt * 16 + 4 * (col & 3);
      v_at[dt][h] = L::HALF + tile_offset<D>(16 * h + 4 * sigma + (col >> 2), c >> 3) + (c & 7) * 2;
    }

  // Page numbers of the keys of tile t (and of the next 32, not used).
  const auto fetch_ids = [&](int t) __attribute__((always_inline)) {
    const int key = t * FEW_KEYS + lane < u.keys ? t * FEW_KEYS + lane : u.keys - 1;
    const int32_t *src = table + (key >> a.pages.page_shift);
    load_word_to_lds(src, lds_base + L::IDS + (t & 3) * (WAVE * 4));
  };
  fetch_ids(u.from);
  fetch_ids(u.from + 1);
  uint4 q[CT][D / 32];
  int limit[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ct++) {
    const int row = ct * 16 + col < u.rows ? ct * 16 + col : u.rows - 1;
    limit[ct] = u.first_limit + row / a.group;
    const uint16_t *src = a.q.at(u.row + row / a.group, u.head * a.group + row % a.group);
#pragma unroll
    for (int k = 0; k < D / 32; k++) q[ct][k] = load_unit(src, 32 * k + 8 * quarter, a.dim);
  }
#pragma unroll
  for (int ct = 0; ct < CT; ct++) {
    r.top[ct] = -INFINITY;
    r.sum[ct] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) r.o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const auto fetch = [&](int t) __attribute__((always_inline)) {
    const uint32_t dst = lds_base + (t & 1) * L::STAGE;
    const int key0 = t * FEW_KEYS, id = ids[(t & 3) * WAVE + (lane & (FEW_KEYS - 1))];
    const bool there = key0 + (lane & (FEW_KEYS - 1)) < u.keys;
    const bool named = id >= 0 && id < a.pages.n_pages;
    if (plain && __all(there && named)) {
      // A load's rows lie in one page: its base is the same for all lanes.
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const int64_t off = ((int64_t)__builtin_amdgcn_readlane(id, i * LOAD_ROWS) * a.kv_heads + u.head) * head_bytes +
                            ((key0 + i * LOAD_ROWS) & slot_mask) * row_bytes;
        if (lane_live[i % 4]) {
          stream_to_lds((const char *)a.pages.k + off, lane_at[i % 4], dst + i * (WAVE * 16));
          stream_to_lds((const char *)a.pages.v + off, lane_at[i % 4], dst + L::HALF + i * (WAVE * 16));
        }
      }
      return;
    }
    if (there && !named && a.failure != nullptr) *a.failure = a.code;
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int r = load_row + i * LOAD_ROWS, unit8 = load_slot ^ tile_swizzle<D>(r);
      const int page = __shfl(id, r);
      const int64_t off = ((int64_t)page * a.kv_heads + u.head) * head_bytes + ((key0 + r) & slot_mask) * row_bytes + unit8 * 16;
      const bool live = key0 + r < u.keys && page >= 0 && page < a.pages.n_pages && unit8 * 8 < a.dim;
      load_to_lds(live ? (const void *)((const char *)a.pages.k + off) : (const void *)&g_zeros, dst + i * (WAVE * 16));
      load_to_lds(live ? (const void *)((const char *)a.pages.v + off) : (const void *)&g_zeros,
                  dst + L::HALF + i * (WAVE * 16));
    }
  };

  // In flight while tile t is multiplied: the page numbers of t + 2 (older),
  // then the 2 LOADS loads of tile t + 1.
#pragma unroll
  for (int ct = 0; ct < CT; ct++) arrived(q[ct]);
  wait_loads();
  fetch(u.from);
  fetch_ids(u.from + 2);
  if (u.from + 1 < u.to) fetch(u.from + 1);
  for (int t = u.from; t < u.to; t++) {
    if (t + 1 < u.to) wait_but<2 * LOADS>();
    else wait_loads();
    unsigned char *kt = mine + (t & 1) * L::STAGE;
    const int key0 = t * FEW_KEYS;
    f32x4 w[CT][2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
      for (int ct = 0; ct < CT; ct++) w[ct][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < D / 32; k++) {
        const uint4 x = *reinterpret_cast<const uint4 *>(kt + k_at[k] + b * (16 * D * 2));
#pragma unroll
        for (int ct = 0; ct < CT; ct++) w[ct][b] = E::mfma16(x, q[ct][k], w[ct][b]);
      }
    }
    const bool masked = key0 + FEW_KEYS - 1 > u.first_limit;
    if (masked) {
#pragma unroll
      for (int ct = 0; ct < CT; ct++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (key0 + 16 * b + 4 * sigma + i > limit[ct]) w[ct][b][i] = -INFINITY;
    }
    uint4 p[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      float high = w[ct][0][0];
#pragma unroll
      for (int i = 1; i < 8; i++) high = fmaxf(high, w[ct][i >> 2][i & 3]);
      high = fold_quarters(high, FMax()) * a.scale_log2;
      if (__any(high > r.top[ct] + AT_RESCALE)) {
        // (each row by its own scores alone: what other rows see changes no bit of it)
        const float now = high > r.top[ct] + AT_RESCALE ? high : r.top[ct];
        const float factor = now == r.top[ct] ? 1.0f : exp2f(r.top[ct] - now);
        r.top[ct] = now;
        r.sum[ct] *= factor;
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) r.o[ct][dt] *= factor;
      }
      const float shift = r.top[ct] == -INFINITY ? 0.0f : r.top[ct];
      f32x8 x;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = __builtin_amdgcn_exp2f(fmaf(w[ct][i >> 2][i & 3], a.scale_log2, -shift));
        r.sum[ct] += x[i];
      }
      p[ct] = E::pack(x);
    }
    // Tokens of the unit see different keys of this tile: a value that a row
    // does not see must not reach it, and 0 * NaN would.  Values that are not
    // finite are added one by one and taken out of the tile.
    if (masked && u.tokens > 1) {
      bool found = false;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const uint4 x = *reinterpret_cast<const uint4 *>(kt + L::HALF + (i * WAVE + lane) * 16);
        for (uint32_t y : {x.x, x.y, x.z, x.w})
          found = found || (y & E::exponent) == E::exponent || (y >> 16 & E::exponent) == E::exponent;
      }
      if (__any(found)) {
        for (int j = 0; j < FEW_KEYS; j++)
#pragma unroll
          for (int dt = 0; dt < D / 16; dt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int d = dt * 16 + 4 * quarter + i;
              const uint16_t bits =
                  *reinterpret_cast<const uint16_t *>(kt + L::HALF + tile_offset<D>(j, d >> 3) + (d & 7) * 2);
#pragma unroll
              for (int ct = 0; ct < CT; ct++)
                if ((bits & E::exponent) == E::exponent && key0 + j <= limit[ct]) r.o[ct][dt][i] += E::load(bits);
            }
#pragma unroll
        for (int i = 0; i < LOADS * 8; i++) {
          uint16_t *x = reinterpret_cast<uint16_t *>(kt + L::HALF) + (i / 8 * WAVE + lane) * 8 + i % 8;
          if ((*x & E::exponent) == E::exponent) *x = 0;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) {
      const auto read = [&](int h) __attribute__((always_inline)) {
        return bit_cast<uint2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (i16x4 __attribute__((address_space(3))) *)(kt + v_at[dt][h])));
      };
      const uint2 lo = read(0), hi = read(1);
#pragma unroll
      for (int ct = 0; ct < CT; ct++) r.o[ct][dt] = E::mfma16(uint4{lo.x, lo.y, hi.x, hi.y}, p[ct], r.o[ct][dt]);
    }
    // The tile has been read (its reads have returned before its products); the
    // stage takes the next but one.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + 2 < u.to) {
      fetch_ids(t + 3);
      fetch(t + 2);
    }
  }
  wait_loads();
}

// Rows of a result, straight to the output.
template <class E, int D, int ROWS>
__device__ __forceinline__ void few_store(const AttentionArgs &a, const FewRun &u, const FewResult<D, ROWS> &r) {
  const int quarter = lane_id() >> 4;
#pragma unroll
  for (int ct = 0; ct < ROWS / 16; ct++) {
    const int row = ct * 16 + (lane_id() & 15);
    const float all = fold_quarters(r.sum[ct], FAdd());
    if (row >= u.rows) continue;
    const int64_t out_row = u.row + row / a.group;
    const int q_head = u.head * a.group + row % a.group;
    const bool empty = all == 0.0f;  // only scores of -inf (and no NaN)
    const float inverse = empty ? 0.0f : 1.0f / all;
    uint16_t *dst = a.out.at(out_row, q_head);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) {
      const int d = dt * 16 + 4 * quarter;
      uint32_t x[4];
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = E::store(empty ? 0.0f : r.o[ct][dt][i] * inverse);
      if (d < a.dim) *reinterpret_cast<uint2 *>(dst + d) = uint2{x[0] | x[1] << 16, x[2] | x[3] << 16};
    }
    if (a.lse != nullptr && quarter == 0)
      a.lse[out_row * a.heads + q_head] = empty ? -INFINITY : (r.top[ct] + log2f(all)) * LN2;
  }
}
// Rows of a result as a part: sums at o + row * D, maximum and sum at ml + 2 * row.
template <int D, int ROWS>
__device__ __forceinline__ void few_store_part(const FewRun &u, const FewResult<D, ROWS> &r, float *o, float *ml) {
  const int quarter = lane_id() >> 4;
#pragma unroll
  for (int ct = 0; ct < ROWS / 16; ct++) {
    const int row = ct * 16 + (lane_id() & 15);
    const float all = fold_quarters(r.sum[ct], FAdd());
    if (row >= u.rows) continue;
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) *reinterpret_cast<f32x4 *>(o + row * D + dt * 16 + 4 * quarter) = r.o[ct][dt];
    if (quarter == 0) {
      ml[2 * row] = r.top[ct];
      ml[2 * row + 1] = all;
    }
  }
}

template <class E, int D, int ROWS>
__global__ __launch_bounds__(FEW_THREADS, D == 128 ? 1 : 2) void attention_few_kernel(AttentionArgs a) {
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ FewTable seqs;
  const int per_tile = ROWS / a.group;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int64_t number = (int64_t)blockIdx.x * FEW_WAVES + wave;
  const FewLine line = few_line<D>(a, per_tile, seqs);
  if (blockIdx.x == 0 && threadIdx.x == 0) *few_units(a, ROWS, D) = line.units;
  int64_t at = number * line.piece;
  const int64_t end = at + line.piece < line.total ? at + line.piece : line.total;
  if (at >= end) return;
  few_clear<D>(lds + wave * FewLds<D>::BYTES, a.dim);
  // The first of the sequences among which the piece begins (the loop below walks
  // on to the one), and the places and units before it.
  int64_t seq = __builtin_amdgcn_readfirstlane(seqs.thread[wave]) * line.each;
  int64_t precede = seqs.before[wave], units_before = seqs.units_before[wave];
  while (at < end) {
    const FewSeq s = line.seq(a, per_tile, seq, seqs.reach[wave]);
    const int length = line.unit(s);
    const int64_t places = s.units(a.kv_heads) * length;
    if (at >= precede + places) {
      precede += places;
      units_before += s.units(a.kv_heads);
      line.pass(a, seq, seqs.reach[wave]);
      seq++;
      continue;
    }
    // Place in the sequence: unit and tile.
    const int64_t inside = at - precede;
    const uint32_t unit = few_divide(inside, length);
    const int place = (int)(inside - (int64_t)unit * length);
    const int next = end - at < length - place ? (int)(place + (end - at)) : length;
    at += next - place;
    const int key_tiles = s.key_tiles();
    const int from = place > line.start ? place - line.start : 0;
    const int to = next - line.start < key_tiles ? next - line.start : key_tiles;
    if (from >= to) continue;
    const FewRun u(a, per_tile, s, seq, unit, from, to);
    if (from == 0 && lane_id() == 0 && units_before + unit < a.most_units) {
      const int64_t begin = at - (next - line.start);  // the place of the unit's first tile
      few_unit(a, ROWS, D)[units_before + unit] = FewUnit{
          u.row, (int)number, (int)few_divide(begin + key_tiles - 1, line.piece), u.rows, u.head, {}};
    }
    FewResult<D, ROWS> r;
    few_attend<E, D, ROWS>(a, lds + wave * FewLds<D>::BYTES, u, r);
    if (from == 0 && to == key_tiles) {
      few_store<E, D, ROWS>(a, u, r);
    } else {
      const int64_t part = few_slot(number, from == 0 ? 1 : 0, ROWS);
      few_store_part<D, ROWS>(u, r, a.part_o + part * D, a.part_ml + 2 * part);
    }
  }
}

// A block a unit, its waves a quarter of the keys each, joined in LDS: one launch
// where contexts are short and the units fit the chip at once.
template <class E, int D, int ROWS>
__global__ __launch_bounds__(FEW_THREADS, D == 128 ? 1 : 2) void attention_few_short_kernel(AttentionArgs a) {
  extern __shared__ __align__(16) unsigned char lds[];
  const int per_tile = ROWS / a.group, lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  if (blockIdx.x == 0)
    for (int64_t i = threadIdx.x; i < a.m; i += FEW_THREADS) {
      const FewSegment g(a, i);
      g.seq(a, per_tile, g.ok, true);
    }
  // The sequence of this unit; every wave looks.
  FewSeq s;
  int64_t seq = -1, before = 0;
  SegChain chain;
  for (int64_t base = 0; base < a.m && seq < 0; base += WAVE) {
    const FewSegment g(a, base + lane < a.m ? base + lane : a.m - 1);
    const bool kept = chain.keep(g.ok & (base + lane < a.m), g.first, g.len, a.q_offsets, a.q_lens, a.m, a.q_rows, base);
    const FewSeq mine = g.seq(a, per_tile, kept, false);
    const int64_t units = mine.units(a.kv_heads);
    const int64_t upto = before + wave_incl_scan<int64_t, OpAdd<int64_t>>(units);
    const uint64_t past = __ballot(upto > (int64_t)blockIdx.x);
    if (past == 0) {
      before = read_lane(upto, WAVE - 1);
      continue;
    }
    const int at = __builtin_ctzll(past);
    seq = base + at;
    before = read_lane(upto, at) - read_lane(units, at);
    s = FewSeq{read_lane(mine.first, at), read_lane(mine.past, at), read_lane(mine.len, at), read_lane(mine.row_tiles, at)};
  }
  if (seq < 0) return;
  few_clear<D>(lds + wave * FewLds<D>::BYTES, a.dim);
  const int64_t tiles = s.key_tiles();
  const FewRun u(a, per_tile, s, seq, (uint32_t)(blockIdx.x - before), (int)(tiles * wave / FEW_WAVES),
                 (int)(tiles * (wave + 1) / FEW_WAVES));
  FewResult<D, ROWS> r;
  few_attend<E, D, ROWS>(a, lds + wave * FewLds<D>::BYTES, u, r);
  __syncthreads();
  float *o = reinterpret_cast<float *>(lds), *ml = o + FEW_WAVES * ROWS * D;
  static_assert(FEW_WAVES * ROWS * (D + 2) * 4 <= FewLds<D>::BYTES * FEW_WAVES, "the parts fit where the tiles were");
  few_store_part<D, ROWS>(u, r, o + wave * ROWS * D, ml + 2 * wave * ROWS);
  __syncthreads();
  for (int i = threadIdx.x; i < u.rows * (D / 4); i += FEW_THREADS) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; w++) top = fmaxf(top, ml[2 * (w * ROWS + row)]);
    const float shift = top == -INFINITY ? 0.0f : top;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; w++) {
      const float f = exp2f(ml[2 * (w * ROWS + row)] - shift);
      sum += f * ml[2 * (w * ROWS + row) + 1];
      x += f * *reinterpret_cast<const f32x4 *>(o + (w * ROWS + row) * D + d);
    }
    const bool empty = sum == 0.0f;
    const float inverse = empty ? 0.0f : 1.0f / sum;
    const int64_t out_row = u.row + row / a.group;
    const int q_head = u.head * a.group + row % a.group;
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = E::store(empty ? 0.0f : x[j] * inverse);
    if (d < a.dim) *reinterpret_cast<uint2 *>(a.out.at(out_row, q_head) + d) = uint2{y[0] | y[1] << 16, y[2] | y[3] << 16};
    if (a.lse != nullptr && d == 0) a.lse[out_row * a.heads + q_head] = empty ? -INFINITY : (top + log2f(sum)) * LN2;
  }
}

// Joins the parts: a block a unit and join_rows of its rows.  A thread takes
// four components of a row; where there are fewer rows several threads share the
// parts of one.  Parts are taken in order, WAVE at a time, with the running
// maximum and sum.
template <class E, int D, int ROWS>
__global__ __launch_bounds__(FEW_THREADS) void attention_few_join_kernel(AttentionArgs a, int join_rows) {
  constexpr int FOURS = D / 4, JOIN_ROWS = FEW_THREADS / FOURS, BATCH = 8;
  __shared__ float tops[JOIN_ROWS], sums[JOIN_ROWS], factors[JOIN_ROWS], weights[JOIN_ROWS][WAVE];
  __shared__ f32x4 shared[FEW_THREADS];
  // (both loads at once: the array has a place for every block)
  const int64_t units = *few_units(a, ROWS, D);
  const FewUnit u = few_unit(a, ROWS, D)[blockIdx.x];
  if (blockIdx.x >= units || u.w0 == u.w1) return;
  const int64_t w0 = u.w0, w1 = u.w1;
  const int row0 = blockIdx.y * join_rows;
  int rows = u.rows - row0;
  if (rows <= 0) return;
  if (rows > join_rows) rows = join_rows;
  const auto part = [&](int64_t w) { return few_slot(w, w == w0 ? 1 : 0, ROWS) + row0; };
  if (threadIdx.x < JOIN_ROWS) tops[threadIdx.x] = -INFINITY, sums[threadIdx.x] = 0.0f;
  int share = 1;  // threads that share the parts of one place
  while (2 * share * rows * FOURS <= FEW_THREADS) share *= 2;
  const int row = threadIdx.x / share / FOURS, four = threadIdx.x % (share * FOURS) / share, turn = threadIdx.x % share;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t base = w0; base <= w1; base += WAVE) {
    const int count = w1 - base + 1 < WAVE ? (int)(w1 - base + 1) : WAVE;
    int group = 1;  // lanes for the parts of a row
    while (group < count) group *= 2;
    __syncthreads();
    for (int i = threadIdx.x; i < rows * group; i += FEW_THREADS) {
      const int r = i / group, j = i % group;
      const float *ml = a.part_ml + 2 * (part(base + (j < count ? j : 0)) + r);
      float top = j < count ? ml[0] : -INFINITY, sum = ml[1];
      float f = top;
      for (int step = 1; step < group; step *= 2) top = fmaxf(top, __shfl_xor(top, step));
      top = fmaxf(top, tops[r]);
      f = exp2f(f - (top == -INFINITY ? 0.0f : top));
      weights[r][j] = f;
      sum *= f;
      for (int step = 1; step < group; step *= 2) sum += __shfl_xor(sum, step);
      if (j == 0) {
        factors[r] = top == -INFINITY ? 1.0f : exp2f(tops[r] - top);
        sums[r] = sums[r] * factors[r] + sum;
        tops[r] = top;
      }
    }
    __syncthreads();
    if (row >= rows) continue;
    o *= factors[row];
    for (int j0 = turn; j0 < count; j0 += BATCH * share) {
      f32x4 x[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int j = j0 + i * share;
        x[i] = *reinterpret_cast<const f32x4 *>(a.part_o + (part(base + (j < count ? j : turn)) + row) * D + 4 * four);
      }
#pragma unroll
      for (int i = 0; i < BATCH; i++) {
        const int j = j0 + i * share;
        if (j < count) o += weights[row][j] * x[i];
      }
    }
  }
  for (int step = share / 2; step > 0; step /= 2) {
    __syncthreads();
    shared[threadIdx.x] = o;
    __syncthreads();
    if (turn < step) o += shared[threadIdx.x + step];
  }
  if (row >= rows || turn != 0) return;
  const bool empty = sums[row] == 0.0f;
  const float inverse = empty ? 0.0f : 1.0f / sums[row];
  const int64_t out_row = u.row + (row0 + row) / a.group;
  const int q_head = u.head * a.group + (row0 + row) % a.group;
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = E::store(empty ? 0.0f : o[i] * inverse);
  if (4 * four < a.dim)
    *reinterpret_cast<uint2 *>(a.out.at(out_row, q_head) + 4 * four) = uint2{x[0] | x[1] << 16, x[2] | x[3] << 16};
  if (a.lse != nullptr && four == 0)
    a.lse[out_row * a.heads + q_head] = empty ? -INFINITY : (tops[row] + log2f(sums[row])) * LN2;
}

int few_rows(int64_t n, int64_t heads, int64_t kv_heads, int64_t m) {
  const int64_t group = heads / kv_heads;
  for (int rows : {16, 32, 64})
    if (group <= rows && n * group <= rows * m) return rows;
  return 0;
}

static int64_t few_most_units(int rows, int64_t n, int64_t group, int64_t kv_heads, int64_t m) {
  return most_tiles(n, m, rows / group) * kv_heads;
}

// Whether a block a unit, in one launch, is the faster way: the units fit the chip
// at once, and a wave's quarter of the longest table takes no longer than its piece
// of the line and the second launch.  (Heads of 128, 4 to 32 sequences of up to 512
// keys 12.7 us against 16 to 19 on the line, of 1040 19 against 17, of 2048 31
// against 21; heads of 64, 500 keys 9.7 against 13.9, 1040 11.4 against 14.5, 2048
// 20 against 22 where units fill the chip, 4000 30 against 15.5.)  Only the table's
// width is known here: four sequences of up to 500 keys take 15 us behind a table of
// 16384 positions.
template <int D> static bool few_in_one_launch(int64_t units, int64_t keys) {
  return units * FEW_WAVES <= few_waves<D>() && keys <= (D == 128 ? 1024 : 1536);
}

size_t few_workspace(int rows, int64_t n, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t m, int64_t keys) {
  const int64_t units = few_most_units(rows, n, heads / kv_heads, kv_heads, m);
  if (head_dim <= 64 ? few_in_one_launch<64>(units, keys) : few_in_one_launch<128>(units, keys)) return 0;
  const int64_t floats = head_dim <= 64 ? few_part_floats(few_waves<64>(), rows, 64)
                                        : few_part_floats(few_waves<128>(), rows, 128);
  return (size_t)floats * sizeof(float) + 16 + (size_t)units * sizeof(FewUnit);
}

template <class E, int D, int ROWS>
static int launch_few_of(hipStream_t stream, AttentionArgs a, void *workspace) {
  const int64_t units = few_most_units(ROWS, a.q_rows, a.group, a.kv_heads, a.m);
  if (units > AT_MOST_BLOCKS) return FA_ENOTSUP;
  constexpr int LDS = FewLds<D>::BYTES * FEW_WAVES;
  const auto kernel = attention_few_kernel<E, D, ROWS>, short_kernel = attention_few_short_kernel<E, D, ROWS>;
  static const hipError_t raised =
      hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  static const hipError_t raised_short =
      hipFuncSetAttribute((const void *)short_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (raised != hipSuccess) return (int)raised;
  if (raised_short != hipSuccess) return (int)raised_short;
  if (few_in_one_launch<D>(units, a.pages.cols << a.pages.page_shift)) {
    short_kernel<<<dim3((unsigned)units), FEW_THREADS, LDS, stream>>>(a);
    return launch_status();
  }
  a.part_o = (float *)workspace;
  a.part_ml = a.part_o + (int64_t)2 * few_waves<D>() * ROWS * D;
  a.most_units = units;
  kernel<<<dim3(few_waves<D>() / FEW_WAVES), FEW_THREADS, LDS, stream>>>(a);
  const int rc = launch_status();
  if (rc != 0) return rc;
  // Rows a block of the second kernel joins: as many as its threads hold, fewer
  // while there are less than two blocks a CU (17 sequences with up to nine tokens
  // 20.0 -> 18.6 us, against one a CU; four a CU the same).
  const int64_t rows = ROWS / a.group * a.group;  // of a unit, at most
  int join_rows = FEW_THREADS / (D / 4);
  while (join_rows > 1 && units * ceil_div(rows, join_rows) < 2 * NUM_CUS_HINT) join_rows /= 2;
  const dim3 grid((unsigned)units, (unsigned)ceil_div(rows, join_rows));
  attention_few_join_kernel<E, D, ROWS><<<grid, FEW_THREADS, 0, stream>>>(a, join_rows);
  return launch_status();
}

template <class E> static int launch_few_type(hipStream_t stream, int rows, const AttentionArgs &a, void *workspace) {
  if (a.dim <= 64) {
    if (rows == 16) return launch_few_of<E, 64, 16>(stream, a, workspace);
    if (rows == 32) return launch_few_of<E, 64, 32>(stream, a, workspace);
    return launch_few_of<E, 64, 64>(stream, a, workspace);
  }
  if (rows == 16) return launch_few_of<E, 128, 16>(stream, a, workspace);
  if (rows == 32) return launch_few_of<E, 128, 32>(stream, a, workspace);
  return launch_few_of<E, 128, 64>(stream, a, workspace);
}

int launch_few(hipStream_t stream, fa_dtype t, int rows, const AttentionArgs &a, void *workspace) {
  return t == FA_F16 ? launch_few_type<ElemF16>(stream, rows, a, workspace)
                     : launch_few_type<ElemBF16>(stream, rows, a, workspace);
}

}  // namespace fa
