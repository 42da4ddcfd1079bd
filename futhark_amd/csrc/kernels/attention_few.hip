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
// computed in.
#include "attention.hip.h"

namespace fa {

constexpr int FEW_KEYS = 32;        // keys of a tile
// What beginning a unit costs a wave, in tiles: every unit is that much longer
// on the line, or waves that meet many short sequences end last (64 ragged
// sequences: the last wave at 121 us with the mean at 86 us).
constexpr int FEW_START = 2;
constexpr int FEW_LEAST = 4 + FEW_START;  // a piece is at least this long
constexpr int FEW_THREADS = 256, FEW_WAVES = FEW_THREADS / WAVE;

// Waves a launch has: what fits the LDS of the chip (four waves of 33 KiB a CU,
// twice as many for D = 64).
template <int D> constexpr int few_waves() { return NUM_CUS_HINT * FEW_WAVES * (D == 128 ? 1 : 2); }
static_assert((NUM_CUS_HINT & (NUM_CUS_HINT - 1)) == 0, "a power of two");

// LDS of a wave: two stages of K and V, four slots of page numbers.
template <int D> struct FewLds {
  static constexpr int HALF = FEW_KEYS * D * 2, STAGE = 2 * HALF, IDS = 2 * STAGE, BYTES = IDS + 4 * WAVE * 4;
};

// A sequence as the line sees it: each of its row tiles and key heads is a unit
// of FEW_START places and one for each of its key tiles.
struct FewSeq {
  int first, past, len, row_tiles;
  __device__ __forceinline__ int key_tiles() const { return (int)(((int64_t)past + len + FEW_KEYS - 1) / FEW_KEYS); }
  __device__ __forceinline__ int unit() const { return key_tiles() + FEW_START; }
  __device__ __forceinline__ int64_t units(int kv_heads) const { return (int64_t)row_tiles * kv_heads; }
  __device__ __forceinline__ int64_t places(int kv_heads) const { return units(kv_heads) * unit(); }
};
__device__ __forceinline__ FewSeq few_seq(const AttentionArgs &a, int per_tile, int64_t i, bool report) {
  FewSeq s = {0, 0, 0, 0};
  int64_t first, len;
  const int64_t past = a.pages.past_lens[i], room = a.pages.capacity();
  bool ok = segment_ok(a.q_offsets, a.q_lens, i, a.q_rows, first, len);
  ok = ok && (len == 0 || (past >= 0 && past <= room && len <= room - past));
  if (ok) {
    s.first = (int)first;
    s.past = len > 0 ? (int)past : 0;
    s.len = (int)len;
    s.row_tiles = (int)(((uint32_t)len + (uint32_t)per_tile - 1) / (uint32_t)per_tile);
  } else if (report && a.failure != nullptr) {
    *a.failure = a.code;
  }
  return s;
}

// What a block knows of the line.  Thread t counts the sequences t * each ..
// (t + 1) * each - 1: before[t] places precede them (units[t] units, which the
// second kernel asks for).  Up to FEW_THREADS sequences are kept.
struct FewTable {
  int64_t before[FEW_THREADS], wave_places[FEW_WAVES], wave_units[FEW_WAVES];
  FewSeq seq[FEW_THREADS];
};
struct FewLine {
  int64_t total, piece, each;  // places in all and of a piece
  const FewTable *table;
  __device__ __forceinline__ FewSeq seq(const AttentionArgs &a, int per_tile, int64_t i) const {
    return each == 1 ? table->seq[i] : few_seq(a, per_tile, i, false);
  }
};
__device__ __forceinline__ FewLine few_line(const AttentionArgs &a, int per_tile, int waves, FewTable &table,
                                            int64_t *units_before = nullptr) {
  FewLine line;
  line.each = (a.m + FEW_THREADS - 1) / FEW_THREADS;
  line.table = &table;
  int64_t places = 0, units = 0;
  for (int64_t i = threadIdx.x * line.each; i < (threadIdx.x + 1) * line.each && i < a.m; i++) {
    const FewSeq s = few_seq(a, per_tile, i, blockIdx.x == 0);
    places += s.places(a.kv_heads);
    units += s.units(a.kv_heads);
    table.seq[threadIdx.x] = s;
  }
  const int64_t places_upto = wave_incl_scan<int64_t, OpAdd<int64_t>>(places);
  const int64_t units_upto = units_before == nullptr ? 0 : wave_incl_scan<int64_t, OpAdd<int64_t>>(units);
  const int wave = threadIdx.x / WAVE;
  if (lane_id() == WAVE - 1) table.wave_places[wave] = places_upto, table.wave_units[wave] = units_upto;
  __syncthreads();
  int64_t places_base = 0, units_base = 0;
  line.total = 0;
  for (int w = 0; w < FEW_WAVES; w++) {
    if (w < wave) places_base += table.wave_places[w], units_base += table.wave_units[w];
    line.total += table.wave_places[w];
  }
  table.before[threadIdx.x] = places_base + places_upto - places;
  if (units_before != nullptr) units_before[threadIdx.x] = units_base + units_upto - units;
  __syncthreads();
  const int64_t even = (line.total + waves - 1) >> __builtin_ctz(waves);  // a power of two
  line.piece = even < FEW_LEAST ? FEW_LEAST : even;
  return line;
}
// x / y where the quotient fits 32 bits; mostly both do.
__device__ __forceinline__ uint32_t few_divide(int64_t x, int64_t y) {
  return ((x | y) >> 32) == 0 ? (uint32_t)x / (uint32_t)y : (uint32_t)(x / y);
}
// The thread that counted place `at` of the line; the same for the whole wave.
__device__ __forceinline__ int few_thread(const int64_t *starts, int64_t at) {
  int thread = -1;
  for (int b = 0; b < FEW_THREADS; b += WAVE) thread += __popcll(__ballot(starts[b + lane_id()] <= at));
  return thread;
}

// Where a wave leaves the part of the unit its piece begins in (slot 0) or ends
// in (slot 1): [rows][D] sums and [rows][2] maximum and sum.
__device__ __forceinline__ int64_t few_slot(int64_t wave, int slot, int rows) { return (2 * wave + slot) * rows; }

template <int N> __device__ __forceinline__ void wait_older_than() {
  // all but the N youngest loads have arrived
  if constexpr (N == 16) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  static_assert(N == 16 || N == 8, "loads of a tile");
}

template <class E, int D, int ROWS>
__global__ __launch_bounds__(FEW_THREADS, D == 128 ? 1 : 2) void attention_few_kernel(AttentionArgs a) {
  using L = FewLds<D>;
  constexpr int CT = ROWS / 16;                 // column tiles of 16 query rows
  constexpr int LOADS = L::HALF / (WAVE * 16);  // loads a lane and operand
  constexpr int LOAD_ROWS = FEW_KEYS / LOADS;
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ FewTable seqs;
  const int per_tile = ROWS / a.group;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int quarter = lane >> 4, col = lane & 15;
  const FewLine line = few_line(a, per_tile, gridDim.x * FEW_WAVES, seqs);
  const int64_t number = (int64_t)blockIdx.x * FEW_WAVES + wave;
  int64_t at = number * line.piece;
  const int64_t end = at + line.piece < line.total ? at + line.piece : line.total;
  if (at >= end) return;
  // The sequence the piece begins in (the loop below walks on to it) and the
  // tiles before that.
  int64_t seq = few_thread(seqs.before, at), precede = seqs.before[seq];
  seq *= line.each;

  unsigned char *mine = lds + wave * L::BYTES;
  const uint32_t lds_base = lds_address(mine);
  int *ids = reinterpret_cast<int *>(mine + L::IDS);
  const int load_row = lane / (D / 8), load_slot = lane % (D / 8);
  const int64_t row_bytes = a.dim * 2, head_bytes = row_bytes << a.pages.page_shift;
  const int slot_mask = (1 << a.pages.page_shift) - 1;
  // The usual case: whole rows, and pages of at least the rows a load covers.
  // lane_at: this lane's place among them (the swizzle repeats every 16 rows).
  const bool plain = a.dim == D && (LOAD_ROWS - 1 & ~slot_mask) == 0;
  uint32_t lane_at[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    lane_at[i] = load_row * (D * 2) + (load_slot ^ tile_swizzle<D>(load_row + i * LOAD_ROWS)) * 16;

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

  while (at < end) {
    const FewSeq s = line.seq(a, per_tile, seq);
    const int64_t places = s.places(a.kv_heads);
    if (at >= precede + places) {
      precede += places;
      seq++;
      continue;
    }
    // Place in the sequence: row tile, head, key tile.
    const int64_t inside = at - precede;
    const uint32_t unit = few_divide(inside, s.unit());
    const int place = (int)(inside - (int64_t)unit * s.unit());
    const int next = end - at < s.unit() - place ? (int)(place + (end - at)) : s.unit();
    at += next - place;
    const int key_tiles = s.key_tiles();
    const int from = place > FEW_START ? place - FEW_START : 0, to = next - FEW_START;
    if (from >= to) continue;
    const int head = (int)(unit % (uint32_t)a.kv_heads), t0 = (int)(unit / (uint32_t)a.kv_heads) * per_tile;
    const int tokens = s.len - t0 < per_tile ? s.len - t0 : per_tile, rows = tokens * a.group;
    const int first_limit = s.past + t0;              // last key the first token sees
    const int keys = first_limit + tokens;            // keys the last one sees
    const int64_t table = seq * a.pages.cols;

    // Page numbers of the keys of tile t (and of the next 32, not used).
    const auto fetch_ids = [&](int t) __attribute__((always_inline)) {
      const int key = t * FEW_KEYS + lane < keys ? t * FEW_KEYS + lane : keys - 1;
      const int32_t *src = a.pages.table + table + (key >> a.pages.page_shift);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(
                       __builtin_amdgcn_readfirstlane(lds_base + L::IDS + (t & 3) * (WAVE * 4))),
                   "v"(src)
                   : "memory", "m0");
    };
    fetch_ids(from);
    fetch_ids(from + 1);
    uint4 q[CT][D / 32];
    int limit[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      const int row = ct * 16 + col < rows ? ct * 16 + col : rows - 1;
      limit[ct] = first_limit + row / a.group;
      const uint16_t *src = a.q.at((int64_t)s.first + t0 + row / a.group, head * a.group + row % a.group);
#pragma unroll
      for (int k = 0; k < D / 32; k++) {
        const int c = 32 * k + 8 * quarter;
        q[ct][k] = c < a.dim ? *reinterpret_cast<const uint4 *>(src + c) : uint4{0, 0, 0, 0};
      }
    }
    f32x4 o[CT][D / 16];
    float top[CT], sum[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      top[ct] = -INFINITY;
      sum[ct] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const auto fetch = [&](int t) __attribute__((always_inline)) {
      const uint32_t dst = lds_base + (t & 1) * L::STAGE;
      const int key0 = t * FEW_KEYS, id = ids[(t & 3) * WAVE + (lane & (FEW_KEYS - 1))];
      const bool there = key0 + (lane & (FEW_KEYS - 1)) < keys && t < to;
      const bool named = id >= 0 && id < a.pages.n_pages;
      if (plain && __all(there && named)) {
        // A load's rows lie in one page: its base is the same for all lanes.
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          const int64_t off = ((int64_t)__builtin_amdgcn_readlane(id, i * LOAD_ROWS) * a.kv_heads + head) * head_bytes +
                              ((key0 + i * LOAD_ROWS) & slot_mask) * row_bytes;
          load_to_lds(a.pages.k, off, lane_at[i % 4], dst + i * (WAVE * 16));
          load_to_lds(a.pages.v, off, lane_at[i % 4], dst + L::HALF + i * (WAVE * 16));
        }
        return;
      }
      if (there && !named && a.failure != nullptr) *a.failure = a.code;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const int r = load_row + i * LOAD_ROWS, unit8 = load_slot ^ tile_swizzle<D>(r);
        const int page = __shfl(id, r);
        const int64_t off = ((int64_t)page * a.kv_heads + head) * head_bytes + ((key0 + r) & slot_mask) * row_bytes + unit8 * 16;
        const bool live = key0 + r < keys && t < to && page >= 0 && page < a.pages.n_pages && unit8 * 8 < a.dim;
        load_to_lds(live ? (const void *)((const char *)a.pages.k + off) : (const void *)&g_zeros, dst + i * (WAVE * 16));
        load_to_lds(live ? (const void *)((const char *)a.pages.v + off) : (const void *)&g_zeros,
                    dst + L::HALF + i * (WAVE * 16));
      }
    };

    // In flight while tile t is multiplied: the page numbers of t + 2 (older),
    // then the 2 LOADS loads of tile t + 1.
    // The queries have arrived before the loop: inside it the compiler would wait for
    // them, and with them for the tiles in flight, in every round.
#pragma unroll
    for (int ct = 0; ct < CT; ct++)
#pragma unroll
      for (int k = 0; k < D / 32; k++)
        asm volatile("" : "+v"(q[ct][k].x), "+v"(q[ct][k].y), "+v"(q[ct][k].z), "+v"(q[ct][k].w));
    wait_loads();
    fetch(from);
    fetch_ids(from + 2);
    fetch(from + 1);
    for (int t = from; t < to; t++) {
      wait_older_than<2 * LOADS>();
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
      const bool masked = key0 + FEW_KEYS - 1 > first_limit;
      if (masked) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
          for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (key0 + 16 * b + 4 * sigma + i > limit[ct]) w[ct][b][i] = -INFINITY;
        // Tokens of the unit see different keys of this tile: a value that a row
        // does not see must not reach it, and 0 * NaN would.  Values that are not
        // finite are added one by one and taken out of the tile.
        if (tokens > 1) {
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
                    if ((bits & E::exponent) == E::exponent && key0 + j <= limit[ct]) o[ct][dt][i] += E::load(bits);
                }
#pragma unroll
            for (int i = 0; i < LOADS * 8; i++) {
              uint16_t *x = reinterpret_cast<uint16_t *>(kt + L::HALF) + (i / 8 * WAVE + lane) * 8 + i % 8;
              if ((*x & E::exponent) == E::exponent) *x = 0;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
      }
      uint4 p[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ct++) {
        float high = w[ct][0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) high = fmaxf(high, w[ct][i >> 2][i & 3]);
        high = fold_quarters(high, FMax()) * a.scale_log2;
        if (__any(high > top[ct] + AT_RESCALE)) {
          const float now = fmaxf(top[ct], high);
          const float factor = now == -INFINITY ? 1.0f : exp2f(top[ct] - now);
          top[ct] = now;
          sum[ct] *= factor;
#pragma unroll
          for (int dt = 0; dt < D / 16; dt++) o[ct][dt] *= factor;
        }
        const float shift = top[ct] == -INFINITY ? 0.0f : top[ct];
        f32x8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[i] = __builtin_amdgcn_exp2f(fmaf(w[ct][i >> 2][i & 3], a.scale_log2, -shift));
          sum[ct] += x[i];
        }
        p[ct] = E::pack(x);
      }
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) {
        const auto read = [&](int h) __attribute__((always_inline)) {
          return bit_cast<uint2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (i16x4 __attribute__((address_space(3))) *)(kt + v_at[dt][h])));
        };
        const uint2 lo = read(0), hi = read(1);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) o[ct][dt] = E::mfma16(uint4{lo.x, lo.y, hi.x, hi.y}, p[ct], o[ct][dt]);
      }
      // The tile has been read (its reads have returned before its products); the
      // stage takes the next but one.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      fetch_ids(t + 3);
      fetch(t + 2);
    }
    wait_loads();

    const bool whole = from == 0 && to == key_tiles;
    const int64_t part = few_slot(number, from == 0 ? 1 : 0, ROWS);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      const int row = ct * 16 + col;
      const float all = fold_quarters(sum[ct], FAdd());
      if (row >= rows) continue;
      if (!whole) {
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++)
          *reinterpret_cast<f32x4 *>(a.part_o + (part + row) * D + dt * 16 + 4 * quarter) = o[ct][dt];
        if (quarter == 0) {
          a.part_ml[2 * (part + row)] = top[ct];
          a.part_ml[2 * (part + row) + 1] = all;
        }
        continue;
      }
      const int64_t out_row = (int64_t)s.first + t0 + row / a.group;
      const int q_head = head * a.group + row % a.group;
      const bool empty = top[ct] == -INFINITY;  // only scores of -inf
      const float inverse = empty ? 0.0f : 1.0f / all;
      uint16_t *dst = a.out.at(out_row, q_head);
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) {
        const int d = dt * 16 + 4 * quarter;
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = E::store(empty ? 0.0f : o[ct][dt][i] * inverse);
        if (d < a.dim) *reinterpret_cast<uint2 *>(dst + d) = uint2{x[0] | x[1] << 16, x[2] | x[3] << 16};
      }
      if (a.lse != nullptr && quarter == 0)
        a.lse[out_row * a.heads + q_head] = empty ? -INFINITY : (top[ct] + log2f(all)) * LN2;
    }
  }
}

// Joins the parts: a block a unit and join_rows of its rows.  A thread takes
// four components of a row; where there are fewer rows several threads share the
// parts of one.  Parts are taken in order, WAVE at a time, with the running
// maximum and sum.
template <class E, int D, int ROWS>
__global__ __launch_bounds__(FEW_THREADS) void attention_few_join_kernel(AttentionArgs a, int waves, int join_rows) {
  constexpr int FOURS = D / 4, JOIN_ROWS = FEW_THREADS / FOURS, BATCH = 8;
  __shared__ FewTable seqs;
  __shared__ int64_t units_before[FEW_THREADS];
  __shared__ float tops[JOIN_ROWS], sums[JOIN_ROWS], factors[JOIN_ROWS], weights[JOIN_ROWS][WAVE];
  __shared__ f32x4 shared[FEW_THREADS];
  const int per_tile = ROWS / a.group;
  const FewLine line = few_line(a, per_tile, waves, seqs, units_before);
  // The unit of this number, in the order of the line: the row tiles of a
  // sequence, heads inside them.
  const int thread = few_thread(units_before, blockIdx.x);
  int64_t number = blockIdx.x - units_before[thread], precede = seqs.before[thread];
  FewSeq s;
  for (int64_t i = thread * line.each;; i++) {
    if (i >= (thread + 1) * line.each || i >= a.m) return;
    s = line.seq(a, per_tile, i);
    const int64_t units = s.units(a.kv_heads);
    if (number < units) break;
    number -= units;
    precede += s.places(a.kv_heads);
  }
  const int head = (int)(number % a.kv_heads), t0 = (int)(number / a.kv_heads) * per_tile;
  // Its first and last tile, and the waves that had them.
  const int64_t begin = precede + number * s.unit() + FEW_START, last = begin + s.key_tiles() - 1;
  const int64_t w0 = few_divide(begin, line.piece), w1 = few_divide(last, line.piece);
  const int row0 = blockIdx.y * join_rows;
  int rows = (s.len - t0 < per_tile ? s.len - t0 : per_tile) * a.group - row0;
  if (w0 == w1 || rows <= 0) return;  // one wave had it all
  if (rows > join_rows) rows = join_rows;
  const auto part = [&](int64_t w) { return few_slot(w, w * line.piece <= begin ? 1 : 0, ROWS) + row0; };
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
      f = top == -INFINITY ? 0.0f : exp2f(f - top);
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
  const bool empty = tops[row] == -INFINITY;
  const float inverse = empty ? 0.0f : 1.0f / sums[row];
  const int64_t out_row = (int64_t)s.first + t0 + (row0 + row) / a.group;
  const int q_head = head * a.group + (row0 + row) % a.group;
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

size_t few_workspace(int rows, int64_t head_dim) {
  const int64_t waves = head_dim <= 64 ? few_waves<64>() : few_waves<128>();
  return (size_t)(2 * waves * rows) * ((head_dim <= 64 ? 64 : 128) + 2) * sizeof(float);
}

template <class E, int D, int ROWS>
static int launch_few_of(hipStream_t stream, AttentionArgs a, void *workspace) {
  constexpr int LDS = FewLds<D>::BYTES * FEW_WAVES;
  const auto kernel = attention_few_kernel<E, D, ROWS>;
  static const hipError_t raised =
      hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (raised != hipSuccess) return (int)raised;
  a.part_o = (float *)workspace;
  a.part_ml = a.part_o + (int64_t)2 * few_waves<D>() * ROWS * D;
  const int64_t units = most_tiles(a.q_rows, a.m, ROWS / a.group) * a.kv_heads;
  if (units > INT32_MAX) return FA_ENOTSUP;
  kernel<<<dim3(few_waves<D>() / FEW_WAVES), FEW_THREADS, LDS, stream>>>(a);
  const int rc = launch_status();
  if (rc != 0) return rc;
  // Rows a block of the second kernel joins: as many as its threads hold, fewer
  // while there are blocks to spare.
  const int64_t rows = ROWS / a.group * a.group;  // of a unit, at most
  int join_rows = FEW_THREADS / (D / 4);
  while (join_rows > 1 && units * ceil_div(rows, join_rows) < NUM_CUS_HINT) join_rows /= 2;
  const dim3 grid((unsigned)units, (unsigned)ceil_div(rows, join_rows));
  attention_few_join_kernel<E, D, ROWS><<<grid, FEW_THREADS, 0, stream>>>(a, few_waves<D>(), join_rows);
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
