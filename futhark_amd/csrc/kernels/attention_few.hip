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
constexpr int FEW_LEAST_TILES = 8;  // a piece is at least this long
constexpr int FEW_THREADS = 256, FEW_WAVES = FEW_THREADS / WAVE;

// Waves a launch has: what fits the LDS of the chip (four waves of 33 KiB a CU,
// twice as many for D = 64).
template <int D> constexpr int few_waves() { return NUM_CUS_HINT * FEW_WAVES * (D == 128 ? 1 : 2); }

// LDS of a wave: two stages of K and V, four slots of page numbers.
template <int D> struct FewLds {
  static constexpr int HALF = FEW_KEYS * D * 2, STAGE = 2 * HALF, IDS = 2 * STAGE, BYTES = IDS + 4 * WAVE * 4;
};

// A sequence as the line of tiles sees it.
struct FewSeq {
  int64_t first, past;
  int len, row_tiles, key_tiles;
  __device__ __forceinline__ int64_t tiles(int kv_heads) const { return (int64_t)row_tiles * key_tiles * kv_heads; }
};
__device__ __forceinline__ FewSeq few_seq(const AttentionArgs &a, int per_tile, int64_t i, bool report) {
  FewSeq s = {0, 0, 0, 0, 0};
  int64_t first, len;
  bool ok = segment_ok(a.q_offsets, a.q_lens, i, a.q_rows, first, len);
  const int64_t past = a.pages.past_lens[i], room = a.pages.capacity();
  ok = ok && (len == 0 || (past >= 0 && past <= room && len <= room - past));
  if (ok) {
    s.first = first;
    s.past = past;
    s.len = (int)len;
    s.row_tiles = (int)((len + per_tile - 1) / per_tile);
    s.key_tiles = len > 0 ? (int)((past + len + FEW_KEYS - 1) / FEW_KEYS) : 0;
  } else if (report && a.failure != nullptr) {
    *a.failure = a.code;
  }
  return s;
}

// The line's length and the place where a block's threads look for a position:
// thread t counts sequences t * each .. (t + 1) * each - 1, before[t] tiles precede them.
struct FewLine {
  int64_t total, piece, each;
  int64_t *before;  // [FEW_THREADS] in LDS
};
__device__ __forceinline__ FewLine few_line(const AttentionArgs &a, int per_tile, int waves, int64_t *before) {
  FewLine line;
  line.each = (a.m + FEW_THREADS - 1) / FEW_THREADS;
  line.before = before;
  int64_t mine = 0;
  for (int64_t i = threadIdx.x * line.each; i < (threadIdx.x + 1) * line.each && i < a.m; i++)
    mine += few_seq(a, per_tile, i, blockIdx.x == 0).tiles(a.kv_heads);
  const int64_t upto = wave_incl_scan<int64_t, OpAdd<int64_t>>(mine);
  __shared__ int64_t wave_total[FEW_WAVES];
  if (lane_id() == WAVE - 1) wave_total[threadIdx.x / WAVE] = upto;
  __syncthreads();
  int64_t base = 0;
  line.total = 0;
  for (int w = 0; w < FEW_WAVES; w++) {
    if (w < (int)(threadIdx.x / WAVE)) base += wave_total[w];
    line.total += wave_total[w];
  }
  before[threadIdx.x] = base + upto - mine;
  __syncthreads();
  const int64_t even = (line.total + waves - 1) / waves;
  line.piece = even < FEW_LEAST_TILES ? FEW_LEAST_TILES : even;
  return line;
}
// The sequence that holds position `at` < total, and how many tiles precede it;
// the same for the whole wave.
__device__ __forceinline__ int64_t few_find(const AttentionArgs &a, int per_tile, const FewLine &line, int64_t at,
                                            int64_t &precede) {
  int thread = -1;
  for (int b = 0; b < FEW_THREADS; b += WAVE) thread += __popcll(__ballot(line.before[b + lane_id()] <= at));
  int64_t i = thread * line.each;
  precede = line.before[thread];
  for (;; i++) {
    const int64_t tiles = few_seq(a, per_tile, i, false).tiles(a.kv_heads);
    if (at < precede + tiles || i + 1 >= a.m) return i;
    precede += tiles;
  }
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
  __shared__ int64_t before[FEW_THREADS];
  const int per_tile = ROWS / a.group;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int quarter = lane >> 4, col = lane & 15;
  const FewLine line = few_line(a, per_tile, gridDim.x * FEW_WAVES, before);
  const int64_t number = (int64_t)blockIdx.x * FEW_WAVES + wave;
  int64_t at = number * line.piece;
  const int64_t end = at + line.piece < line.total ? at + line.piece : line.total;
  if (at >= end) return;
  int64_t precede, seq = few_find(a, per_tile, line, at, precede);

  unsigned char *mine = lds + wave * L::BYTES;
  const uint32_t lds_base = lds_address(mine);
  int *ids = reinterpret_cast<int *>(mine + L::IDS);
  const int load_row = lane / (D / 8), load_slot = lane % (D / 8);
  const int64_t row_bytes = a.dim * 2, head_bytes = row_bytes << a.pages.page_shift;
  const int slot_mask = (1 << a.pages.page_shift) - 1;

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
    const FewSeq s = few_seq(a, per_tile, seq, false);
    const int64_t tiles = s.tiles(a.kv_heads);
    if (at >= precede + tiles) {
      precede += tiles;
      seq++;
      continue;
    }
    // Position in the sequence: row tile, head, key tile.
    const int64_t inside = at - precede, unit = inside / s.key_tiles;
    const int from = (int)(inside - unit * s.key_tiles);
    const int to = end - at < s.key_tiles - from ? (int)(from + (end - at)) : s.key_tiles;
    at += to - from;
    const int head = (int)(unit % a.kv_heads), t0 = (int)(unit / a.kv_heads) * per_tile;
    const int tokens = s.len - t0 < per_tile ? s.len - t0 : per_tile, rows = tokens * a.group;
    const int first_limit = (int)s.past + t0;         // last key the first token sees
    const int keys = first_limit + tokens;            // keys the last one sees
    const int64_t table = seq * a.pages.cols;

    uint4 q[CT][D / 32];
    int limit[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      const int row = ct * 16 + col < rows ? ct * 16 + col : rows - 1;
      limit[ct] = first_limit + row / a.group;
      const uint16_t *src = a.q.at(s.first + t0 + row / a.group, head * a.group + row % a.group);
#pragma unroll
      for (int k = 0; k < D / 32; k++) {
        const int c = 32 * k + 8 * quarter;
        q[ct][k] = c < a.dim ? *reinterpret_cast<const uint4 *>(src + c) : uint4{0, 0, 0, 0};
      }
    }
    // The queries are here before the loop: inside it the compiler would wait for
    // them, and with them for the tiles in flight, in every round.
#pragma unroll
    for (int ct = 0; ct < CT; ct++)
#pragma unroll
      for (int k = 0; k < D / 32; k++)
        asm volatile("" : "+v"(q[ct][k].x), "+v"(q[ct][k].y), "+v"(q[ct][k].z), "+v"(q[ct][k].w));
    f32x4 o[CT][D / 16];
    float top[CT], sum[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
      top[ct] = -INFINITY;
      sum[ct] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++) o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // Page numbers of the keys of tile t (and of the next 32, not used).
    const auto fetch_ids = [&](int t) __attribute__((always_inline)) {
      const int key = t * FEW_KEYS + lane < keys ? t * FEW_KEYS + lane : keys - 1;
      const int32_t *src = a.pages.table + table + (key >> a.pages.page_shift);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(
                       __builtin_amdgcn_readfirstlane(lds_base + L::IDS + (t & 3) * (WAVE * 4))),
                   "v"(src)
                   : "memory", "m0");
    };
    const auto fetch = [&](int t) __attribute__((always_inline)) {
      const uint32_t dst = lds_base + (t & 1) * L::STAGE;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        const int r = load_row + i * LOAD_ROWS, key = t * FEW_KEYS + r;
        const int unit8 = load_slot ^ tile_swizzle<D>(r);
        const int id = ids[(t & 3) * WAVE + r];
        const bool named = id >= 0 && id < a.pages.n_pages, there = key < keys && t < to;
        bad = bad || (there && !named);
        const int64_t off = ((int64_t)id * a.kv_heads + head) * head_bytes + (key & slot_mask) * row_bytes + unit8 * 16;
        const bool live = there && named && unit8 * 8 < a.dim;
        const void *ks = live ? (const void *)((const char *)a.pages.k + off) : (const void *)&g_zeros;
        const void *vs = live ? (const void *)((const char *)a.pages.v + off) : (const void *)&g_zeros;
        load_to_lds(ks, dst + i * (WAVE * 16));
        load_to_lds(vs, dst + L::HALF + i * (WAVE * 16));
      }
      if (bad && a.failure != nullptr) *a.failure = a.code;
    };

    // In flight while tile t is multiplied: the page numbers of t + 2 (older),
    // then the 2 LOADS loads of tile t + 1.
    fetch_ids(from);
    wait_loads();
    fetch_ids(from + 1);
    fetch(from);
    wait_older_than<2 * LOADS>();
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

    const bool whole = from == 0 && to == s.key_tiles;
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
      const int64_t out_row = s.first + t0 + row / a.group;
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

// Joins the parts: a block a unit, a wave a query row.
template <class E, int D, int ROWS> __global__ __launch_bounds__(FEW_THREADS) void attention_few_join_kernel(AttentionArgs a, int waves) {
  __shared__ int64_t before[FEW_THREADS];
  const int per_tile = ROWS / a.group, lane = lane_id();
  const FewLine line = few_line(a, per_tile, waves, before);
  // Units in the order of the line: a sequence's row tiles, heads inside them.
  SegTile t;
  if (!find_tile(a.q_offsets, a.q_lens, a.q_rows, nullptr, nullptr, 0, a.m, per_tile, blockIdx.x / a.kv_heads, t)) return;
  const FewSeq s = few_seq(a, per_tile, t.seg, false);
  if (s.key_tiles == 0) return;
  const int head = blockIdx.x % a.kv_heads;
  int64_t precede = line.before[t.seg / line.each];
  for (int64_t i = t.seg / line.each * line.each; i < t.seg; i++) precede += few_seq(a, per_tile, i, false).tiles(a.kv_heads);
  const int64_t begin = precede + (t.tile * a.kv_heads + head) * s.key_tiles;
  const int64_t w0 = begin / line.piece, w1 = (begin + s.key_tiles - 1) / line.piece;
  if (w0 == w1) return;  // one wave had it all
  const int t0 = (int)t.tile * per_tile, tokens = s.len - t0 < per_tile ? s.len - t0 : per_tile;
  for (int row = threadIdx.x / WAVE; row < tokens * a.group; row += FEW_WAVES) {
    const auto part = [&](int64_t w) { return few_slot(w, w * line.piece <= begin ? 1 : 0, ROWS) + row; };
    float top = -INFINITY;
    for (int64_t w = w0 + lane; w <= w1; w += WAVE) top = fmaxf(top, a.part_ml[2 * part(w)]);
    for (int step = 1; step < WAVE; step *= 2) top = fmaxf(top, __shfl_xor(top, step));
    float sum = 0.0f, o[D / WAVE] = {};
    if (top != -INFINITY) {
      for (int64_t base = w0; base <= w1; base += WAVE) {
        const int64_t w = base + lane;
        float f = 0.0f;
        if (w <= w1) {
          f = exp2f(a.part_ml[2 * part(w)] - top);
          sum += f * a.part_ml[2 * part(w) + 1];
        }
        const int count = w1 - base + 1 < WAVE ? (int)(w1 - base + 1) : WAVE;
#pragma unroll 8
        for (int j = 0; j < count; j++) {
          const float g = read_lane(f, j);
          const float *src = a.part_o + part(base + j) * D + lane;
#pragma unroll
          for (int c = 0; c < D / WAVE; c++) o[c] += g * src[c * WAVE];
        }
      }
      for (int step = 1; step < WAVE; step *= 2) sum += __shfl_xor(sum, step);
    }
    const int64_t out_row = s.first + t0 + row / a.group;
    const int q_head = head * a.group + row % a.group;
#pragma unroll
    for (int c = 0; c < D / WAVE; c++) {
      const int d = c * WAVE + lane;
      if (d < a.dim) a.out.at(out_row, q_head)[d] = E::store(top == -INFINITY ? 0.0f : o[c] / sum);
    }
    if (a.lse != nullptr && lane == 0)
      a.lse[out_row * a.heads + q_head] = top == -INFINITY ? -INFINITY : (top + log2f(sum)) * LN2;
  }
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
  attention_few_join_kernel<E, D, ROWS><<<dim3((unsigned)units), FEW_THREADS, 0, stream>>>(a, few_waves<D>());
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
