// What the attention kernels (attention.hip, attention_few.hip, attention_grad.hip,
// kv_append.hip) share: argument checks on the host, 16-bit element types, arrays of heads and
// the walk over segments on the device.
#pragma once
#include "dispatch.hip.h"

namespace fa {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>), in order.
template <int N, class F> __device__ __forceinline__ void static_for(F &&f) {
  if constexpr (N > 0) {
    static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>());
  }
}

// 16-bit element types.  `store` and `pack` round to nearest even; `mfma` is
// C += A B with A 32 x 16, B 16 x 32: lane l holds row (column) l % 32 of A (B)
// and the eight k from 8 (l / 32), and of C column l % 32, rows
// 8 (i / 4) + 4 (l / 32) + i % 4 for i < 16.
struct ElemF16 {
  static constexpr uint32_t exponent = 0x7c00;  // all ones: infinity or NaN
  static __device__ __forceinline__ float load(uint16_t b) { return (float)bit_cast<_Float16>(b); }
  static __device__ __forceinline__ uint16_t store(float f) { return bit_cast<uint16_t>((_Float16)f); }
  static __device__ __forceinline__ uint4 pack(f32x8 x) {
    return bit_cast<uint4>(__builtin_convertvector(x, f16x8));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return bit_cast<uint32_t>(__builtin_convertvector(f32x2{lo, hi}, f16x2));
  }
  static __device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(bit_cast<f16x8>(a), bit_cast<f16x8>(b), c, 0, 0, 0);
  }
  // 16 x 32 times 32 x 16: row (column) l % 16, k from 8 (l / 16); C rows 4 (l / 16) + i.
  static __device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(bit_cast<f16x8>(a), bit_cast<f16x8>(b), c, 0, 0, 0);
  }
};
struct ElemBF16 {
  static constexpr uint32_t exponent = 0x7f80;
  static __device__ __forceinline__ float load(uint16_t b) { return bit_cast<float>((uint32_t)b << 16); }
  static __device__ __forceinline__ uint16_t store(float f) { return bit_cast<uint16_t>((__bf16)f); }
  static __device__ __forceinline__ uint4 pack(f32x8 x) {
    return bit_cast<uint4>(__builtin_convertvector(x, bf16x8));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return bit_cast<uint32_t>(__builtin_convertvector(f32x2{lo, hi}, bf16x2));
  }
  static __device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bit_cast<bf16x8>(a), bit_cast<bf16x8>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bit_cast<bf16x8>(a), bit_cast<bf16x8>(b), c, 0, 0, 0);
  }
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

// What the forward kernels take.
struct AttentionArgs {
  Heads q, k, v, out;
  float *lse;
  int64_t q_rows, k_rows;
  int heads, kv_heads, group, dim;
  const int64_t *q_offsets, *q_lens, *k_offsets, *k_lens;
  int64_t m;
  float scale_log2;  // scale * log2(e)
  int causal;
  bool by_keys;  // the order of tiles (find_tile_by_keys)
  int32_t *failure, code;
  // paged only: the cache; keys of a unit that one block takes, and where parts go
  Pages pages;
  int chunk, splits;
  float *part_o, *part_ml;
  int64_t most_units;
};

// A wave rescales its output only when a maximum has grown by 2^8 since it last
// did: until then weights are at most 2^8, which f16 and bf16 hold as well as 1.
constexpr float AT_RESCALE = 8.0f;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

// attention_few.hip: attention over the cache for few query rows a sequence.
// Rows a unit of work holds for such a call, or 0 if the other kernel should take it.
int few_rows(int64_t n, int64_t heads, int64_t kv_heads, int64_t m);
// Its workspace, 0 where one launch does it (`keys`: what a row of the table holds).
size_t few_workspace(int rows, int64_t n, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t m, int64_t keys);
int launch_few(hipStream_t stream, fa_dtype t, int rows, const AttentionArgs &a, void *workspace);

// ------------------------------------------------------------------ segments
// Segment i as the rules of fa_segred_irregular read it: inside [0, n), not
// before the end of its predecessor.  All loads are issued before any is looked at.
__device__ __forceinline__ bool segment_ok(const int64_t *offsets, const int64_t *lens, int64_t i,
                                           int64_t n, int64_t &first, int64_t &len) {
  const int64_t j = i > 0 ? i - 1 : 0, before = offsets[j], taken = lens[j];
  first = offsets[i];
  len = lens[i];
  // (unsigned: differences of whatever the arrays hold, and negative lengths are large)
  const bool inside = (first >= 0) & (first <= n) & ((uint64_t)len <= (uint64_t)n - (uint64_t)first);
  const bool behind = (i == 0) | ((before >= 0) & (before <= first) & ((uint64_t)taken <= (uint64_t)first - (uint64_t)before));
  return inside & behind;
}

// Where a segment ends, 0 for one that does not lie inside [0, n).
__device__ __forceinline__ int segment_end(int64_t first, int64_t len, int64_t n) {
  return (first >= 0) & (first <= n) & ((uint64_t)len <= (uint64_t)n - (uint64_t)first) ? (int)(first + len) : 0;
}
// A segment that lies behind its predecessor lies behind all earlier ones as long as
// those keep the rules.  Behind a broken one it has to be compared with all of them.
// A wave looks at its segments in order, WAVE at a time; this is what goes from one
// batch to the next.
struct SegChain {
  bool broken = false;  // a segment so far breaks the rules; `end` is then the end of all so far
  int end = 0;
  // Whether segment base + lane, ok by segment_ok, also starts behind all before it.
  __device__ __forceinline__ bool keep(bool ok, int64_t first, int64_t len, const int64_t *offsets, const int64_t *lens,
                                       int64_t m, int64_t n, int64_t base) {
    const bool live = base + lane_id() < m;
    if (!broken) {
      if (!__any(live & !ok)) return ok;
      broken = true;
      if (base > 0) end = (int)(offsets[base - 1] + lens[base - 1]);
    }
    const int upto = wave_incl_scan<int, OpMax<int>>(live ? segment_end(first, len, n) : 0);
    const int before = OpMax<int>::apply(wave_shift_up1<int, OpMax<int>>(upto), end);
    end = OpMax<int>::apply(end, read_lane(upto, WAVE - 1));
    return ok & (first >= before);
  }
};

// Work on a segment comes in tiles of `per_tile` rows, numbered through the
// segments in order; the tile of number `number`, or false if there are fewer.
// The same for the whole wave, which looks at 64 segments at a time.  A broken
// segment (also one whose partner in `offsets2` is broken, or that overlaps an
// earlier one) has no tiles.
struct SegTile {
  int64_t seg, tile, tiles;  // segment, tile in it, tiles it has
  int64_t first, len;
  int64_t first2, len2;  // the partner segment's
};
__device__ __forceinline__ bool find_tile(const int64_t *offsets, const int64_t *lens, int64_t n,
                                          const int64_t *offsets2, const int64_t *lens2, int64_t n2, int64_t m,
                                          int per_tile, int64_t number, SegTile &t) {
  int64_t before = 0;
  SegChain chain, chain2;
  for (int64_t base = 0; base < m; base += WAVE) {
    const int64_t i = base + lane_id(), at = i < m ? i : m - 1;
    int64_t f, l, f2 = 0, l2 = 0;
    bool ok = segment_ok(offsets, lens, at, n, f, l) & (i < m);
    if (offsets2 != nullptr) {
      const bool ok2 = segment_ok(offsets2, lens2, at, n2, f2, l2);
      ok = chain.keep(ok, f, l, offsets, lens, m, n, base) & chain2.keep(ok2, f2, l2, offsets2, lens2, m, n2, base);
    } else {
      ok = chain.keep(ok, f, l, offsets, lens, m, n, base);
    }
    // lengths are below 2^31
    const int64_t tiles = ok ? ((uint32_t)l + (uint32_t)per_tile - 1) / (uint32_t)per_tile : 0;
    const int64_t upto = before + wave_incl_scan<int64_t, OpAdd<int64_t>>(tiles);
    const uint64_t past = __ballot(upto > number);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      t.seg = base + at;
      t.tiles = read_lane(tiles, at);
      t.tile = number - (read_lane(upto, at) - t.tiles);
      t.first = read_lane(f, at);
      t.len = read_lane(l, at);
      t.first2 = read_lane(f2, at);
      t.len2 = read_lane(l2, at);
      return true;
    }
    before = read_lane(upto, WAVE - 1);
  }
  return false;
}

// The same for up to WAVE segments, a segment a lane (`ok` if it has one), with the
// tiles that see most keys first, whatever segment they are of: started in this
// order, blocks end together.  A tile's level is the number of keys it sees, in
// tiles, `seen` keys for the first one: of the one `tile` behind it top - tile if
// causal, else top.  The highest level is found that more than `number` tiles reach.
__device__ __forceinline__ void find_tile_by_keys(bool ok, int64_t first, int64_t len, int64_t first2, int64_t len2, int64_t seen,
                                                  int per_tile, bool causal, int64_t number, SegTile &t, bool &found) {
  const int tiles = ok ? (int)(((uint32_t)len + (uint32_t)per_tile - 1) / (uint32_t)per_tile) : 0;
  const int top = tiles > 0 ? (int)(seen / per_tile) : INT32_MIN / 2;
  const auto upto_level = [&](int x) {
    const int n = top - x + 1;
    return n <= 0 ? 0 : !causal || n > tiles ? tiles : n;
  };
  int high = wave_reduce<int, OpMax<int>>(top);
  int low = wave_reduce<int, OpMin<int>>(tiles > 0 ? causal ? top - tiles + 1 : top : INT32_MAX / 2);
  const int64_t all = wave_reduce<int64_t, OpAdd<int64_t>>(tiles);
  found = number < all;
  if (!found) return;
  while (low < high) {
    const int x = low + (high - low + 1) / 2;
    if (wave_reduce<int, OpAdd<int>>(upto_level(x)) > (int)number) low = x;
    else high = x - 1;
  }
  const int above = upto_level(low + 1), here = upto_level(low) - above;
  const int rank = (int)number - wave_reduce<int, OpAdd<int>>(above);
  const int upto = wave_incl_scan<int, OpAdd<int>>(here);
  const int at = __builtin_ctzll(__ballot(upto > rank));
  t.seg = at;
  t.tiles = read_lane(tiles, at);
  t.tile = read_lane(above, at) + rank - (read_lane(upto, at) - read_lane(here, at));
  t.first = read_lane(first, at);
  t.len = read_lane(len, at);
  t.first2 = read_lane(first2, at);
  t.len2 = read_lane(len2, at);
}

// Whether blocks of units (at most `units`, of 128 query rows) take the tiles by
// keys: where the chip holds half of them or more at a time (two blocks a CU, three
// for D = 64).  With more the long ones even out, and tiles of one segment next to
// each other share their keys in L2.  (600 units of six sequences with up to 8192
// cached tokens, not split over keys, 288 -> 267 us, 1100 of forty prompts of up to
// 333 15.4 -> 13.5; but 1400 of twenty sequences, forward and gradient, 290 -> 306.)
inline bool takes_by_keys(int64_t units, int64_t m, int64_t dim) {
  return m <= WAVE && units <= 2 * NUM_CUS_HINT * (dim <= 64 ? 3 : 2);
}

// Tiles that n rows in m segments make at most (empty segments make none).
inline int64_t most_tiles(int64_t n, int64_t m, int64_t per_tile) {
  const int64_t by_parts = (n + m * (per_tile - 1)) / per_tile;
  return by_parts < n ? by_parts : n;
}

// ------------------------------------------------------------- tiles in LDS
// Rows of D 16-bit components (D 64 or 128) in 16-byte units; unit u of row r
// sits in slot u ^ f(r).  f makes both ways of reading a tile free of bank
// conflicts: 16 consecutive rows, one unit each (128-bit operand reads; f
// differs for all rows that share a bank), and four rows (4-aligned) of 64
// consecutive bytes (the transposing reads; f differs in the bits above the
// lowest two, which move 64-byte groups).
template <int D> __device__ __forceinline__ int tile_swizzle(int r) {
  static_assert(D == 64 || D == 128, "rows of 128 or 256 bytes");
  if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}
template <int D> __device__ __forceinline__ int tile_offset(int r, int unit) {
  return r * (D * 2) + ((unit ^ tile_swizzle<D>(r)) << 4);
}

// Sixteen bytes a lane from global memory into LDS at `lds` (wave uniform) +
// 16 * lane.  The compiler does not see this load: wait_loads() and a barrier
// come before what it brings is read.
__device__ __forceinline__ void load_to_lds(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                   __builtin_amdgcn_readfirstlane(lds)),
               "v"(src)
               : "memory", "m0");
}
// The same from base + offset, base the same for the wave.
__device__ __forceinline__ uint64_t wave_address(const void *base) {
  const uint64_t at = (uint64_t)base;
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at);
}
__device__ __forceinline__ void load_to_lds(const void *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                   __builtin_amdgcn_readfirstlane(lds)),
               "v"(offset), "s"(wave_address(base))
               : "memory", "m0");
}
// Four bytes a lane.
__device__ __forceinline__ void load_word_to_lds(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(
                   __builtin_amdgcn_readfirstlane(lds)),
               "v"(src)
               : "memory", "m0");
}
// And for data that is read once: the non-temporal policy (decoding 64 sequences
// 98.8 -> 87.3 us, 5.9 TB/s).
__device__ __forceinline__ void stream_to_lds(const void *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(
                   __builtin_amdgcn_readfirstlane(lds)),
               "v"(offset), "s"(wave_address(base))
               : "memory", "m0");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// All but the N youngest loads have arrived.
template <int N> __device__ __forceinline__ void wait_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// A barrier that leaves younger loads in flight; what was read of LDS has arrived.
__device__ __forceinline__ void block_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char *)p;
}

// How a lane reads a tile for the 32 x 32 x 16 products; places are kept, so that
// a read is an instruction with a constant offset.
template <int D> struct TileReads {
  int row[D / 16], column[D / 32][2];
  __device__ __forceinline__ TileReads() {
    const int l = lane_id(), r = l & 15;
#pragma unroll
    for (int s = 0; s < D / 16; s++) row[s] = tile_offset<D>(l & 31, 2 * s + (l >> 5));
#pragma unroll
    for (int t = 0; t < D / 32; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int c = t * 32 + ((l >> 4) & 1) * 16 + 4 * (r & 3);
        column[t][h] = tile_offset<D>(8 * h + 4 * (l >> 5) + (r >> 2), c >> 3) + (c & 7) * 2;
      }
  }
  // Operand of a product over components: row r0 + l % 32 (r0 a multiple of 32),
  // components 16 s + 8 (l / 32) ...
  __device__ __forceinline__ uint4 rows(const unsigned char *tile, int r0, int s) const {
    return *reinterpret_cast<const uint4 *>(tile + r0 * (D * 2) + row[s]);
  }
  // Operand of a product over rows: for lane l component 32 t + l % 32 of the rows
  // r0 + 4 (l / 32) + {0..3, 8..11} (r0 a multiple of 16): the rows whose products a
  // lane holds in registers 0..7 of an MFMA result, so that a result is the other
  // operand as it stands.
  __device__ __forceinline__ uint4 columns(const unsigned char *tile, int r0, int t) const {
    const auto read = [&](int h) __attribute__((always_inline)) {
      const unsigned char *p = tile + r0 * (D * 2) + column[t][h];
      return bit_cast<uint2>(
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((i16x4 __attribute__((address_space(3))) *)(p)));
    };
    const uint2 lo = read(0), hi = read(1);
    return uint4{lo.x, lo.y, hi.x, hi.y};
  }
};

static __device__ uint4 g_zeros;  // what is loaded in place of rows and units that are not there

// A block's loads of a tile of 64 rows.  Load i of a wave brings ROWS rows from
// first_row + i * STEP on; a lane brings 16-byte unit `unit` of row `lane_row` of
// them (its slot and, with it, its unit are the same in all its rows).  Lanes
// whose unit lies past dim load nothing: those places are cleared beforehand.
template <int D, int THREADS> struct TileLoads {
  static constexpr int BYTES = 64 * D * 2, COUNT = BYTES / (THREADS * 16), STEP = 64 / COUNT, ROWS = WAVE / (D / 8);
  static_assert(COUNT > 0 && STEP % 16 == 0, "the swizzle repeats every 16 rows");
  int first_row, lane_row, unit;
  bool live;
  uint32_t lds;  // where the wave's first load goes in the tile at LDS address 0
  __device__ __forceinline__ explicit TileLoads(int dim) {
    first_row = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE) * ROWS;
    lane_row = lane_id() / (D / 8);
    unit = (threadIdx.x % (D / 8)) ^ tile_swizzle<D>(first_row + lane_row);
    live = unit * 8 < dim;
    lds = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE) * 1024;
  }
  // The row load i of this lane brings.
  __device__ __forceinline__ int row(int i) const { return first_row + lane_row + i * STEP; }
  // This lane's place from its load's first row on.
  __device__ __forceinline__ uint32_t offset(int64_t row_stride) const {
    return (uint32_t)lane_row * (uint32_t)row_stride * 2 + unit * 16;
  }
  __device__ __forceinline__ uint32_t place(uint32_t tile, int i) const { return tile + lds + i * (THREADS * 16); }
  // A whole tile of equally spaced rows.
  __device__ __forceinline__ void load(const uint16_t *first, int64_t row_stride, uint32_t offset, uint32_t tile) const {
    if (live) {
#pragma unroll
      for (int i = 0; i < COUNT; i++) load_to_lds(first + (int64_t)(first_row + i * STEP) * row_stride, offset, place(tile, i));
    }
  }
  // The same where only the first `rows` are there: the rest are zeros.
  __device__ __forceinline__ void load(const uint16_t *first, int64_t row_stride, int rows, uint32_t tile) const {
    if (live) {
#pragma unroll
      for (int i = 0; i < COUNT; i++) load(first + row(i) * row_stride, row(i) < rows, tile, i);
    }
  }
  // Load i from this lane's row, or zeros.
  __device__ __forceinline__ void load(const uint16_t *row_data, bool there, uint32_t tile, int i) const {
    load_to_lds(there ? (const void *)(row_data + unit * 8) : (const void *)&g_zeros, place(tile, i));
  }
};
// Clears `bytes` of LDS (a multiple of 16) where units past dim would stay as they
// are; a barrier comes before the first loads.
template <int D> __device__ __forceinline__ void clear_unloaded(unsigned char *lds, int bytes, int dim) {
  if (dim == D) return;
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<uint4 *>(lds + i) = uint4{0, 0, 0, 0};
  __syncthreads();
}

// Eight components of a row from c on, zeros past dim.  (A load under a condition
// would be waited for before the next is issued.)
__device__ __forceinline__ uint4 load_unit(const uint16_t *row, int c, int dim) {
  const uint4 x = *reinterpret_cast<const uint4 *>(row + (c < dim ? c : 0));
  return c < dim ? x : uint4{0, 0, 0, 0};
}

// The compiler's own loads into x have arrived here.  Left to itself it waits for
// them where x is first used, and inside a loop with every load in flight.
template <int N> __device__ __forceinline__ void arrived(uint4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+v"(x[i].x), "+v"(x[i].y), "+v"(x[i].z), "+v"(x[i].w));
}

// Maximum (sum) over the lanes 16 and 32 apart, and over lanes 32 apart alone.
// A swap of a register with itself leaves the even rows (the lower half) in one
// result and the odd rows (the upper half) in the other, for all lanes.
template <class F> __device__ __forceinline__ float fold_halves(float x, F f) {
  const auto r = __builtin_amdgcn_permlane32_swap(bit_cast<uint32_t>(x), bit_cast<uint32_t>(x), false, false);
  return f(bit_cast<float>((uint32_t)r[0]), bit_cast<float>((uint32_t)r[1]));
}
template <class F> __device__ __forceinline__ float fold_quarters(float x, F f) {
  const auto r = __builtin_amdgcn_permlane16_swap(bit_cast<uint32_t>(x), bit_cast<uint32_t>(x), false, false);
  return fold_halves(f(bit_cast<float>((uint32_t)r[0]), bit_cast<float>((uint32_t)r[1])), f);
}
struct FMax {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct FAdd {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// A lane's column of a transposed result (C of E::mfma, D / 32 of them), times
// factor, as a row of 16-bit components; zeros if `zero`, nothing unless `there`.
// Two lanes of the wave's halves hold four of every eight components each; they
// trade so that each stores 16 bytes.  All lanes of the wave take part.
template <class E, int D>
__device__ __forceinline__ void store_column(const f32x16 (&x)[D / 32], float factor, uint16_t *dst, int dim, bool there,
                                             bool zero = false) {
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        w[j] = zero ? 0 : E::pack(x[t][i + 2 * j] * factor, x[t][i + 2 * j + 1] * factor);
      const auto lo = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto hi = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      const int d = t * 32 + 2 * i + 8 * (lane_id() >> 5);
      if (there && d < dim)
        *reinterpret_cast<uint4 *>(dst + d) = uint4{(uint32_t)lo[0], (uint32_t)hi[0], (uint32_t)lo[1], (uint32_t)hi[1]};
    }
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

// Lanes reach the rows of a load by 32-bit offsets.
constexpr int64_t AT_MOST_STRIDE = (int64_t)1 << 27;

inline int check_heads(const fa_heads *x, int64_t rows, int64_t heads, int64_t dim, bool written) {
  if (x == nullptr || (x->data == nullptr && rows > 0)) return FA_EINVAL;
  if (x->row_stride < 0 || x->head_stride < 0) return FA_EINVAL;
  if (!is_aligned(x->data, 16) || x->row_stride % 8 != 0 || x->head_stride % 8 != 0) return FA_EALIGN;
  if (!heads_span_ok(rows, heads, dim, x)) return FA_EINVAL;
  if (rows > 1 && x->row_stride >= AT_MOST_STRIDE) return FA_ENOTSUP;
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

// Most blocks of 256 threads along one dimension of a launch (2^32 threads).
constexpr int64_t AT_MOST_BLOCKS = ((int64_t)1 << 24) - 1;
// Most rows and positions: 32-bit numbers that may run a few tiles past them.
constexpr int64_t AT_MOST_ROWS = INT32_MAX - 4095;

// Scores are scaled by scale * log2(e), in f32.
inline int check_scale(float scale) { return scale > 0.0f && scale * LOG2E <= FLT_MAX ? 0 : FA_EINVAL; }

inline int check_segments(const int64_t *offsets, const int64_t *lens, int64_t m, int64_t n) {
  if (m < 0 || n < 0) return FA_EINVAL;
  if (m > AT_MOST_ROWS || n > AT_MOST_ROWS) return FA_ENOTSUP;
  if (m > 0 && (offsets == nullptr || lens == nullptr)) return FA_EINVAL;
  if (!is_aligned(offsets, 8) || !is_aligned(lens, 8)) return FA_EALIGN;
  return 0;
}

inline int check_pages(const void *k_pages, const void *v_pages, int64_t n_pages, int64_t page_size,
                       const int32_t *table, int64_t cols, const int64_t *past_lens, int64_t kv_heads,
                       int64_t head_dim) {
  if (n_pages < 0 || page_size <= 0 || cols < 0) return FA_EINVAL;
  if ((page_size & (page_size - 1)) != 0 || n_pages > INT32_MAX) return FA_ENOTSUP;
  if ((__int128)cols * page_size > AT_MOST_ROWS) return FA_ENOTSUP;
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
