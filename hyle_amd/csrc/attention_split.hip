// attention_split.hip -- attention of a few query rows over many keys, split over the keys and joined: f16 / bf16 queries,
// keys and values of their type or e4m3, in memory or in a paged cache, there also in 4 bits.
//
// Bound by the bytes of keys and values, which are read once for all rows of a key head (its query heads times the new
// tokens).  The keys of all sequences, in tiles of 128, are dealt to a fixed number of chunks, however long each sequence is: a
// chunk is ceil(tiles / chunks) tiles of one sequence.  A block takes one chunk of one key head:
//   S^T[key, row] = K Q^T,  p = 2^(S^T c - m),  O^T[dim, row] = V^T P^T   (c = scale * log2(e))
// with the running maximum m and sum l of the softmax per lane (a lane's row is its column).  Weights are rounded once to the
// queries' type, which the matrix unit asks for (the mean distance of bf16 outputs from 64 bits, with weights in f32 / here: over 4 bits, one
// sequence of 131055 keys, 3.2e-4 / 3.4e-4, over 2048 keys of each key head in bf16 7.3e-5 / 1.09e-4; the outputs' own rounding is most
// of it); sums, statistics and what chunks leave are f32.  Up to 16 rows, its four waves each
// take 32 keys of every tile and do not meet before the end; 32 or 64 rows are dealt to the waves, which share the tile's keys
// in LDS (64 rows to every wave spilled: 93 sequences of 8 new tokens, 8 key heads of 128, 118 us, shared 68).  Keys go through LDS
// too, not only the values that are read by columns: whole rows side by side are whole cache lines, and only of those are
// non-temporal loads fast (64 sequences of 30 to 16384 keys, 8 key heads of 128, bf16, 760 MB: 130 us, 5.8 TB/s of the 7.0 that a
// large read reaches; loads of 64 bytes of a row 200, by plain loads 150; 16 of 20000 to 32768 in e4m3, 852 MB: 146 us, 5.85 TB/s).
// The next tile's keys are asked for when this one's are in LDS, its values likewise, the page numbers of the one after it too.
// A cache in 4 bits is a quarter of the bytes for the same products, and there the waves' own work bounds a tile: codes to LDS, four
// conversions to eight keys' elements, products, maximum, powers, values widened to LDS, products (64 sequences of 30 to 16384 keys, 8 key
// heads of 128, 203 MB: 57.8 us, 3.5 TB/s; 51 with all pages one and the same, the vector unit busy for half of that, 57 with two
// blocks to a unit instead of three, 121 with four, which spill; keys widened on the way to LDS instead of behind it 62.7).  The matrix unit's
// own products with 4-bit numbers and their scales were tried with the queries as three rows of e4m3: it drops what is below 2^-12 of
// the largest term, so logarithms of sums were off by 1.7e-4.
// The waves' (m, l, O) are joined in LDS; a sequence of one chunk is then done, others leave theirs in the workspace for the
// second kernel.
#include "attention_math.h"

namespace hyle_hip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWaveLanes;
constexpr int kStep = 32, kTile = kWaves * kStep;  // keys of a wave's step and of a block's

// How a sequence's tiles are dealt: `tiles` of them, the first `sinks` of which hold the sinks before `low`, the window's first key
// (rounded down to a wave's step).
struct SplitTiles {
  int low, sinks, tiles;
};
__device__ __forceinline__ SplitTiles tiles_of(const AttentionParams &p, const AttentionSequence &s) {
  const AttentionSpan first = attention_span(p, s.keys, s.first), last = attention_span(p, s.keys, s.first + s.rows - 1);
  SplitTiles t;
  t.low = min(first.low, last.high) / kStep * kStep;
  t.sinks = (min(min(p.sinks, t.low), last.high) + kTile - 1) / kTile;
  t.tiles = t.sinks + (last.high - t.low + kTile - 1) / kTile;
  return t;
}

struct SplitChunk {
  int index, chunk, chunks;  // sequence, which of its chunks, how many it has
  int first_slot, tiles_each;
  int mark;  // the sequence's
};
__device__ __forceinline__ uint32_t scanned(uint32_t v, int lane) {
  uint32_t up;
  up = lane_up<1>(v), v += lane >= 1 ? up : 0u;
  up = lane_up<2>(v), v += lane >= 2 ? up : 0u;
  up = lane_up<4>(v), v += lane >= 4 ? up : 0u;
  up = lane_up<8>(v), v += lane >= 8 ? up : 0u;
  up = lane_up<16>(v), v += lane >= 16 ? up : 0u;
  up = lane_up<32>(v), v += lane >= 32 ? up : 0u;
  return v;
}
// The sequence and chunk that a slot of the grid is; false past the last.  Every wave of a launch comes to the same answer
// from the marks alone.  target, chunks that all tiles are dealt to, is 0 where every sequence is one.  A block of one tile has
// nothing to load while it computes, so a chunk has two at least where the tiles are more than the resident blocks (one sequence
// of 32751 keys, 2 key heads of 256: 24 us with chunks of two tiles, 34 with one, 26 with four).  Tiles of 4 bits are a quarter of the
// bytes, so a block's start and end weigh more, and key heads with pages of their own are many short sequences alike: there up to `least` = four,
// where all chunks are then resident at once.  (us with two at least / up to four.  4 bits, depths 64, 128 and 256, bf16: one of 131055 keys 34.1 / 30.5,
// 45.1 / 45.1, 50.5 / 37.5; 16 of 4000, 4 new tokens each 23.9 / 18.9, 36.4 / 32.5, 39.5 / 31.3; 8 of 3000 12.4 / 12.5, 14.5 / 14.7, 19.0 / 19.1; 64 ragged
// ones 38.9 / 40.1, 57.8 / 57.7, 59.3 / 55.0; f16 alike.  128 key heads of 2048 keys of their own: bf16 17.8 / 17.8, 33.1 / 30.6, 66.2 / 62.1, e4m3
// 15.6 / 15.6, 25.0 / 21.7, 40.3 / 35.6, 4 bits 14.6 / 14.7, 20.9 / 17.5, 44.5 / 35.2; 32 of them or fewer the same within 3 %.)
// Every wave goes through all marks for its answer: little of a block's time for 64 sequences and a multiple of it for thousands, which pages of
// key heads come to sooner (640 keys, 8 key heads of 128, bf16, pages of the sequences / of each key head: 64 sequences 39 / 58, 256 117 / 235,
// 1024 523 / 1770; 2048 keys, 16 30 / 32, 64 92 / 107).
__device__ __forceinline__ bool chunk_of(const AttentionParams &p, const int32_t *marks, int slot, int target, int blocks, int least, SplitChunk *c) {
  const int lane = (int)threadIdx.x % kWaveLanes;
  if (target == 0) {
    if (slot >= p.sequences) return false;
    *c = SplitChunk{slot, 0, 1, slot, 1 << 24, __builtin_amdgcn_readfirstlane(attention_mark(p, marks, slot))};
    return true;
  }
  // ceil(all / blocks) within 1 .. least, by comparisons: a second division of 64 bits is 0.2 us of every block
  auto at_least = [&](uint64_t all) {
    int tiles = 1;
    for (int i = 1; i < least; ++i) tiles += all > (uint64_t)i * (uint32_t)blocks;
    return tiles;
  };
  if (p.sequences == 1) {
    const int mark = __builtin_amdgcn_readfirstlane(attention_mark(p, marks, 0)), tiles = tiles_of(p, attention_sequence_of(p, 0, mark)).tiles;
    const int each = max((int)(((uint32_t)tiles + (uint32_t)target - 1) / (uint32_t)target), at_least((uint32_t)tiles));
    *c = SplitChunk{0, slot, max(1, (tiles + each - 1) / each), 0, each, mark};
    return slot < c->chunks;
  }
  auto tiles_at = [&](int index, int mark) { return index < p.sequences ? (uint32_t)tiles_of(p, attention_sequence_of(p, index, mark)).tiles : 0u; };
  const int first_mark = attention_mark(p, marks, min(lane, p.sequences - 1));
  const uint32_t first = tiles_at(lane, first_mark);  // (64 sequences of 2^24 tiles at most fit 32 bits)
  uint64_t total = (uint32_t)__builtin_amdgcn_readlane((int)scanned(first, lane), kWaveLanes - 1);
  for (int base = kWaveLanes; base < p.sequences; base += kWaveLanes) {
    const int index = base + lane;
    total += (uint32_t)__builtin_amdgcn_readlane((int)scanned(tiles_at(index, attention_mark(p, marks, min(index, p.sequences - 1))), lane), kWaveLanes - 1);
  }
  // (never more than a sequence can have)
  const int each = (int)min(max((total + (uint32_t)target - 1) / (uint32_t)target, (uint64_t)at_least(total)), (uint64_t)1 << 24);
  int before = 0;
  for (int base = 0; base < p.sequences; base += kWaveLanes) {
    const int index = base + lane, mark = base == 0 ? first_mark : attention_mark(p, marks, min(index, p.sequences - 1));
    const uint32_t tiles = base == 0 ? first : tiles_at(index, mark);
    const uint32_t mine = index < p.sequences ? max(1u, (tiles + (uint32_t)each - 1) / (uint32_t)each) : 0u;
    const uint32_t through = scanned(mine, lane);
    const uint64_t holds = __ballot(slot < before + (int)through);
    if (holds != 0) {
      const int at = __builtin_ctzll(holds);
      c->index = base + at;
      c->chunks = __builtin_amdgcn_readlane((int)mine, at);
      c->first_slot = before + __builtin_amdgcn_readlane((int)through, at) - c->chunks;
      c->chunk = slot - c->first_slot;
      c->tiles_each = each;
      c->mark = __builtin_amdgcn_readlane(mark, at);
      return true;
    }
    before += __builtin_amdgcn_readlane((int)through, kWaveLanes - 1);
  }
  return false;
}

template <class T> __device__ __forceinline__ f32x4 product16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, BF16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 4 e4m3 values as two words of T: exact.
template <class T> __device__ __forceinline__ uint2 widened(uint32_t w) {
  uint2 out;
  if constexpr (std::is_same<T, BF16>::value) {
    out.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    out.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
  } else {
    out.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    out.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  }
  return out;
}
template <class T> __device__ __forceinline__ void widened(u32x4 w, u32x4 *low, u32x4 *high) {
  const uint2 a = widened<T>(w.x), b = widened<T>(w.y), c = widened<T>(w.z), d = widened<T>(w.w);
  *low = u32x4{a.x, a.y, b.x, b.y};
  *high = u32x4{c.x, c.y, d.x, d.y};
}
// Eight values in 4 bits as four words of T by their scale: exact, but for f16's range.
template <class T> __device__ __forceinline__ u32x4 widened4(uint32_t w, float scale) {
  u32x4 out;
  if constexpr (std::is_same<T, BF16>::value) {
    out.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    out.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    out.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    out.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  } else {
    out.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
    out.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
    out.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
    out.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
  }
  return out;
}
__device__ __forceinline__ float rows_max(float v) {  // over the lanes of one column: 16 apart
  const auto a = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
  v = fmaxf(bits_f32(a[0]), bits_f32(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return fmaxf(bits_f32(b[0]), bits_f32(b[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
  v = bits_f32(a[0]) + bits_f32(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return bits_f32(b[0]) + bits_f32(b[1]);
}

struct SplitLayout {
  int target;     // chunks that all tiles are dealt to, 0: none is split
  int blocks;     // resident at once, of one key head and tile of rows
  int rows;       // query rows of a key head: query heads of it x new tokens, token by token
  Divisor row_tiles, lanes, lines;  // tiles of 16 kRowWaves rows; those of all key heads; rows of all key heads
  float *partial; // [slots, heads, rows, depth]
  float2 *stats;  // [slots, heads, rows]: m, l
  int2 *places;   // [sequences]: first slot, chunks
};

// T: queries and outputs, C: keys and values, kDepth: padded depth (kWhole: the depth itself), kRowWaves: waves of 16 rows each that share a tile's
// keys (1: every wave has all rows and its own keys)
// Blocks of a compute unit: what the registers hold of keys, values, queries and outputs without spilling, and LDS of shared keys.
constexpr int resident(bool narrow, int depth, int row_waves) {
  if (row_waves > 1) return depth <= 64 ? 3 : depth <= 128 ? 2 : 1;
  return depth <= 64 ? 4 : depth <= 128 ? (narrow ? 3 : 2) : narrow ? 2 : 1;
}
template <class T, class C, int kDepth, int kRowWaves, bool kWhole>
__global__ __launch_bounds__(kThreads, resident(!std::is_same<C, T>::value, kDepth, kRowWaves)) void attention_split(AttentionParams p, AttentionBuffers b, SplitLayout layout) {
  constexpr bool kNarrow = std::is_same<C, E4M3>::value, kFour = std::is_same<C, MX4>::value;
  constexpr int kSteps = kDepth / 32, kDims = kDepth / 16;
  constexpr int kLoad = kFour ? 32 : kNarrow ? 16 : 8;   // elements of a 16-byte vector
  constexpr int kVectors = kDepth / kLoad;               // of a row
  constexpr int kLoads = kStep * kVectors / kWaveLanes;  // of a lane, for a step's keys or values
  constexpr int kRow = kDepth * 2 + 32;                  // bytes of a row in LDS: 8 rows of 32 bytes fill the banks
  constexpr int kCodeRow = kDepth / 2 + 16;              // of a row of codes; the step's scales, a word each, stand behind them
  constexpr int kJoinRow = kDepth + 4;                   // floats
  constexpr int kGroups = kWaves / kRowWaves;            // of waves that have keys of their own
  constexpr int kHeld = (kRowWaves == 1 ? 1 : 2) * kWaves * kStep * kRow, kJoined = kWaves * 16 * kJoinRow * 4;
  __shared__ __attribute__((aligned(16))) unsigned char held[kHeld > kJoined ? kHeld : kJoined];
  __shared__ float joined_top[kWaves][16], joined_sum[kWaves][16];
  __shared__ uint32_t shared_alive[kWaves];
  __shared__ int no_number;  // 1 + the tile whose values hold an infinity or NaN

  const int slot = (int)layout.lanes.quotient(blockIdx.x), rest = (int)blockIdx.x - slot * (int)layout.lanes.divisor;
  const int group = (int)layout.row_tiles.quotient((uint32_t)rest), row_tile = rest - group * (int)layout.row_tiles.divisor;
  SplitChunk chunk;
  if (!chunk_of(p, b.marks, slot, layout.target, layout.blocks, kFour || p.apart.divisor != 1 ? 4 : 2, &chunk)) return;
  if (layout.target != 0 && chunk.chunk == 0 && rest == 0 && threadIdx.x == 0) layout.places[chunk.index] = int2{chunk.first_slot, chunk.chunks};
  const AttentionSequence s = attention_sequence_of(p, chunk.index, chunk.mark);
  const SplitTiles tiles = tiles_of(p, s);
  const int begin = chunk.chunk * chunk.tiles_each, end = min(begin + chunk.tiles_each, tiles.tiles);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWaveLanes), lane = (int)threadIdx.x % kWaveLanes;
  const int column = lane % 16, quarter = lane / 16;
  const int row_wave = wave % kRowWaves, key_group = wave / kRowWaves;
  const int first_row = row_tile * 16 * kRowWaves;
  // what some row of the sequence sees, and what this tile of rows does (its first and last tokens)
  const AttentionSpan any{attention_span(p, s.keys, s.first).low, attention_span(p, s.keys, s.first + s.rows - 1).high};
  const AttentionSpan tile_first = attention_span(p, s.keys, s.first + (int)p.shared.quotient((uint32_t)first_row));
  const AttentionSpan tile_last = attention_span(p, s.keys, s.first + (int)p.shared.quotient((uint32_t)min(first_row + 16 * kRowWaves, layout.rows) - 1u));

  // a positive c, so that the maximum of S c is that of S and hidden scores stay -inf: its sign, or a scale of 0, goes into the queries
  const float c = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * kLog2E;

  f32x4 out[kDims];
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < kDims; ++d) out[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const unsigned char *keys = static_cast<const unsigned char *>(b.key) + (int64_t)(group + s.head) * p.k_head;
  const unsigned char *values = static_cast<const unsigned char *>(b.value) + (int64_t)(group + s.head) * p.v_head;
  const bool paged = kFour || p.kind == AttentionKind::kPaged;
  const int32_t *table = paged ? b.table + (int64_t)chunk.index * p.table_row : nullptr;
  auto first_of = [&](int tile) { return tile < tiles.sinks ? tile * kTile : tiles.low + (tile - tiles.sinks) * kTile; };
  auto first_key = [&](int tile) { return first_of(tile) + wave * kStep; };  // of the wave's own keys
  // A lane's key of a step, and the page that holds it; past the last key the last one's place is asked for.
  // (4 bits: the lane's own rows of the loads)
  constexpr int kPlaces = kFour ? kLoads : 1;
  auto row_of = [&](int k) { return kFour ? k * (kWaveLanes / kVectors) + lane / kVectors : lane % kStep; };
  int page[kPlaces];
  // What lies behind the chunk's last tile is asked for too, all of it at one place: a load that is sometimes left out makes every wait for
  // those before it one for all.  It pays where a block has its unit almost to itself and a cache in 4 bits (both kernels, us, without / so.  Depth 256,
  // bf16 and f16: one of 131055 keys 41.6 / 37.5, 70.3 / 61.4; 64 ragged ones 64.8 / 55.0, 94.8 / 81.0; 8 of 3000 18.8 / 19.1, 23.2 / 22.2; 320 key heads of
  // 1024 keys of their own 72.2 / 55.8, 8 of 4096 14.7 / 15.8.  128 and 64, bf16: one of 131055 45.1 / 45.7, 30.5 / 32.5; 64 ragged ones 57.7 / 58.2, 40.1 /
  // 41.9; 8 of 3000 14.7 / 16.1, 12.5 / 14.0).
  constexpr bool kPast = kFour && kDepth == 256;
  auto ask_pages = [&](int tile) {
    if (kPast) tile = min(tile, end - 1);
#pragma unroll
    for (int k = 0; k < kPlaces; ++k) page[k] = paged ? table[p.page.quotient((uint32_t)min(first_key(tile) + row_of(k), any.high - 1))] : 0;
  };
  // One step's keys and values, whole rows side by side: a load's 64 vectors are whole cache lines, which non-temporal loads
  // need.  The next keys are asked for once these are in LDS, and so are the values.
  u32x4 key_words[kLoads], value_words[kLoads];
  uint32_t key_scales[kFour ? kLoads : 1], value_scales[kFour ? kLoads : 1];  // words that hold them
  uint32_t alive = 0;  // bit j: key j of the step is there and some row sees it
  int64_t value_at[kPlaces] = {};
  int scales_at[kPlaces] = {};  // from the codes of a row to its scales
  const int vectors = p.depth / kLoad;  // of a row; zeros past them
  const int vector = lane % kVectors;
  constexpr bool kEvenScales = kWhole && kDepth >= 128;  // a row's scales are whole words
  uint32_t key_shifts[kPlaces], value_shifts[kPlaces];
  auto scale_of = [&](uint32_t word, uint32_t shift) { return (word >> (kEvenScales ? (uint32_t)(vector % 4) * 8 : shift)) & 255u; };
  auto fetch = [&](const unsigned char *from, const int64_t (&places)[kPlaces], u32x4 (&words)[kLoads], uint32_t *scales, uint32_t (&shifts)[kPlaces]) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      if (!kWhole) words[k] = u32x4{0, 0, 0, 0};
      if constexpr (kFour) {
        if (!kWhole) scales[k] = 0, shifts[k] = 0;
        if (kWhole || vector < vectors) {
          words[k] = load16_words(from + places[k], vector);
          // (the word that holds the byte: a byte that is carried round the loop is widened, and so waited for, where it was loaded)
          const unsigned char *byte = from + places[k] + scales_at[k] + vector;
          if (!kEvenScales) shifts[k] = ((uint32_t)reinterpret_cast<uintptr_t>(byte) & 3u) * 8;
          scales[k] = *reinterpret_cast<const uint32_t *>(byte - (kEvenScales ? vector % 4 : (int)(reinterpret_cast<uintptr_t>(byte) & 3u)));
        }
      } else {
        const int row = k * (kWaveLanes / kVectors) + lane / kVectors;
        const int64_t at = ((int64_t)__shfl((int)(places[0] >> 32), row, kWaveLanes) << 32) | (uint32_t)__shfl((int)places[0], row, kWaveLanes);
        if (kWhole || vector < vectors) words[k] = load16_stream(from + at, vector);
      }
    }
  };
  auto fetch_keys = [&](int tile) {
    int64_t key_at[kPlaces];
    uint64_t lanes[kPlaces];  // whose key is there
#pragma unroll
    for (int k = 0; k < kPlaces; ++k) {
      const int key = first_key(tile) + row_of(k), known = !kFour || tile < end ? min(key, any.high - 1) : 0;
      bool there = (key < any.high) & ((key >= any.low) | (key < p.sinks)) & ((tile >= tiles.sinks) | (key < tiles.low)) & (!kFour || tile < end);
      if (paged) {
        there &= (uint32_t)page[k] < (uint32_t)p.pages;
        const uint32_t at = (uint32_t)known - p.page.quotient((uint32_t)known) * p.page.divisor;
        // (a page that is not there is read as the cache's first row, which is there: its keys are not alive)
        key_at[k] = value_at[k] = there ? (int64_t)page[k] * p.k_sequence + (int64_t)at * p.k_row : 0;
        if constexpr (kFour) scales_at[k] = (int)p.scale_offset - (there ? (int)at * ((int)p.k_row / 16 * 15) : 0);
      } else {
        key_at[k] = (int64_t)chunk.index * p.k_sequence + (int64_t)known * p.k_row;
        value_at[k] = (int64_t)chunk.index * p.v_sequence + (int64_t)known * p.v_row;
      }
      lanes[k] = __ballot(there);
    }
    if constexpr (kFour) {
      uint64_t all = lanes[0];
#pragma unroll
      for (int k = 1; k < kPlaces; ++k) all &= lanes[k];
      alive = 0xFFFFFFFFu;
      if (all != ~0ull) {
        alive = 0;
#pragma unroll
        for (int k = 0; k < kPlaces; ++k)
#pragma unroll 1
          for (int r = 0; r < kWaveLanes / kVectors; ++r) alive |= (uint32_t)((lanes[k] >> (r * kVectors)) & 1) << (k * (kWaveLanes / kVectors) + r);
      }
    } else {
      alive = (uint32_t)lanes[0];
    }
    fetch(keys, key_at, key_words, key_scales, key_shifts);
  };
  auto fetch_values = [&]() { fetch(values, value_at, value_words, value_scales, value_shifts); };
  // Rows widened from 4 bits are written by lanes whose pieces begin 64 bytes apart: eights of dims change places (by the turn of 64 dims
  // that they are in, of depth 64 of the row), so that a write's pieces of 16 bytes, and a read's, lie in all banks.
  auto swizzled = [](int row, int eight) { return kFour ? eight ^ (kDepth == 64 ? row / 2 % 2 : eight / 8 % 4) : eight; };
  int put_at[4] = {}, read_at[2] = {};  // where a lane's four pieces go, and where it reads eights of even and odd turns
  if constexpr (kFour) {
#pragma unroll
    for (int w = 0; w < 4; ++w) put_at[w] = lane / kVectors * kRow + 16 * swizzled(lane / kVectors, 4 * vector + w);
    const int row = 4 * quarter + column / 4, eight = column % 4 / 2;  // (16 rows on, the same places)
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) read_at[turn] = row * kRow + 16 * (eight ^ (kDepth == 64 ? row / 2 % 2 : turn)) + column % 2 * 8;
  }
  // a step's vectors to the wave's rows in LDS, e4m3 and 4 bits as the elements of T that they stand for (kClean: numbers alone)
  auto put = [&](unsigned char *base, const u32x4 (&words)[kLoads], const uint32_t *scales, const uint32_t (&shifts)[kPlaces], auto clean) {
    constexpr bool kClean = decltype(clean)::value;
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses are in order)
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int row = k * (kWaveLanes / kVectors) + lane / kVectors;
      unsigned char *to = base + row * kRow + vector * kLoad * 2;
      if constexpr (kFour) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          u32x4 wide = widened4<T>(words[k][w], bits_f32(scale_of(scales[k], shifts[kFour ? k : 0]) << 23));
          if (kClean) wide = numbers_only<T>(wide);
          *reinterpret_cast<u32x4 *>(base + put_at[w] + k * (kWaveLanes / kVectors) * kRow) = wide;
        }
      } else if constexpr (kNarrow) {
        u32x4 low, high;
        widened<T>(words[k], &low, &high);
        *reinterpret_cast<u32x4 *>(to) = low;
        *reinterpret_cast<u32x4 *>(to + 16) = high;
      } else {
        *reinterpret_cast<u32x4 *>(to) = words[k];
      }
    }
    __builtin_amdgcn_wave_barrier();  // other lanes' rows are read next
  };

  // Keys in 4 bits go to LDS as they are and are widened where they are multiplied: a lane then has kDepth / 4 neighbouring dims of its
  // key, and its queries' in the same order.
  auto put_codes = [&](unsigned char *base) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int row = k * (kWaveLanes / kVectors) + lane / kVectors;
      *reinterpret_cast<u32x4 *>(base + row * kCodeRow + vector * 16) = key_words[k];
      *reinterpret_cast<uint32_t *>(base + kStep * kCodeRow + (row * kVectors + vector) * 4) = scale_of(key_scales[k], key_shifts[k]) << 23;
    }
    __builtin_amdgcn_wave_barrier();
  };
  auto dims_of = [&](int k) { return kFour ? quarter * kSteps + k : 4 * k + quarter; };  // of a product, in eights
  auto key_rows = [&](int part) { return held + part * kStep * kRow; };
  auto value_rows = [&](int part) { return held + ((kRowWaves == 1 ? 0 : kWaves) + part) * kStep * kRow; };
  if (begin < end) ask_pages(begin);
  // queries: a lane's row is its column, its dims 8 quarter on of every 32 (with keys in 4 bits, a quarter of all in a row)
  u32x4 query[kSteps];
  AttentionSpan span;
  {
    const int row = first_row + 16 * row_wave + column, known = min(row, layout.rows - 1), token = (int)p.shared.quotient((uint32_t)known);
    const unsigned char *from = attention_query(p, b, s, token, (group + s.head) * (int)p.shared.divisor + known - token * (int)p.shared.divisor);
    span = attention_span(p, s.keys, s.first + token);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      query[k] = u32x4{0, 0, 0, 0};
      if (row < layout.rows && (kWhole || dims_of(k) * 8 < p.depth)) query[k] = load16(from, dims_of(k));
    }
  }
  if (kRowWaves > 1 && threadIdx.x == 0) no_number = 0;
  if (begin < end) {
    fetch_keys(begin);
    if constexpr (kFour) {
      __builtin_amdgcn_sched_barrier(0);  // (in the loop's order: its waits count what was asked for since)
      ask_pages(begin + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    fetch_values();
    if (!kFour && begin + 1 < end) ask_pages(begin + 1);
    if constexpr (kFour) __builtin_amdgcn_sched_barrier(0);
  }
  if (p.scale <= 0.0f) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) query[k] = p.scale == 0.0f ? u32x4{0, 0, 0, 0} : query[k] ^ 0x80008000u;
  }
  if (kRowWaves > 1) __syncthreads();  // no_number is cleared
  // every row of the block sees every key from `first` on
  auto seen_whole = [&](int first) { return first + kStep <= tile_first.high && first >= tile_last.low; };
  // keys that are not alive bring zeros
  auto clear_dead = [&](uint32_t these) {
    if (these == 0xFFFFFFFFu) return;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int row = k * (kWaveLanes / kVectors) + lane / kVectors;
      if (((these >> row) & 1u) == 0) {
        value_words[k] = u32x4{0, 0, 0, 0};
        if constexpr (kFour) value_scales[k] = 0;
      }
    }
  };
  // Values that are no numbers, of keys that not every row sees: a weight of 0 would make NaN of them in the product.  They are
  // added to the rows that see them (a finite weight changes nothing about them) and zeroed.
  auto add_no_numbers = [&](const unsigned char *from, uint32_t these, int first) {
#pragma unroll 1
    for (int j = 0; j < kStep; ++j) {
      if (((these >> j) & 1u) == 0) continue;
      const bool sees = attention_sees(p, span, first + j);
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = Traits<T>::load(from + j * kRow, 8 * swizzled(j, 2 * d + quarter / 2) + quarter % 2 * 4 + r);
          v[r] = fabsf(x) < INFINITY ? 0.0f : x;
        }
        if (sees) out[d] += f32x4{v[0], v[1], v[2], v[3]};
        asm volatile("" : : : "memory");  // (a dim at a time: all at once would cost every step its registers)
      }
    }
  };
  auto any_no_number = [&]() {
    uint32_t found = 0;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      // (of 4 bits by the scale: from which on 6 of it, or 4, may pass T's range, and NaN)
      if constexpr (kFour) found |= (uint32_t)(scale_of(value_scales[k], value_shifts[k]) >= (std::is_same<T, BF16>::value ? 253u : 141u));
      else found |= no_numbers<C>(value_words[k]);
    }
    return __ballot(found != 0) != 0;
  };
  auto keep_numbers = [&]() {  // (4 bits are cleaned on the way to LDS)
    if constexpr (!kFour) {
#pragma unroll
      for (int k = 0; k < kLoads; ++k) value_words[k] = numbers_only<C>(value_words[k]);
    }
  };
  constexpr std::false_type kAsRead{};
  constexpr std::true_type kNumbers{};

  for (int tile = begin; tile < end; ++tile) {
    const uint32_t own = alive;
    if constexpr (kFour) put_codes(key_rows(wave));
    else put(key_rows(wave), key_words, key_scales, key_shifts, kAsRead);
    if constexpr (kRowWaves == 1) {
      __builtin_amdgcn_sched_barrier(0);  // (loads that move up further need registers of their own)
      if (kPast || tile + 1 < end) {
        fetch_keys(tile + 1);
        if (kPast || tile + 2 < end) ask_pages(tile + 2);
      }
    } else {
      clear_dead(own);
      if (lane == 0) shared_alive[wave] = own;
      const bool odd = s.rows > 1 && !(own == 0xFFFFFFFFu && seen_whole(first_key(tile))) && any_no_number();
      if (odd && lane == 0) no_number = tile + 1;
      put(value_rows(wave), value_words, value_scales, value_shifts, kAsRead);
      __syncthreads();
      if (no_number == tile + 1) {
#pragma unroll 1
        for (int sub = 0; sub < kRowWaves; ++sub) {
          const int part = key_group * kRowWaves + sub;
          add_no_numbers(value_rows(part), shared_alive[part], first_of(tile) + part * kStep);
        }
        __syncthreads();
        keep_numbers();
        put(value_rows(wave), value_words, value_scales, value_shifts, kNumbers);
        __syncthreads();
      }
      __builtin_amdgcn_sched_barrier(0);
      if (tile + 1 < end) {
        fetch_keys(tile + 1);
        if (tile + 2 < end) ask_pages(tile + 2);
        fetch_values();
      }
    }
#pragma unroll 1
    for (int sub = 0; sub < kRowWaves; ++sub) {
      const int part = kRowWaves == 1 ? wave : key_group * kRowWaves + sub, first = first_of(tile) + part * kStep;
      const uint32_t these = kRowWaves == 1 ? own : (uint32_t)__builtin_amdgcn_readfirstlane((int)shared_alive[part]);
      const bool whole = these == 0xFFFFFFFFu && seen_whole(first);
      f32x4 score[2];
      const unsigned char *from = key_rows(part);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        score[half] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (kFour) {
          const unsigned char *codes = from + (16 * half + column) * kCodeRow + quarter * (kSteps * 4);
          const unsigned char *scales = from + kStep * kCodeRow + (16 * half + column) * kVectors * 4 + quarter * kSteps / 4 * 4;
          uint32_t words[kSteps];
          if constexpr (kSteps == 2) {
            const uint2 w = *reinterpret_cast<const uint2 *>(codes);
            words[0] = w.x, words[1] = w.y;
          } else {
#pragma unroll
            for (int v = 0; v < kSteps / 4; ++v) {
              const u32x4 w = reinterpret_cast<const u32x4 *>(codes)[v];
              words[4 * v] = w.x, words[4 * v + 1] = w.y, words[4 * v + 2] = w.z, words[4 * v + 3] = w.w;
            }
          }
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
            score[half] = product16<T>(widened4<T>(words[k], reinterpret_cast<const float *>(scales)[k / 4]), query[k], score[half]);
        } else {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(from + (16 * half + column) * kRow + (4 * k + quarter) * 16);
            score[half] = product16<T>(w, query[k], score[half]);
          }
        }
      }
      if (!whole) {
        asm volatile("" : : : "memory");  // (a branch: as selects, the comparisons are every step's)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * half + 4 * quarter + r;
            if (((these >> j) & 1u) == 0 || !attention_sees(p, span, first + j)) score[half][r] = -INFINITY;
          }
      }
      const float most = rows_max(fmaxf(fmaxf(fmaxf(score[0][0], score[0][1]), fmaxf(score[0][2], score[0][3])),
                                        fmaxf(fmaxf(score[1][0], score[1][1]), fmaxf(score[1][2], score[1][3])))) *
                         c;
      if (__ballot(most > top + kSlack) != 0) {
        const float next = fmaxf(top, most);
        const float keep = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - next);  // (what there is without a maximum is zeros and what is no number)
        top = next;
        sum *= keep;
#pragma unroll
        for (int d = 0; d < kDims; ++d) out[d] *= keep;
      }
      u32x4 weights;
      const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          score[half][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[half][r], c, -shift));
          sum += score[half][r];
        }
        weights[2 * half] = pack2<T>(score[half][0], score[half][1]);
        weights[2 * half + 1] = pack2<T>(score[half][2], score[half][3]);
      }
      if constexpr (kRowWaves == 1) {
        clear_dead(these);
        const bool odd = !whole && s.rows > 1 && any_no_number();
        if (odd) {
          put(value_rows(wave), value_words, value_scales, value_shifts, kAsRead);
          add_no_numbers(value_rows(wave), these, first);
          keep_numbers();
        }
        put(value_rows(wave), value_words, value_scales, value_shifts, kAsRead);
        if (kFour && odd) put(value_rows(wave), value_words, value_scales, value_shifts, kNumbers);
        __builtin_amdgcn_sched_barrier(0);
        if (kPast || tile + 1 < end) fetch_values();
        if constexpr (kFour) __builtin_amdgcn_sched_barrier(0);
      }
      from = value_rows(part);
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        const unsigned char *at = kFour ? from + read_at[kDepth == 64 ? 0 : d / 4 % 2] + 32 * (d ^ (kDepth == 64 ? 0 : d / 8 % 2))
                                        : from + (4 * quarter + column / 4) * kRow + (d * 16 + column % 4 * 4) * 2;
        const uint2 near = read_transposed(at), far = read_transposed(at + 16 * kRow);
        const u32x4 value = {near.x, near.y, far.x, far.y};
        out[d] = product16<T>(value, weights, out[d]);
      }
    }
    if (kRowWaves > 1) __syncthreads();  // the rows in LDS are read
  }

  // join the waves of the same rows
  float *joined = reinterpret_cast<float *>(held);
  constexpr int kRowThreads = 16 / kRowWaves;  // threads of a row
  const int join_row = (int)threadIdx.x / kRowThreads, join_wave = join_row / 16, join_column = join_row % 16;
  __syncthreads();
  const float total = rows_sum(sum);
  if (quarter == 0) joined_top[wave][column] = top, joined_sum[wave][column] = total;
#pragma unroll
  for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4 *>(joined + (wave * 16 + column) * kJoinRow + d * 16 + 4 * quarter) = out[d];
  __syncthreads();
  const int row = first_row + join_row;
  if (row >= layout.rows) return;
  float most = joined_top[join_wave][join_column];
#pragma unroll
  for (int g = 1; g < kGroups; ++g) most = fmaxf(most, joined_top[g * kRowWaves + join_wave][join_column]);
  const float shift = most == -INFINITY ? 0.0f : most;
  float keep[kGroups], all = 0.0f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    keep[g] = __builtin_amdgcn_exp2f(joined_top[g * kRowWaves + join_wave][join_column] - shift);
    all += joined_sum[g * kRowWaves + join_wave][join_column] * keep[g];
  }
  const int token = (int)p.shared.quotient((uint32_t)row);
  const int64_t at = (s.row + token) * p.queries + (group + s.head) * (int)p.shared.divisor + row - token * (int)p.shared.divisor;
  const int64_t part = ((int64_t)slot * p.heads + group) * layout.rows + row;
  const float inverse = all == 0.0f ? 0.0f : 1.0f / all;
  for (int d = (int)threadIdx.x % kRowThreads * 4; d < p.depth; d += kRowThreads * 4) {
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) o += *reinterpret_cast<const f32x4 *>(joined + ((g * kRowWaves + join_wave) * 16 + join_column) * kJoinRow + d) * keep[g];
    if (chunk.chunks == 1) {
      uint2 w;
      w.x = pack2<T>(o[0] * inverse, o[1] * inverse);
      w.y = pack2<T>(o[2] * inverse, o[3] * inverse);
      *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(b.out) + (at * p.depth + d) * 2) = w;
    } else {
      *reinterpret_cast<f32x4 *>(layout.partial + part * p.depth + d) = o;
    }
  }
  if (threadIdx.x % kRowThreads == 0) {
    if (chunk.chunks != 1) layout.stats[part] = float2{most, all};
    else if (b.logs != nullptr) b.logs[at] = all == 0.0f ? -INFINITY : (most + __builtin_amdgcn_logf(all)) * kLn2;
  }
}

// The chunks of a query row joined, four dims to a thread.  kSide: kParts chunks side by side, a row to a block, for few rows of
// many chunks; otherwise a row to kLanes threads.
constexpr int join_threads(int depth, bool side) { return side && depth == 256 ? 512 : 256; }
template <class T, int kDepth, bool kSide>
__global__ __launch_bounds__(join_threads(kDepth, kSide)) void attention_join(AttentionParams p, AttentionBuffers b, SplitLayout layout) {
  constexpr int kLanes = kDepth / 4, kParts = kSide ? join_threads(kDepth, kSide) / kLanes : 1, kRows = kSide ? 1 : join_threads(kDepth, kSide) / kLanes;
  const uint32_t line = blockIdx.x * kRows + (kSide ? 0u : threadIdx.x / kLanes);
  const int index = (int)layout.lines.quotient(line), rest = (int)line - index * (int)layout.lines.divisor;  // key head and row
  if (!kSide && index >= p.sequences) return;
  const int2 place = layout.places[index];
  if (place.y == 1) return;  // the split kernel's block was the whole sequence
  const int64_t stride = (int64_t)p.heads * layout.rows, first = (int64_t)place.x * stride + rest;
  const int lane = (int)threadIdx.x % (kSide ? kWaveLanes : kLanes);
  float most = -INFINITY;  // every wave, or row, looks at all chunks' maxima
  for (int i = lane; i < place.y; i += kSide ? kWaveLanes : kLanes) most = fmaxf(most, layout.stats[first + i * stride].x);
  most = group_max<kSide ? kWaveLanes : kLanes>(most);
  const float shift = most == -INFINITY ? 0.0f : most;
  const int dim = (int)threadIdx.x % kLanes * 4, part = kSide ? (int)threadIdx.x / kLanes : 0;
  f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f;
  const bool has = dim < p.depth;
#pragma unroll 8
  for (int i = part; i < place.y; i += kParts) {
    const float2 stat = layout.stats[first + i * stride];
    const f32x4 o = *reinterpret_cast<const f32x4 *>(layout.partial + (first + i * stride) * p.depth + (has ? dim : 0));
    const float keep = __builtin_amdgcn_exp2f(stat.x - shift);
    sum = __builtin_fmaf(stat.y, keep, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = __builtin_fmaf(o[e], keep, out[e]);
  }
  if constexpr (kSide) {
    __shared__ __attribute__((aligned(16))) f32x4 joined[kParts][kLanes];
    __shared__ float sums[kParts];
    joined[part][dim / 4] = out;
    if (dim == 0) sums[part] = sum;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int i = 1; i < kParts; ++i) out += joined[i][dim / 4], sum += sums[i];
  }
  const int group = rest / layout.rows, row = rest - group * layout.rows, token = (int)p.shared.quotient((uint32_t)row);
  const int batch = (int)p.apart.quotient((uint32_t)index), head = group + index - batch * (int)p.apart.divisor;
  const int64_t at = ((int64_t)batch * p.rows + token) * p.queries + head * (int)p.shared.divisor + row - token * (int)p.shared.divisor;
  if (has) {
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint2 w;
    w.x = pack2<T>(out[0] * inverse, out[1] * inverse);
    w.y = pack2<T>(out[2] * inverse, out[3] * inverse);
    *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(b.out) + (at * p.depth + dim) * 2) = w;
  }
  if (b.logs != nullptr && dim == 0) b.logs[at] = sum == 0.0f ? -INFINITY : (most + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace

template <class C, int kDepth, int kRowWaves, bool kWhole> struct AttentionSplitTag {
  static std::string text() {
    return std::string("attention_split/") + (std::is_same<C, E4M3>::value ? "e4m3/" : std::is_same<C, MX4>::value ? "mx4/" : "") + (kWhole ? "d" : "below-d") + std::to_string(kDepth) + "/" + std::to_string(16 * kRowWaves) + "-rows";
  }
};
template <int kDepth, bool kSide> struct AttentionJoinTag {
  static std::string text() { return "attention_join/d" + std::to_string(kDepth) + (kSide ? "/row-to-block" : "/rows"); }
};

namespace {
int padded_depth(const AttentionParams &p) { return p.depth <= 64 ? 64 : p.depth <= 128 ? 128 : 256; }
int row_waves_of(const AttentionParams &p) {
  const int64_t rows = (int64_t)p.rows * p.shared.divisor;
  return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}
int row_tiles_of(const AttentionParams &p) {
  const int64_t each = 16 * row_waves_of(p);
  return (int)(((int64_t)p.rows * p.shared.divisor + each - 1) / each);
}
}  // namespace

// Sequences of so few tiles are not split: a tile takes a block about 1 us, the second kernel 4.  (us, 512 keys unsplit / split, sequences
// x key heads, depth 64: 4 x 8 7.7 / 8.7, 128 x 8 17.8 / 27.5; 128: 4 x 8 10.3 / 9.9, 32 x 8 11.7 / 14.9, 128 x 8 39.7 / 61; 256: 4 x 8 20.5 / 14.4,
// 32 x 8 22.1 / 36.2, 128 x 8 95 / 105; 800 keys, depth 128: 4 x 8 15 / 10.9, 32 x 8 17.5 / 25.9.  So few sequences of depth 256 would
// rather be split, and longer ones of a full device not.)
constexpr int kUnsplit = 4;

AttentionSplit attention_split_of(const AttentionParams &p, int compute_units) {
  AttentionSplit split;
  // The chunks of one key head and tile of rows: three rounds of the blocks that the device holds, so that the last ones of
  // ragged sequences leave it idle for a third of a block (us with a half, one, two, three and four rounds: 64 ragged sequences 158,
  // 140, 134, 130, 130; 16 long ones in e4m3 151, 178, 157, 146, 148).
  const int64_t lanes = (int64_t)p.heads * row_tiles_of(p);
  const int64_t blocks = (int64_t)compute_units * resident(p.narrow_cache || p.four_bits, padded_depth(p), row_waves_of(p));
  const int64_t target = (3 * blocks + lanes - 1) / lanes;
  split.blocks = (int)((blocks + lanes - 1) / lanes);
  // tiles of a sequence: of all its keys, or of the window of its new tokens and the sinks
  int64_t most = ((int64_t)p.keys + kTile - 1) / kTile;
  if (p.window != 0) {
    const int64_t seen = ((int64_t)p.window + p.rows + kStep + kTile - 1) / kTile + ((int64_t)p.sinks + kTile - 1) / kTile;
    if (seen < most) most = seen;
  }
  split.target = (int)target;
  // The sum over the sequences of ceil(tiles / each), at least one for each of them, where each is at least total / target and,
  // with more tiles than blocks, 2.  (Sinks and a window that begins between two tiles can be one tile more than all keys, `most` + 1:
  // half of that, rounded up, is within `most` / 2 and the sequence's own one.)
  int64_t slots = most * p.sequences / 2 > split.blocks ? most * p.sequences / 2 : split.blocks;
  if (target < slots) slots = target;
  slots += p.sequences;
  split.slots = (int)slots;
  split.joined = most > kUnsplit && target > 1;
  if (!split.joined) split.target = 0, split.slots = p.sequences;
  const uint64_t lines = (uint64_t)p.rows * p.shared.divisor * (uint64_t)p.heads * (uint64_t)p.sequences;
  split.launches = axis_holds((uint64_t)split.slots * (uint64_t)lanes, kThreads) &&
                   (!split.joined || axis_holds(lines * (uint64_t)(padded_depth(p) / 4) + join_threads(padded_depth(p), false), 1));
  const int64_t rows = (int64_t)p.rows * p.shared.divisor * p.heads * split.slots;
  split.stats_offset = ((size_t)rows * (size_t)p.depth * sizeof(float) + 255) / 256 * 256;
  split.places_offset = split.stats_offset + ((size_t)rows * sizeof(float2) + 255) / 256 * 256;
  split.workspace = split.joined ? split.places_offset + (size_t)p.sequences * sizeof(int2) : 0;
  return split;
}

// (vectors of codes are read at addresses of whole words)
bool attention_split_serves(Elem type, const AttentionParams &p, bool vector_aligned) {
  if (type == Elem::kF32 || p.kind == AttentionKind::kPacked || !vector_aligned || p.depth % (p.four_bits ? 32 : p.narrow_cache ? 16 : 8) != 0) return false;
  if (p.four_bits) return ((p.q_sequence | p.q_row | p.q_head) % 16 | (p.k_sequence | p.k_head | p.value_offset) % 4) == 0 && p.scale_offset <= INT32_MAX / 2;
  return ((p.q_sequence | p.q_row | p.q_head | p.k_sequence | p.k_row | p.k_head | p.v_sequence | p.v_row | p.v_head) % 16) == 0;
}

namespace {
template <class T, class C, int kDepth, int kRowWaves>
void start_split(const AttentionParams &p, const AttentionBuffers &b, const SplitLayout &layout, const AttentionSplit &split, hipStream_t stream) {
  const dim3 grid((uint32_t)split.slots * layout.lanes.divisor), block(kThreads);
  if (p.depth == kDepth) {
    note_variant<AttentionSplitTag<C, kDepth, kRowWaves, true>>();
    hipLaunchKernelGGL((attention_split<T, C, kDepth, kRowWaves, true>), grid, block, 0, stream, p, b, layout);
  } else {
    note_variant<AttentionSplitTag<C, kDepth, kRowWaves, false>>();
    hipLaunchKernelGGL((attention_split<T, C, kDepth, kRowWaves, false>), grid, block, 0, stream, p, b, layout);
  }
  if (!split.joined) return;
  // Chunks side by side where rows are few (us of both kernels, side by side / a row to few threads, depth 64: 1024 rows of 16000 keys
  // 31.1 / 48.3, 512 of 4000 26.1 / 28.8, 2048 of 4000 76.6 / 75.5, 4096 of 700 41.4 / 37.8; depth 256: 1024 of 16000 115 / 118, 2048 of 700
  // 93 / 89, 4096 of 700 54.6 / 48.2).
  const uint32_t lines = layout.lines.divisor * (uint32_t)p.sequences;
  if (lines <= 2048) {
    note_variant<AttentionJoinTag<kDepth, true>>();
    hipLaunchKernelGGL((attention_join<T, kDepth, true>), dim3(lines), dim3(join_threads(kDepth, true)), 0, stream, p, b, layout);
  } else {
    constexpr uint32_t kRows = join_threads(kDepth, false) / (kDepth / 4);
    note_variant<AttentionJoinTag<kDepth, false>>();
    hipLaunchKernelGGL((attention_join<T, kDepth, false>), dim3((lines + kRows - 1) / kRows), dim3(join_threads(kDepth, false)), 0, stream, p, b, layout);
  }
}
template <class T, class C, int kDepth>
void split_by_rows(const AttentionParams &p, const AttentionBuffers &b, const SplitLayout &layout, const AttentionSplit &split, hipStream_t stream) {
  switch (row_waves_of(p)) {
    case 1: start_split<T, C, kDepth, 1>(p, b, layout, split, stream); break;
    case 2: start_split<T, C, kDepth, 2>(p, b, layout, split, stream); break;
    default: start_split<T, C, kDepth, 4>(p, b, layout, split, stream);
  }
}
template <class T, class C>
void split_by_depth(const AttentionParams &p, const AttentionBuffers &b, const SplitLayout &layout, const AttentionSplit &split, hipStream_t stream) {
  switch (padded_depth(p)) {
    case 64: split_by_rows<T, C, 64>(p, b, layout, split, stream); break;
    case 128: split_by_rows<T, C, 128>(p, b, layout, split, stream); break;
    default: split_by_rows<T, C, 256>(p, b, layout, split, stream);
  }
}
}  // namespace

hipError_t launch_attention_split(Elem type, const AttentionParams &p, const AttentionBuffers &b, const AttentionSplit &split, void *workspace,
                                  hipStream_t stream) {
  SplitLayout layout;
  layout.target = split.target;
  layout.blocks = split.blocks;
  layout.rows = p.rows * (int)p.shared.divisor;
  layout.row_tiles = Divisor((uint32_t)row_tiles_of(p));
  layout.lanes = Divisor((uint32_t)(p.heads * row_tiles_of(p)));
  layout.lines = Divisor((uint32_t)(p.heads * layout.rows));
  layout.partial = static_cast<float *>(workspace);
  layout.stats = reinterpret_cast<float2 *>(static_cast<unsigned char *>(workspace) + split.stats_offset);
  layout.places = reinterpret_cast<int2 *>(static_cast<unsigned char *>(workspace) + split.places_offset);
  if (type == Elem::kF16) {
    if (p.four_bits) split_by_depth<F16, MX4>(p, b, layout, split, stream);
    else if (p.narrow_cache) split_by_depth<F16, E4M3>(p, b, layout, split, stream);
    else split_by_depth<F16, F16>(p, b, layout, split, stream);
  } else {
    if (p.four_bits) split_by_depth<BF16, MX4>(p, b, layout, split, stream);
    else if (p.narrow_cache) split_by_depth<BF16, E4M3>(p, b, layout, split, stream);
    else split_by_depth<BF16, BF16>(p, b, layout, split, stream);
  }
  return hipGetLastError();
}

}  // namespace hyle_hip
