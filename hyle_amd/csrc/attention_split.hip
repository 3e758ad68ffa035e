// attention_split.hip -- attention of a few query rows over many keys, split over the keys and joined: f16 / bf16 queries,
// keys and values of their type or e4m3, in memory or in a paged cache.
//
// Bound by the bytes of keys and values, which are read once for all rows of a key head (its query heads times the new
// tokens).  The keys of all sequences, in tiles of 128, are dealt to about as many chunks as the device holds blocks, however
// long each sequence is: a chunk is ceil(tiles / chunks) tiles of one sequence.  A block takes one chunk of one key head; its
// four waves each take 32 keys of every tile and do not meet before the end:
//   S^T[key, row] = K Q^T        (A: rows of K straight from memory, B: the queries)
//   p = 2^(S^T c - m), O^T[dim, row] = V^T P^T   (A: columns of V by transposing reads of the wave's own LDS rows)
// with the running maximum m and sum l of the softmax per lane (a lane's row is its column).  The next step's keys and values
// are loaded while one is computed, the page numbers of the one after it too.  The waves' (m, l, O) are joined in LDS; a
// sequence of one chunk is then done, others leave theirs in the workspace for the second kernel.
#include "attention_math.h"

namespace hyle_hip {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWaveLanes;
constexpr int kStep = 32, kTile = kWaves * kStep;  // keys of a wave's step and of a block's

// How a sequence's tiles are dealt: `tiles` of them, the first `sinks` of which hold the sinks before the window's first key
// `low` (rounded down to a tile).
struct SplitTiles {
  int low, sinks, tiles;
};
__device__ __forceinline__ SplitTiles tiles_of(const AttentionParams &p, const AttentionSequence &s) {
  const AttentionSpan first = attention_span(p, s.keys, s.first), last = attention_span(p, s.keys, s.first + s.rows - 1);
  SplitTiles t;
  t.low = min(first.low, last.high) / kTile * kTile;
  t.sinks = (min(min(p.sinks, t.low), last.high) + kTile - 1) / kTile;
  t.tiles = t.sinks + (last.high - t.low + kTile - 1) / kTile;
  return t;
}

// The sequence and chunk of a slot.  Every wave of a launch comes to the same answer from the marks alone.
struct SplitChunk {
  int index, chunk, chunks;  // sequence, which of its chunks, how many it has
  int first_slot, tiles_each;
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
__device__ __forceinline__ int tiles_each(const AttentionParams &p, const int32_t *marks, int target) {
  const int lane = (int)threadIdx.x % kWaveLanes;
  uint64_t total = 0;
  for (int base = 0; base < p.sequences; base += kWaveLanes) {
    uint32_t mine = 0;
    if (base + lane < p.sequences) mine = (uint32_t)tiles_of(p, attention_sequence(p, marks, base + lane)).tiles;
    total += (uint32_t)__builtin_amdgcn_readlane((int)scanned(mine, lane), kWaveLanes - 1);  // (64 sequences of 2^24 tiles at most)
  }
  const uint64_t each = (total + (uint32_t)target - 1) / (uint32_t)target;
  return (int)(each < 1 ? 1 : each);
}
__device__ __forceinline__ bool chunk_of(const AttentionParams &p, const int32_t *marks, int slot, int each, SplitChunk *c) {
  const int lane = (int)threadIdx.x % kWaveLanes;
  int before = 0;
  for (int base = 0; base < p.sequences; base += kWaveLanes) {
    uint32_t mine = 0;
    if (base + lane < p.sequences) mine = (uint32_t)max(1, (tiles_of(p, attention_sequence(p, marks, base + lane)).tiles + each - 1) / each);
    const uint32_t through = scanned(mine, lane);
    const uint64_t holds = __ballot(slot < before + (int)through);
    if (holds != 0) {
      const int at = __builtin_ctzll(holds);
      c->index = base + at;
      c->chunks = __builtin_amdgcn_readlane((int)mine, at);
      c->first_slot = before + __builtin_amdgcn_readlane((int)through, at) - c->chunks;
      c->chunk = slot - c->first_slot;
      c->tiles_each = each;
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
  int target;     // chunks that all tiles are dealt to
  int rows;       // query rows of a key head: query heads of it x new tokens, token by token
  int row_tiles;  // of 16 kBlocks
  float *partial; // [slots, heads, rows, depth]
  float2 *stats;  // [slots, heads, rows]: m, l
};

// T: queries and outputs, C: keys and values, kDepth: padded depth, kBlocks: blocks of 16 rows
template <class T, class C, int kDepth, int kBlocks>
__global__ __launch_bounds__(kThreads) void attention_split(AttentionParams p, AttentionBuffers b, SplitLayout layout) {
  constexpr bool kNarrow = std::is_same<C, E4M3>::value;
  constexpr int kSteps = kDepth / 32, kDims = kDepth / 16;
  constexpr int kLoad = kNarrow ? 16 : 8;                // elements of a 16-byte vector
  constexpr int kKeyLoads = kDepth / (4 * kLoad);        // of a lane and 16 keys
  constexpr int kValueLoads = kDepth / (2 * kLoad);      // of a lane and 32 keys
  constexpr int kValueRow = kDepth * 2 + 32;             // 8 rows of 32 bytes fill the banks
  constexpr int kJoinRow = kDepth + 4;                   // floats
  constexpr int kHeld = kWaves * kStep * kValueRow, kJoined = kWaves * 16 * kJoinRow * 4;
  __shared__ __attribute__((aligned(16))) unsigned char held[kHeld > kJoined ? kHeld : kJoined];
  __shared__ float joined_top[kWaves][16], joined_sum[kWaves][16];

  const int lanes = p.heads * layout.row_tiles, slot = (int)(blockIdx.x / (uint32_t)lanes), rest = (int)(blockIdx.x % (uint32_t)lanes);
  const int group = rest / layout.row_tiles, row_tile = rest % layout.row_tiles;
  SplitChunk chunk;
  const int each = tiles_each(p, b.marks, layout.target);
  if (!chunk_of(p, b.marks, slot, each, &chunk)) return;
  const AttentionSequence s = attention_sequence(p, b.marks, chunk.index);
  const SplitTiles tiles = tiles_of(p, s);
  const int begin = chunk.chunk * each, end = min(begin + each, tiles.tiles);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWaveLanes), lane = (int)threadIdx.x % kWaveLanes;
  const int column = lane % 16, quarter = lane / 16;
  const int first_row = row_tile * 16 * kBlocks;
  // what some row of the sequence sees, and what this tile of rows does (its first and last tokens)
  const AttentionSpan any{attention_span(p, s.keys, s.first).low, attention_span(p, s.keys, s.first + s.rows - 1).high};
  const AttentionSpan tile_first = attention_span(p, s.keys, s.first + first_row / p.shared);
  const AttentionSpan tile_last = attention_span(p, s.keys, s.first + (min(first_row + 16 * kBlocks, layout.rows) - 1) / p.shared);

  // queries: a lane's row is its column, its dims those that its key loads bring: vector j holds elements
  // (4 j + quarter) kLoad on, of which e4m3 makes two operands
  u32x4 query[kBlocks][kSteps];
  AttentionSpan span[kBlocks];
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
  for (int n = 0; n < kBlocks; ++n) {
    const int row = first_row + 16 * n + column, token = min(row, layout.rows - 1) / p.shared;
    const unsigned char *from = attention_query(p, b, s, chunk.index, token, group * p.shared + min(row, layout.rows - 1) % p.shared);
    span[n] = attention_span(p, s.keys, s.first + token);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int dim = kNarrow ? (k / 2 * 4 + quarter) * 16 + k % 2 * 8 : (4 * k + quarter) * 8;
      u32x4 w = {0, 0, 0, 0};
      if (row < layout.rows && dim < p.depth && p.scale != 0.0f) w = load16(from, dim / 8);
      query[n][k] = w ^ flip;
    }
  }
  const float c = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * kLog2E;

  f32x4 out[kBlocks][kDims];
  float top[kBlocks], sum[kBlocks];
#pragma unroll
  for (int n = 0; n < kBlocks; ++n) {
    top[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) out[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const unsigned char *keys = static_cast<const unsigned char *>(b.key) + (int64_t)group * p.k_head;
  const unsigned char *values = static_cast<const unsigned char *>(b.value) + (int64_t)group * p.v_head;
  const bool paged = p.kind == AttentionKind::kPaged;
  const int32_t *table = paged ? b.table + (int64_t)chunk.index * p.table_row : nullptr;
  auto first_key = [&](int tile) { return (tile < tiles.sinks ? tile * kTile : tiles.low + (tile - tiles.sinks) * kTile) + wave * kStep; };
  // a lane's two keys of a step: its column and 16 on; past the last key the last one's place is asked for
  auto pages = [&](int tile, int (&page)[2]) {
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      page[sub] = 0;
      if (paged) page[sub] = table[p.page.quotient((uint32_t)min(first_key(tile) + 16 * sub + column, any.high - 1))];
    }
  };
  u32x4 next_keys[2][kKeyLoads], next_values[kValueLoads];
  uint32_t next_alive;  // bit j: key j of the step is there and some row sees it
  auto fetch = [&](int tile, const int (&page)[2]) {
    int64_t key_at[2], value_at[2];
    bool there[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int key = first_key(tile) + 16 * sub + column, known = min(key, any.high - 1);
      there[sub] = attention_sees(p, any, key);
      if (paged) {
        there[sub] = there[sub] && (uint32_t)page[sub] < (uint32_t)p.pages;
        const uint32_t at = (uint32_t)known - p.page.quotient((uint32_t)known) * p.page.divisor;
        // (a page that is not there is read as the cache's first row, which is there: its keys are not alive)
        key_at[sub] = value_at[sub] = there[sub] ? (int64_t)page[sub] * p.k_sequence + (int64_t)at * p.k_row : 0;
      } else {
        key_at[sub] = (int64_t)chunk.index * p.k_sequence + (int64_t)known * p.k_row;
        value_at[sub] = (int64_t)chunk.index * p.v_sequence + (int64_t)known * p.v_row;
      }
    }
    next_alive = ((uint32_t)__ballot(there[0]) & 0xFFFFu) | ((uint32_t)__ballot(there[1]) << 16);
    const int last = p.depth / kLoad - 1;  // vectors past the depth: the row's last one, in whose place zeros are used
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) next_keys[sub][k] = load16(keys + key_at[sub], (size_t)min(4 * k + quarter, last));
    const int64_t at = (lane & 16) != 0 ? value_at[1] : value_at[0];
#pragma unroll
    for (int k = 0; k < kValueLoads; ++k) next_values[k] = load16(values + at, (size_t)min(2 * k + lane / 32, last));
  };

  unsigned char *rows = held + wave * kStep * kValueRow;
  int page[2], next_page[2] = {0, 0};
  if (begin < end) {
    pages(begin, page);
    if (begin + 1 < end) pages(begin + 1, next_page);
    fetch(begin, page);
  }
  for (int tile = begin; tile < end; ++tile) {
    u32x4 key_words[2][kKeyLoads], value_words[kValueLoads];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) key_words[sub][k] = next_keys[sub][k];
#pragma unroll
    for (int k = 0; k < kValueLoads; ++k) value_words[k] = next_values[k];
    const uint32_t alive = next_alive;
    if (tile + 1 < end) {
      page[0] = next_page[0], page[1] = next_page[1];
      if (tile + 2 < end) pages(tile + 2, next_page);
      fetch(tile + 1, page);
    }
    if (alive == 0) continue;
    const int first = first_key(tile);
    const bool whole = alive == 0xFFFFFFFFu && first + kStep <= tile_first.high && first >= tile_last.low;

    f32x4 score[kBlocks][2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) score[n][sub] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) {
        u32x4 w = key_words[sub][k];
        if (p.depth != kDepth && (4 * k + quarter) * kLoad >= p.depth) w = u32x4{0, 0, 0, 0};
        if constexpr (kNarrow) {
          u32x4 low, high;
          widened<T>(w, &low, &high);
#pragma unroll
          for (int n = 0; n < kBlocks; ++n) score[n][sub] = product16<T>(low, query[n][2 * k], score[n][sub]);
#pragma unroll
          for (int n = 0; n < kBlocks; ++n) score[n][sub] = product16<T>(high, query[n][2 * k + 1], score[n][sub]);
        } else {
#pragma unroll
          for (int n = 0; n < kBlocks; ++n) score[n][sub] = product16<T>(w, query[n][k], score[n][sub]);
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * sub + 4 * quarter + r;
            if (((alive >> j) & 1u) == 0 || !attention_sees(p, span[n], first + j)) score[n][sub][r] = -INFINITY;
          }
    }
    float most[kBlocks];
    bool grown = false;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      most[n] = fmaxf(fmaxf(fmaxf(score[n][0][0], score[n][0][1]), fmaxf(score[n][0][2], score[n][0][3])),
                      fmaxf(fmaxf(score[n][1][0], score[n][1][1]), fmaxf(score[n][1][2], score[n][1][3])));
      most[n] = rows_max(most[n]) * c;
      grown |= most[n] > top[n] + kSlack;
    }
    if (__ballot(grown) != 0) {
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) {
        const float next = fmaxf(top[n], most[n]);
        const float keep = top[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[n] - next);
        top[n] = next;
        sum[n] *= keep;
#pragma unroll
        for (int d = 0; d < kDims; ++d) out[n][d] *= keep;
      }
    }
    u32x4 weights[kBlocks];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const float shift = top[n] == -INFINITY ? 0.0f : top[n];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          score[n][sub][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][sub][r], c, -shift));
          sum[n] += score[n][sub][r];
        }
        weights[n][2 * sub] = pack2<T>(score[n][sub][0], score[n][sub][1]);
        weights[n][2 * sub + 1] = pack2<T>(score[n][sub][2], score[n][sub][3]);
      }
    }

    // values to the wave's rows in LDS; keys that are not alive bring zeros
    const bool mine = ((alive >> (lane % 32)) & 1u) != 0;
    auto put = [&]() {
#pragma unroll
      for (int k = 0; k < kValueLoads; ++k) {
        unsigned char *to = rows + lane % 32 * kValueRow + (2 * k + lane / 32) * kLoad * 2;
        const u32x4 w = value_words[k];
        if constexpr (kNarrow) {
          u32x4 low, high;
          widened<T>(w, &low, &high);
          *reinterpret_cast<u32x4 *>(to) = low;
          *reinterpret_cast<u32x4 *>(to + 16) = high;
        } else {
          *reinterpret_cast<u32x4 *>(to) = w;
        }
      }
      __builtin_amdgcn_wave_barrier();  // other lanes' rows are read next: a wave's LDS accesses are in order
    };
    if (alive != 0xFFFFFFFFu) {
#pragma unroll
      for (int k = 0; k < kValueLoads; ++k) value_words[k] = mine ? value_words[k] : u32x4{0, 0, 0, 0};
    }
    if (!whole && s.rows > 1) {
      // Values that are no numbers, of keys that not every row sees: a weight of 0 would make NaN of them in the product.
      // They are added to the rows that see them (a finite weight changes nothing about them) and zeroed.
      uint32_t found = 0;
#pragma unroll
      for (int k = 0; k < kValueLoads; ++k) found |= no_numbers<C>(value_words[k]);
      if (__ballot(found != 0) != 0) {
        put();
        for (int j = 0; j < kStep; ++j) {
          if (((alive >> j) & 1u) == 0) continue;
#pragma unroll
          for (int n = 0; n < kBlocks; ++n) {
            const bool sees = attention_sees(p, span[n], first + j);
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float v = Traits<T>::load(rows + j * kValueRow, 16 * d + 4 * quarter + r);
                if (sees && !(fabsf(v) < INFINITY)) out[n][d][r] += v;
              }
          }
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < kValueLoads; ++k) value_words[k] = numbers_only<C>(value_words[k]);
      }
    }
    put();
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      const unsigned char *at = rows + (4 * quarter + column / 4) * kValueRow + (d * 16 + column % 4 * 4) * 2;
      const uint2 near = read_transposed(at), far = read_transposed(at + 16 * kValueRow);
      const u32x4 value = {near.x, near.y, far.x, far.y};
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) out[n][d] = product16<T>(value, weights[n], out[n][d]);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // join the waves, 16 rows at a time
  float *joined = reinterpret_cast<float *>(held);
  const int join_row = (int)threadIdx.x / 16;
#pragma unroll
  for (int n = 0; n < kBlocks; ++n) {
    __syncthreads();
    const float total = rows_sum(sum[n]);
    if (quarter == 0) joined_top[wave][column] = top[n], joined_sum[wave][column] = total;
#pragma unroll
    for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4 *>(joined + (wave * 16 + column) * kJoinRow + d * 16 + 4 * quarter) = out[n][d];
    __syncthreads();
    const int row = first_row + 16 * n + join_row;
    if (row < layout.rows) {
      float most = joined_top[0][join_row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = fmaxf(most, joined_top[w][join_row]);
      const float shift = most == -INFINITY ? 0.0f : most;
      float keep[kWaves], all = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        keep[w] = __builtin_amdgcn_exp2f(joined_top[w][join_row] - shift);
        all += joined_sum[w][join_row] * keep[w];
      }
      const int64_t at = (s.row + row / p.shared) * p.queries + group * p.shared + row % p.shared;
      const int64_t part = ((int64_t)slot * p.heads + group) * layout.rows + row;
      const float inverse = all == 0.0f ? 0.0f : 1.0f / all;
      for (int d = (int)threadIdx.x % 16 * 4; d < p.depth; d += 64) {
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o += *reinterpret_cast<const f32x4 *>(joined + (w * 16 + join_row) * kJoinRow + d) * keep[w];
        if (chunk.chunks == 1) {
          uint2 w;
          w.x = pack2<T>(o[0] * inverse, o[1] * inverse);
          w.y = pack2<T>(o[2] * inverse, o[3] * inverse);
          *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(b.out) + (at * p.depth + d) * 2) = w;
        } else {
          *reinterpret_cast<f32x4 *>(layout.partial + part * p.depth + d) = o;
        }
      }
      if (threadIdx.x % 16 == 0) {
        if (chunk.chunks != 1) layout.stats[part] = float2{most, all};
        else if (b.logs != nullptr) b.logs[at] = all == 0.0f ? -INFINITY : most * kLn2 + logf(all);
      }
    }
  }
}

// The chunks of one query row joined: kThreads / kDepth chunks side by side, a dim to a thread.
template <class T, int kDepth>
__global__ __launch_bounds__(kThreads) void attention_join(AttentionParams p, AttentionBuffers b, SplitLayout layout) {
  constexpr int kParts = kThreads / kDepth;
  __shared__ float joined[kParts][kDepth], tops[kParts], sums[kParts];
  const int lines = p.heads * layout.rows, index = (int)(blockIdx.x / (uint32_t)lines), rest = (int)(blockIdx.x % (uint32_t)lines);
  const int group = rest / layout.rows, row = rest % layout.rows;
  const int each = tiles_each(p, b.marks, layout.target);
  // the slots before this sequence's
  int before = 0, chunks = 0;
  const int lane = (int)threadIdx.x % kWaveLanes;
  for (int base = 0; base <= index; base += kWaveLanes) {
    uint32_t mine = 0;
    if (base + lane <= index) mine = (uint32_t)max(1, (tiles_of(p, attention_sequence(p, b.marks, base + lane)).tiles + each - 1) / each);
    before += __builtin_amdgcn_readlane((int)scanned(mine, lane), kWaveLanes - 1);
    chunks = __builtin_amdgcn_readlane((int)mine, index % kWaveLanes);  // (of the last round)
  }
  if (chunks == 1) return;  // the split kernel's block was the whole sequence
  before -= chunks;
  const AttentionSequence s = attention_sequence(p, b.marks, index);
  const int dim = (int)threadIdx.x % kDepth, part = (int)threadIdx.x / kDepth;
  const int64_t first = ((int64_t)before * p.heads + group) * layout.rows + row, stride = (int64_t)p.heads * layout.rows;
  float most = -INFINITY;
  for (int i = part; i < chunks; i += kParts) most = fmaxf(most, layout.stats[first + i * stride].x);
  const float shift = most == -INFINITY ? 0.0f : most;
  float out = 0.0f, sum = 0.0f;
#pragma unroll 4
  for (int i = part; i < chunks; i += kParts) {
    const float2 stat = layout.stats[first + i * stride];
    const float keep = __builtin_amdgcn_exp2f(stat.x - shift);
    sum += stat.y * keep;
    if (dim < p.depth) out += layout.partial[(first + i * stride) * p.depth + dim] * keep;
  }
  joined[part][dim] = out;
  if (dim == 0) tops[part] = most, sums[part] = sum;
  __syncthreads();
  if (part != 0) return;
  float all = tops[0];
#pragma unroll
  for (int i = 1; i < kParts; ++i) all = fmaxf(all, tops[i]);
  const float base = all == -INFINITY ? 0.0f : all;
  out = 0.0f, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const float keep = __builtin_amdgcn_exp2f(tops[i] - base);
    out += joined[i][dim] * keep;
    sum += sums[i] * keep;
  }
  const int64_t at = (s.row + row / p.shared) * p.queries + group * p.shared + row % p.shared;
  if (dim < p.depth) Traits<T>::store(b.out, (size_t)(at * p.depth + dim), sum == 0.0f ? 0.0f : out / sum);
  if (b.logs != nullptr && dim == 0) b.logs[at] = sum == 0.0f ? -INFINITY : all * kLn2 + logf(sum);
}

}  // namespace

template <class C, int kDepth, int kBlocks> struct AttentionSplitTag {
  static std::string text() {
    return std::string("attention_split/") + (std::is_same<C, E4M3>::value ? "e4m3/d" : "d") + std::to_string(kDepth) + "/" + std::to_string(16 * kBlocks) + "-rows";
  }
};
template <int kDepth> struct AttentionJoinTag {
  static std::string text() { return "attention_join/d" + std::to_string(kDepth); }
};

namespace {
int padded_depth(const AttentionParams &p) { return p.depth <= 64 ? 64 : p.depth <= 128 ? 128 : 256; }
int blocks_of(const AttentionParams &p) {
  const int64_t rows = (int64_t)p.rows * p.shared;
  return rows <= 16 ? 1 : rows <= 32 || p.depth > 128 ? 2 : 4;
}
int row_tiles_of(const AttentionParams &p) {
  const int64_t each = 16 * blocks_of(p);
  return (int)(((int64_t)p.rows * p.shared + each - 1) / each);
}
}  // namespace

AttentionSplit attention_split_of(const AttentionParams &p, int compute_units) {
  AttentionSplit split;
  // the chunks of one key head and tile of rows: four blocks to a compute unit over all of them
  const int64_t lanes = (int64_t)p.heads * row_tiles_of(p);
  const int64_t target = ((int64_t)compute_units * 4 + lanes - 1) / lanes;
  const int64_t most = ((int64_t)p.keys + kTile - 1) / kTile + 1;  // tiles of a sequence
  split.target = (int)target;
  // sum over the sequences of ceil(tiles / each) with each >= total / target
  int64_t slots = target + p.sequences;
  if (most * p.sequences < slots) slots = most * p.sequences;
  split.slots = (int)(slots < p.sequences ? p.sequences : slots);
  split.joined = p.keys > kTile && target > 1;
  const int64_t rows = (int64_t)p.rows * p.shared * p.heads * split.slots;
  split.stats_offset = ((size_t)rows * (size_t)p.depth * sizeof(float) + 255) / 256 * 256;
  split.workspace = split.joined ? split.stats_offset + (size_t)rows * sizeof(float2) : 0;
  return split;
}

bool attention_split_serves(Elem type, const AttentionParams &p, bool vector_aligned) {
  if (type == Elem::kF32 || p.kind == AttentionKind::kPacked || !vector_aligned || p.depth % (p.narrow_cache ? 16 : 8) != 0) return false;
  return ((p.q_sequence | p.q_row | p.q_head | p.k_sequence | p.k_row | p.k_head | p.v_sequence | p.v_row | p.v_head) % 16) == 0;
}

namespace {
template <class T, class C, int kDepth, int kBlocks>
void start_split(const AttentionParams &p, const AttentionBuffers &b, const SplitLayout &layout, const AttentionSplit &split, hipStream_t stream) {
  note_variant<AttentionSplitTag<C, kDepth, kBlocks>>();
  hipLaunchKernelGGL((attention_split<T, C, kDepth, kBlocks>), dim3((uint32_t)split.slots * (uint32_t)(p.heads * layout.row_tiles)), dim3(kThreads), 0,
                     stream, p, b, layout);
  if (!split.joined) return;
  note_variant<AttentionJoinTag<kDepth>>();
  hipLaunchKernelGGL((attention_join<T, kDepth>), dim3((uint32_t)(p.heads * layout.rows) * (uint32_t)p.sequences), dim3(kThreads), 0, stream, p, b, layout);
}
template <class T, class C>
void split_by_depth(const AttentionParams &p, const AttentionBuffers &b, const SplitLayout &layout, const AttentionSplit &split, hipStream_t stream) {
  const int blocks = blocks_of(p);
  switch (padded_depth(p)) {
    case 64:
      if (blocks == 1) start_split<T, C, 64, 1>(p, b, layout, split, stream);
      else if (blocks == 2) start_split<T, C, 64, 2>(p, b, layout, split, stream);
      else start_split<T, C, 64, 4>(p, b, layout, split, stream);
      break;
    case 128:
      if (blocks == 1) start_split<T, C, 128, 1>(p, b, layout, split, stream);
      else if (blocks == 2) start_split<T, C, 128, 2>(p, b, layout, split, stream);
      else start_split<T, C, 128, 4>(p, b, layout, split, stream);
      break;
    default:
      if (blocks == 1) start_split<T, C, 256, 1>(p, b, layout, split, stream);
      else start_split<T, C, 256, 2>(p, b, layout, split, stream);
  }
}
}  // namespace

hipError_t launch_attention_split(Elem type, const AttentionParams &p, const AttentionBuffers &b, const AttentionSplit &split, void *workspace,
                                  hipStream_t stream) {
  SplitLayout layout;
  layout.target = split.target;
  layout.rows = p.rows * p.shared;
  layout.row_tiles = row_tiles_of(p);
  layout.partial = static_cast<float *>(workspace);
  layout.stats = reinterpret_cast<float2 *>(static_cast<unsigned char *>(workspace) + split.stats_offset);
  if (type == Elem::kF16) {
    if (p.narrow_cache) split_by_depth<F16, E4M3>(p, b, layout, split, stream);
    else split_by_depth<F16, F16>(p, b, layout, split, stream);
  } else {
    if (p.narrow_cache) split_by_depth<BF16, E4M3>(p, b, layout, split, stream);
    else split_by_depth<BF16, BF16>(p, b, layout, split, stream);
  }
  return hipGetLastError();
}

}  // namespace hyle_hip
