// attention_tiles.hip -- attention of many query rows on the matrix unit: f16 / bf16, depths of whole 16-byte vectors.
//
// A block takes 64 or 128 query rows of one head and walks over the keys that any of them sees, a step of 32 to 128 at a time;
// keys and values of a step are staged in LDS (two buffers: the loads of the next step are in flight while this one is
// computed), the queries stay in registers.  Everything is computed transposed, a query to a lane:
//   S^T[key, query] = K Q^T        (A: rows of K from LDS, B: the queries)
//   m' = max(m, max_key S^T c),  p = 2^(S^T c - m'),  l <- l 2^(m - m') + sum p,   c = scale * log2(e)
//   O^T[dim, query] <- O^T 2^(m - m') + V^T P^T   (A: columns of V by transposing LDS reads, B: p as it stands)
// so the row statistics are per lane (a lane holds half of a query's keys, the lane 32 away the other half), and p feeds the
// second product from the registers it was computed in: a lane's 8 keys of a 16-key step are 4h..4h+3 and 8+4h..8+4h+3 (h =
// lane / 32), and the columns of V are read in that order too, for the sum over the keys does not care.
// Weights are rounded once to the values' type, which the matrix unit asks for; sums and statistics, those that the rounded weights'
// products are divided by too, are f32.  (Outputs in bf16 are off by 0.0021 of their size in root mean square, rounded from f32
// throughout by 0.0016; f16 0.00028 and 0.0002.)
// Bound by the matrix and the vector units, which a wave uses in turn: 8192 causal tokens of 16 heads of 128, bf16, take 304 to
// 352 us by the machine (780 to 905 TFLOP/s of the 1190 of a large matrix product), the matrix unit is busy for 38 % of the cycles,
// the vector unit for 44 % (a quarter-rate power to each weight is 512 of its 1250 cycles of a wave's step, the products are 1024),
// LDS for 30 %, with no bank conflict; the rest is not accounted for.  Steps of 32 keys with three waves a SIMD took 359 where this took
// 307.  Depth 256 is bound by registers: two waves a SIMD spill 45 of them, queries that are read back between the products of every step
// (4096 tokens of 16 heads 277 us, 500 TFLOP/s), one wave a SIMD moves its outputs between the two halves of the register file.
// O is rescaled only when a maximum has grown by more than kSlack (2^8 stays exact in every type here).
#include "attention_math.h"

namespace hyle_hip {
namespace {

__device__ __forceinline__ float other_half_max(float v) {
  const auto both = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return fmaxf(bits_f32(both[0]), bits_f32(both[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
  const auto both = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return bits_f32(both[0]) + bits_f32(both[1]);
}

// Which tile of which sequence a slot of the grid is; false where it is none.  Late tiles, which see the most keys, come first.
// Packed sequence i, whose rows begin at b_i, has the places from first(i) = floor((b_i + (R - 1) i) / R) on: R rows to a tile,
// first(i + 1) - first(i) is at least its ceil(rows / R) tiles, so places need no sum over the sequences before, and each block finds
// its own by a search with 64 probes at a time (65536 sequences of one row, 8 heads: 3.3 ms, with a sum over all of them in each block 148; 7 or 64 sequences the same 8 us).
__device__ __forceinline__ bool tile_of(const AttentionParams &p, const int32_t *marks, int slot, int rows_per_tile, int tiles, int *index, int *tile) {
  if (p.kind != AttentionKind::kPacked) {
    *tile = tiles - 1 - slot / p.sequences;
    *index = slot % p.sequences;
    return true;
  }
  const int lane = (int)threadIdx.x % kWaveLanes;
  auto first = [&](int i, int begin) { return (int)(((uint64_t)begin + (uint64_t)(rows_per_tile - 1) * (uint64_t)i) / (uint32_t)rows_per_tile); };
  const int place = first(p.sequences, p.rows) - 1 - slot;
  int low = 0, count = p.sequences, step;  // the last sequence whose places begin at or before this one is among `count` from `low` on
  do {
    step = (count + kWaveLanes - 1) / kWaveLanes;
    const int at = lane * step;
    const bool before = at < count && first(low + at, min(max(marks[low + min(at, count - 1)], 0), p.rows)) <= place;
    const uint64_t lanes = __ballot(before);
    if (lanes == 0) return false;
    const int last = (kWaveLanes - 1 - __builtin_clzll(lanes)) * step;
    low += last;
    count = min(step, count - last);
  } while (step > 1);
  const AttentionSequence s = attention_sequence(p, marks, low);
  *index = low;
  *tile = place - first(low, (int)s.row);
  return *tile < (s.rows + rows_per_tile - 1) / rows_per_tile;
}

// Waves of a SIMD that the registers are kept for (one instead of two: 8192 tokens of 16 heads of 128 539 us instead of 311).
constexpr int resident(int depth, int row_waves, int key_waves) { return row_waves < 4 ? 1 : depth <= 64 && key_waves == 1 ? 3 : 2; }

// kRowWaves x 32 query rows to a block; kKeyWaves waves share each 32 of them, a kKeys of every step to each
template <class T, int kDepth, int kRowWaves, int kKeyWaves, int kKeys>
__global__ __launch_bounds__(kRowWaves * kKeyWaves * kWaveLanes, resident(kDepth, kRowWaves, kKeyWaves)) void attention_tiles(AttentionParams p, AttentionBuffers b, int tiles) {
  constexpr int kThreads = kRowWaves * kKeyWaves * kWaveLanes, kRows = kRowWaves * 32, kStage = kKeys * kKeyWaves;
  constexpr int kChunks = kDepth / 8;                       // 16-byte vectors of a row
  constexpr int kKeyRow = kDepth * 2 + 16;                  // 8 rows on in LDS lie in other banks
  constexpr int kValueRow = kDepth * 2 + 64;                // 4 rows of 64 bytes fill the banks
  constexpr int kStaged = (kStage * kChunks + kThreads - 1) / kThreads;  // vectors of a thread and step
  constexpr int kSubs = kKeys / 32, kSteps = kDepth / 16, kDims = kDepth / 32;
  constexpr int kBuffer = kStage * (kKeyRow + kValueRow);
  static_assert(kRowWaves * (kKeyWaves - 1) * (kDims * 4 * 16 + 8) * kWaveLanes <= 2 * kBuffer, "the joined waves fit where the keys were");
  __shared__ __attribute__((aligned(16))) unsigned char held[2 * kBuffer];
  __shared__ int no_number;  // 1 + the step whose values hold an infinity or NaN

  // heads that share keys on one XCD where they can be dealt evenly
  int slot, head;
  if (p.queries % 8 == 0) {
    const int each = p.queries / 8, rest = (int)blockIdx.x / 8;
    head = (int)blockIdx.x % 8 * each + rest % each;
    slot = rest / each;
  } else {
    head = (int)blockIdx.x % p.queries;
    slot = (int)blockIdx.x / p.queries;
  }
  int index, tile;
  if (!tile_of(p, b.marks, slot, kRows, tiles, &index, &tile)) return;
  const AttentionSequence s = attention_sequence(p, b.marks, index);
  const int group = (int)p.shared.quotient((uint32_t)head), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWaveLanes);
  const int lane = (int)threadIdx.x % kWaveLanes, row_wave = wave % kRowWaves, key_wave = wave / kRowWaves;
  const int half = lane / 32, column = lane % 32;
  const int block_row = tile * kRows, wave_row = block_row + row_wave * 32;
  const int block_last = min(block_row + kRows, s.rows) - 1, wave_last = min(wave_row + 32, s.rows) - 1;
  if (threadIdx.x == 0) no_number = 0;

  // the keys that some row of the block sees: whole steps of the sinks in front, then from low to high
  const AttentionSpan first_span = attention_span(p, s.keys, s.first + block_row), last_span = attention_span(p, s.keys, s.first + block_last);
  const int low = min(first_span.low, last_span.high) / kStage * kStage;
  const int before = (min(min(p.sinks, low), last_span.high) + kStage - 1) / kStage;
  const int steps = before + (last_span.high - low + kStage - 1) / kStage;
  const AttentionSpan wave_first = attention_span(p, s.keys, s.first + wave_row);
  const AttentionSpan wave_end = attention_span(p, s.keys, s.first + max(wave_last, wave_row));

  // queries: lane's row is column, its dims 8 half .. of every 16 (asked for before the first keys: the other way round took up to
  // 7 % longer)
  u32x4 query[kSteps];
  // a positive c, so that the maximum of S c is that of S and hidden scores stay -inf: its sign, or a scale of 0, goes into the queries
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
  {
    const int row = wave_row + column;
    const unsigned char *from = attention_query(p, b, s, min(row, s.rows - 1), head);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int chunk = 2 * k + half;
      u32x4 w = {0, 0, 0, 0};
      if (row < s.rows && chunk * 8 < p.depth && p.scale != 0.0f) w = load16(from, chunk);
      query[k] = w ^ flip;
    }
  }
  const float c = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * kLog2E;

  f32x16 out[kDims];
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) out[d][r] = 0.0f;

  const unsigned char *keys = static_cast<const unsigned char *>(b.key) + (int64_t)group * p.k_head +
                              (p.kind == AttentionKind::kPacked ? s.row * p.k_row : (int64_t)index * p.k_sequence);
  const unsigned char *values = static_cast<const unsigned char *>(b.value) + (int64_t)group * p.v_head +
                                (p.kind == AttentionKind::kPacked ? s.row * p.v_row : (int64_t)index * p.v_sequence);
  // A thread's vectors of a step.  Where whole rows make up the threads, it has the same vector of every kRowsApart-th row: one
  // offset of its own, and the rest is the same for all.
  constexpr bool kEven = kThreads % kChunks == 0;
  constexpr int kRowsApart = kThreads / kChunks, kOwn = kEven ? 1 : kStaged;
  u32x4 staged_keys[kStaged], staged_values[kStaged];
  int64_t key_from[kOwn], value_from[kOwn];
  bool in_depth[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int at = (int)threadIdx.x + i * kThreads, row = at / kChunks, chunk = at % kChunks;
    key_from[i] = (int64_t)row * p.k_row + chunk * 16;
    value_from[i] = (int64_t)row * p.v_row + chunk * 16;
    in_depth[i] = row < kStage && chunk * 8 < p.depth;
  }
  auto first_key = [&](int step) { return step < before ? step * kStage : low + (step - before) * kStage; };
  auto fetch = [&](int step) {
    const int first = first_key(step);
#pragma unroll
    for (int i = 0; i < kStaged; ++i) {
      const int own = kEven ? 0 : i, row = ((int)threadIdx.x + i * kThreads) / kChunks, apart = first + (kEven ? i * kRowsApart : 0);
      staged_keys[i] = staged_values[i] = u32x4{0, 0, 0, 0};
      if (in_depth[own] && first + row < s.keys) {
        staged_keys[i] = load16(keys + (int64_t)apart * p.k_row + key_from[own], 0);
        staged_values[i] = load16(values + (int64_t)apart * p.v_row + value_from[own], 0);
      }
    }
  };
  // whether every row of the block sees every key of a step
  auto whole_block = [&](int first) { return first + kStage <= first_span.high && first >= last_span.low; };
  auto store = [&](int step) {
    unsigned char *buffer = held + (step & 1) * kBuffer;
    const bool whole = whole_block(first_key(step));
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < kStaged; ++i) {
      const int at = (int)threadIdx.x + i * kThreads, row = at / kChunks, chunk = at % kChunks;
      if (row >= kStage) continue;
      *reinterpret_cast<u32x4 *>(buffer + row * kKeyRow + chunk * 16) = staged_keys[i];
      *reinterpret_cast<u32x4 *>(buffer + kStage * kKeyRow + row * kValueRow + chunk * 16) = staged_values[i];
      if (!whole) found |= no_numbers<T>(staged_values[i]);
    }
    if (found != 0) no_number = step + 1;
  };

  if (steps > 0) {
    fetch(0);
    __syncthreads();  // no_number is cleared
    store(0);
    __syncthreads();
  }
  for (int step = 0; step < steps; ++step) {
    const int first = first_key(step) + key_wave * kKeys;  // the wave's
    unsigned char *buffer = held + (step & 1) * kBuffer + key_wave * kKeys * kKeyRow;
    unsigned char *value_rows = held + (step & 1) * kBuffer + kStage * kKeyRow + key_wave * kKeys * kValueRow;
    if (step + 1 < steps) fetch(step + 1);
    const bool special = no_number == step + 1;
    // a wave none of whose rows sees a key of the step has nothing to do
    const bool idle = wave_row >= s.rows || first >= wave_end.high || (first + kKeys <= wave_first.low && first >= p.sinks);
    u32x4 weights[kKeys / 16];
    const AttentionSpan span = attention_span(p, s.keys, s.first + wave_row + column);
    if (!idle) {
      f32x16 score[kSubs];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
#pragma unroll
        for (int r = 0; r < 16; ++r) score[sub][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const u32x4 key = *reinterpret_cast<const u32x4 *>(buffer + (sub * 32 + column) * kKeyRow + (2 * k + half) * 16);
          score[sub] = product<T>(key, query[k], score[sub]);
        }
      }
      if (!(first + kKeys <= wave_first.high && first >= wave_end.low)) {
        asm volatile("" : : : "memory");  // (a branch: as selects, the comparisons cost every step a third of its instructions)
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = first + sub * 32 + 8 * (r / 4) + 4 * half + r % 4;
            score[sub][r] = attention_sees(p, span, key) ? score[sub][r] : -INFINITY;
          }
      }
      float most = score[0][0];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, score[sub][r]);
      most = other_half_max(most) * c;
      if (__ballot(most > top + kSlack) != 0) {
        const float next = fmaxf(top, most);
        const float keep = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - next);  // (what there is without a maximum is zeros and what is no number)
        top = next;
        sum *= keep;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) out[d][r] *= keep;
      }
      const float shift = top == -INFINITY ? 0.0f : top;
      float total = 0.0f;
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          score[sub][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[sub][r], c, -shift));
          total += score[sub][r];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int w = 0; w < 4; ++w) weights[sub * 2 + u][w] = pack2<T>(score[sub][8 * u + 2 * w], score[sub][8 * u + 2 * w + 1]);
      }
      sum += total;
    }
    if (special) {
      // Values that are no numbers, in a step that not every row sees whole: a weight of 0 would make NaN of them in the
      // product.  They are added to the rows that see them (a finite weight changes nothing about them) and zeroed.
      if (!idle) {
#pragma unroll 1
        for (int j = 0; j < kKeys; ++j) {
          const bool sees = attention_sees(p, span, first + j);
#pragma unroll
          for (int d = 0; d < kDims; ++d) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float v = Traits<T>::load(value_rows + j * kValueRow, 32 * d + 8 * (r / 4) + 4 * half + r % 4);
              if (sees && !(fabsf(v) < INFINITY)) out[d][r] += v;
            }
            asm volatile("" : : : "memory");  // (a block of dims at a time: all at once would cost every step its registers)
          }
        }
      }
      __syncthreads();
      for (int at = threadIdx.x; at < kStage * kDepth; at += kThreads) {
        uint16_t *element = reinterpret_cast<uint16_t *>(held + (step & 1) * kBuffer + kStage * kKeyRow + at / kDepth * kValueRow) + at % kDepth;
        if (!(fabsf(Traits<T>::load(element, 0)) < INFINITY)) *element = 0;
      }
      __syncthreads();
    }
    if (!idle) {
#pragma unroll
      for (int u = 0; u < kKeys / 16; ++u)
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const unsigned char *at = value_rows + (u * 16 + 4 * half + lane % 16 / 4) * kValueRow + (d * 32 + lane % 32 / 16 * 16 + lane % 4 * 4) * 2;
          const uint2 near = read_transposed(at), far = read_transposed(at + 8 * kValueRow);
          const u32x4 value = {near.x, near.y, far.x, far.y};
          out[d] = product<T>(value, weights[u], out[d]);
        }
    }
    if (step + 1 < steps) store(step + 1);
    __syncthreads();
  }

  if constexpr (kKeyWaves > 1) {
    // join the waves of the same rows: lane by lane, for they hold the same queries and dims (a lane's half of the keys each)
    f32x4 *joined = reinterpret_cast<f32x4 *>(held);
    float *stats = reinterpret_cast<float *>(held + kRowWaves * (kKeyWaves - 1) * kDims * 4 * kWaveLanes * 16);
    const int place = (key_wave - 1) * kRowWaves + row_wave;
    if (key_wave != 0) {
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          joined[((place * kDims + d) * 4 + r) * kWaveLanes + lane] = f32x4{out[d][4 * r], out[d][4 * r + 1], out[d][4 * r + 2], out[d][4 * r + 3]};
      stats[place * 2 * kWaveLanes + lane] = top;
      stats[(place * 2 + 1) * kWaveLanes + lane] = sum;
    }
    __syncthreads();
    if (key_wave != 0) return;
#pragma unroll
    for (int w = 0; w < kKeyWaves - 1; ++w) {
      const int from = w * kRowWaves + row_wave;
      const float other = stats[from * 2 * kWaveLanes + lane], next = fmaxf(top, other), shift = next == -INFINITY ? 0.0f : next;
      const float keep = __builtin_amdgcn_exp2f(top - shift), bring = __builtin_amdgcn_exp2f(other - shift);
      top = next;
      sum = sum * keep + stats[(from * 2 + 1) * kWaveLanes + lane] * bring;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 o = joined[((from * kDims + d) * 4 + r) * kWaveLanes + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) out[d][4 * r + e] = __builtin_fmaf(o[e], bring, out[d][4 * r + e] * keep);
        }
    }
  }

  const int row = wave_row + column;
  const float total = other_half_sum(sum);
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
  if (row >= s.rows) return;
  const int64_t at = (s.row + row) * p.queries + head;
  unsigned char *to = static_cast<unsigned char *>(b.out) + at * p.depth * 2;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int dim = 32 * d + 8 * (r / 4) + 4 * half;
      if (dim < p.depth) {
        uint2 w;
        w.x = pack2<T>(out[d][r] * inverse, out[d][r + 1] * inverse);
        w.y = pack2<T>(out[d][r + 2] * inverse, out[d][r + 3] * inverse);
        *reinterpret_cast<uint2 *>(to + dim * 2) = w;
      }
    }
  if (b.logs != nullptr && half == 0) b.logs[at] = total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

}  // namespace

template <int kDepth, int kRowWaves, int kKeyWaves, int kKeys> struct AttentionTilesTag {
  static std::string text() {
    return "attention_tiles/d" + std::to_string(kDepth) + "/" + std::to_string(kRowWaves * 32) + "x" + std::to_string(kKeyWaves) + "x" + std::to_string(kKeys);
  }
};

// Tiles of all sequences, at most: of packed ones, whose lengths are not known here, as many as their rows and the rest of each
// one's last tile fill.
static uint64_t slots_of(const AttentionParams &p, uint64_t rows) {
  if (p.kind == AttentionKind::kPacked) return ((uint64_t)p.rows + (rows - 1) * (uint64_t)p.sequences) / rows;
  return ((uint64_t)p.rows + rows - 1) / rows * (uint64_t)p.sequences;
}

template <class T, int kDepth, int kRowWaves, int kKeyWaves, int kKeys>
static void start(const AttentionParams &p, const AttentionBuffers &b, hipStream_t stream) {
  constexpr int kRows = kRowWaves * 32;
  note_variant<AttentionTilesTag<kDepth, kRowWaves, kKeyWaves, kKeys>>();
  hipLaunchKernelGGL((attention_tiles<T, kDepth, kRowWaves, kKeyWaves, kKeys>), dim3((uint32_t)(slots_of(p, kRows) * (uint64_t)p.queries)),
                     dim3(kRowWaves * kKeyWaves * kWaveLanes), 0, stream, p, b, (p.rows + kRows - 1) / kRows);
}

bool attention_tiles_serves(Elem type, const AttentionParams &p, bool vector_aligned) {
  if (type == Elem::kF32 || p.kind == AttentionKind::kPaged || !vector_aligned || p.depth % 8 != 0) return false;
  // (so many blocks take the shapes of 128 rows, of depth 256 with two waves to each 32)
  if (!axis_holds(slots_of(p, 128) * (uint64_t)p.queries, p.depth <= 128 ? 256 : 512)) return false;
  return ((p.q_sequence | p.q_row | p.q_head | p.k_sequence | p.k_row | p.k_head | p.v_sequence | p.v_row | p.v_head) % 16) == 0;
}

hipError_t launch_attention_tiles(Elem type, const AttentionParams &p, const AttentionBuffers &b, int compute_units, hipStream_t stream) {
  // Two waves to each 32 rows, each with half the keys of a step, where there are too few blocks to fill the device or to hide
  // the loads' latency (us, one wave / two: 1500 tokens of 32 heads, depth 128, 384 blocks 52.1 / 39.2; 3000 of 16, 384 blocks
  // 96.1 / 70.2; 2000 of 32, depth 64, 512 blocks 46.7 / 39.0; 5000 of 16, 640 blocks 171 / 169; 8 padded sequences of 12 heads,
  // depth 64, 672 blocks 33.0 / 44.7; 8192 of 16, 1024 blocks 308 / 335).  One step of keys has no halves (16 tokens 7.3 / 8.2).
  // At depth 256 two waves always, of 64 rows (one wave a SIMD, nothing spilled) up to a block to a compute unit, then of 128 (two
  // waves, 45 registers spilled) (2048 tokens of 16 heads, 128 rows 133, 64 rows 112; 4096 of 16, 277 / 400; with a window of 300,
  // 4 heads, 43.7 / 30.4).
  const uint64_t blocks = slots_of(p, 128) * (uint64_t)p.queries;
  auto typed = [&](auto tag) {
    using T = decltype(tag);
    auto by = [&](auto depth) {
      constexpr int kDepth = decltype(depth)::value;
      if (p.keys <= 64 || blocks > 2 * (uint64_t)compute_units) start<T, kDepth, 4, 1, 64>(p, b, stream);
      else start<T, kDepth, 4, 2, 64>(p, b, stream);
    };
    if (p.depth <= 64) by(std::integral_constant<int, 64>{});
    else if (p.depth <= 96) by(std::integral_constant<int, 96>{});
    else if (p.depth <= 128) by(std::integral_constant<int, 128>{});
    else if (blocks > (uint64_t)compute_units) start<T, 256, 4, 2, 32>(p, b, stream);
    else start<T, 256, 2, 2, 32>(p, b, stream);
  };
  if (type == Elem::kF16) typed(F16{});
  else typed(BF16{});
  return hipGetLastError();
}

}  // namespace hyle_hip
