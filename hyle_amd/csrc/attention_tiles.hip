// attention_tiles.hip -- attention of many query rows on the matrix unit: f16 / bf16, depths of whole 16-byte vectors.
//
// A block takes kWaves * 32 * kBlocks query rows of one head and walks over the keys that any of them sees, kKeys at a time;
// keys and values of a step are staged in LDS (two buffers: the loads of the next step are in flight while this one is
// computed), the queries stay in registers.  Everything is computed transposed, a query to a lane:
//   S^T[key, query] = K Q^T        (A: rows of K from LDS, B: the queries)
//   m' = max(m, max_key S^T c),  p = 2^(S^T c - m'),  l <- l 2^(m - m') + sum p,   c = scale * log2(e)
//   O^T[dim, query] <- O^T 2^(m - m') + V^T P^T   (A: columns of V by transposing LDS reads, B: p as it stands)
// so the row statistics are per lane (a lane holds half of a query's keys, the lane 32 away the other half), and p feeds the
// second product from the registers it was computed in: a lane's 8 keys of a 16-key step are 4h..4h+3 and 8+4h..8+4h+3 (h =
// lane / 32), and the columns of V are read in that order too, for the sum over the keys does not care.
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

// Which tile of which sequence a slot of the grid is; false past the last.  Late tiles, which see the most keys, come first.
__device__ __forceinline__ bool tile_of(const AttentionParams &p, const int32_t *marks, int slot, int rows_per_tile, int tiles, int *index, int *tile) {
  if (p.kind != AttentionKind::kPacked) {
    *tile = tiles - 1 - slot / p.sequences;
    *index = slot % p.sequences;
    return true;
  }
  // packed: sequences have as many tiles as their rows fill; counted from the last one's last
  const int lane = (int)threadIdx.x % kWaveLanes;
  int before = 0;
  for (int last = p.sequences - 1; last >= 0; last -= kWaveLanes) {
    const int mine = last - lane;
    int count = 0;
    if (mine >= 0) {
      const AttentionSequence s = attention_sequence(p, marks, mine);
      count = (s.rows + rows_per_tile - 1) / rows_per_tile;
    }
    int through = count;  // of this lane's sequence and those after it
#pragma unroll
    for (int step = 1; step < kWaveLanes; step *= 2) {
      const int up = __shfl_up(through, step, kWaveLanes);
      if (lane >= step) through += up;
    }
    const uint64_t holds = __ballot(slot < before + through);
    if (holds != 0) {
      const int at = __builtin_ctzll(holds);
      const int end = before + __builtin_amdgcn_readlane(through, at);
      *index = last - at;
      *tile = end - 1 - slot;  // its last tile has the lowest slot
      return true;
    }
    before += __builtin_amdgcn_readlane(through, kWaveLanes - 1);
  }
  return false;
}

template <class T, int kDepth, int kWaves, int kBlocks, int kKeys>
__global__ __launch_bounds__(kWaves * kWaveLanes, kDepth <= 64 ? 3 : kDepth <= 128 ? 2 : 1) void attention_tiles(AttentionParams p, AttentionBuffers b, int tiles) {
  constexpr int kThreads = kWaves * kWaveLanes, kRows = kWaves * 32 * kBlocks;
  constexpr int kChunks = kDepth / 8;                       // 16-byte vectors of a row
  constexpr int kKeyRow = kDepth * 2 + 16;                  // 8 rows on in LDS lie in other banks
  constexpr int kValueRow = kDepth * 2 + 64;                // 4 rows of 64 bytes fill the banks
  constexpr int kStaged = (kKeys * kChunks + kThreads - 1) / kThreads;  // vectors of a thread and step
  constexpr int kSubs = kKeys / 32, kSteps = kDepth / 16, kDims = kDepth / 32;
  constexpr int kBuffer = kKeys * (kKeyRow + kValueRow);
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
  const int group = (int)p.shared.quotient((uint32_t)head), wave = (int)threadIdx.x / kWaveLanes, lane = (int)threadIdx.x % kWaveLanes;
  const int half = lane / 32, column = lane % 32;
  const int block_row = tile * kRows, wave_row = block_row + wave * 32 * kBlocks;
  const int block_last = min(block_row + kRows, s.rows) - 1, wave_last = min(wave_row + 32 * kBlocks, s.rows) - 1;
  if (threadIdx.x == 0) no_number = 0;

  // the keys that some row of the block sees: whole steps of the sinks in front, then from low to high
  const AttentionSpan first_span = attention_span(p, s.keys, s.first + block_row), last_span = attention_span(p, s.keys, s.first + block_last);
  const int low = min(first_span.low, last_span.high) / kKeys * kKeys;
  const int before = (min(min(p.sinks, low), last_span.high) + kKeys - 1) / kKeys;
  const int steps = before + (last_span.high - low + kKeys - 1) / kKeys;
  const AttentionSpan wave_first = attention_span(p, s.keys, s.first + wave_row);
  const AttentionSpan wave_end = attention_span(p, s.keys, s.first + max(wave_last, wave_row));

  // queries: lane's row is column, its dims 8 half .. of every 16
  u32x4 query[kBlocks][kSteps];
  // a positive c, so that the maximum of S c is that of S and hidden scores stay -inf: its sign, or a scale of 0, goes into the queries
  const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
  for (int q = 0; q < kBlocks; ++q) {
    const int row = wave_row + 32 * q + column;
    const unsigned char *from = attention_query(p, b, s, index, min(row, s.rows - 1), head);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int chunk = 2 * k + half;
      u32x4 w = {0, 0, 0, 0};
      if (row < s.rows && chunk * 8 < p.depth && p.scale != 0.0f) w = load16(from, chunk);
      query[q][k] = w ^ flip;
    }
  }
  const float c = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * kLog2E;

  f32x16 out[kBlocks][kDims];
  float top[kBlocks], sum[kBlocks];
#pragma unroll
  for (int q = 0; q < kBlocks; ++q) {
    top[q] = -INFINITY, sum[q] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[q][d][r] = 0.0f;
  }

  const unsigned char *keys = static_cast<const unsigned char *>(b.key) + (int64_t)group * p.k_head +
                              (p.kind == AttentionKind::kPacked ? s.row * p.k_row : (int64_t)index * p.k_sequence);
  const unsigned char *values = static_cast<const unsigned char *>(b.value) + (int64_t)group * p.v_head +
                                (p.kind == AttentionKind::kPacked ? s.row * p.v_row : (int64_t)index * p.v_sequence);
  u32x4 staged_keys[kStaged], staged_values[kStaged];
  auto first_key = [&](int step) { return step < before ? step * kKeys : low + (step - before) * kKeys; };
  auto fetch = [&](int step) {
    const int first = first_key(step);
#pragma unroll
    for (int i = 0; i < kStaged; ++i) {
      const int at = (int)threadIdx.x + i * kThreads, row = at / kChunks, chunk = at % kChunks, key = first + row;
      staged_keys[i] = staged_values[i] = u32x4{0, 0, 0, 0};
      if (row < kKeys && key < s.keys && chunk * 8 < p.depth) {
        staged_keys[i] = load16(keys + (int64_t)key * p.k_row, chunk);
        staged_values[i] = load16(values + (int64_t)key * p.v_row, chunk);
      }
    }
  };
  // whether every row of the block sees every key of a step
  auto whole_block = [&](int first) { return first + kKeys <= first_span.high && first >= last_span.low; };
  auto store = [&](int step) {
    unsigned char *buffer = held + (step & 1) * kBuffer;
    const bool whole = whole_block(first_key(step));
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < kStaged; ++i) {
      const int at = (int)threadIdx.x + i * kThreads, row = at / kChunks, chunk = at % kChunks;
      if (row >= kKeys) continue;
      *reinterpret_cast<u32x4 *>(buffer + row * kKeyRow + chunk * 16) = staged_keys[i];
      *reinterpret_cast<u32x4 *>(buffer + kKeys * kKeyRow + row * kValueRow + chunk * 16) = staged_values[i];
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
    const int first = first_key(step);
    unsigned char *buffer = held + (step & 1) * kBuffer;
    unsigned char *value_rows = buffer + kKeys * kKeyRow;
    if (step + 1 < steps) fetch(step + 1);
    const bool special = no_number == step + 1;
    // a wave none of whose rows sees a key of the step has nothing to do
    const bool idle = wave_row >= s.rows || first >= wave_end.high || (first + kKeys <= wave_first.low && first >= p.sinks);
    u32x4 weights[kBlocks][kKeys / 16];
    if (!idle) {
      f32x16 score[kBlocks][kSubs];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
#pragma unroll
        for (int q = 0; q < kBlocks; ++q)
#pragma unroll
          for (int r = 0; r < 16; ++r) score[q][sub][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const u32x4 key = *reinterpret_cast<const u32x4 *>(buffer + (sub * 32 + column) * kKeyRow + (2 * k + half) * 16);
#pragma unroll
          for (int q = 0; q < kBlocks; ++q) score[q][sub] = product<T>(key, query[q][k], score[q][sub]);
        }
      }
      if (!(first + kKeys <= wave_first.high && first >= wave_end.low)) {
        asm volatile("" : : : "memory");  // (a branch: as selects, the comparisons cost every step a third of its instructions)
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) {
          const AttentionSpan span = attention_span(p, s.keys, s.first + wave_row + 32 * q + column);
#pragma unroll
          for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int key = first + sub * 32 + 8 * (r / 4) + 4 * half + r % 4;
              score[q][sub][r] = attention_sees(p, span, key) ? score[q][sub][r] : -INFINITY;
            }
        }
      }
      float most[kBlocks];
      bool grown = false;
#pragma unroll
      for (int q = 0; q < kBlocks; ++q) {
        most[q] = score[q][0][0];
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r) most[q] = fmaxf(most[q], score[q][sub][r]);
        most[q] = other_half_max(most[q]) * c;
        grown |= most[q] > top[q] + kSlack;
      }
      if (__ballot(grown) != 0) {
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) {
          const float next = fmaxf(top[q], most[q]);
          const float keep = top[q] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[q] - next);
          top[q] = next;
          sum[q] *= keep;
#pragma unroll
          for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[q][d][r] *= keep;
        }
      }
#pragma unroll
      for (int q = 0; q < kBlocks; ++q) {
        const float shift = top[q] == -INFINITY ? 0.0f : top[q];
        float total = 0.0f;
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            score[q][sub][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[q][sub][r], c, -shift));
            total += score[q][sub][r];
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w)
              weights[q][sub * 2 + u][w] = pack2<T>(score[q][sub][8 * u + 2 * w], score[q][sub][8 * u + 2 * w + 1]);
        }
        sum[q] += total;
      }
    }
    if (special) {
      // Values that are no numbers, in a step that not every row sees whole: a weight of 0 would make NaN of them in the
      // product.  They are added to the rows that see them (a finite weight changes nothing about them) and zeroed.
      if (!idle) {
#pragma unroll 1
        for (int j = 0; j < kKeys; ++j) {
#pragma unroll
          for (int q = 0; q < kBlocks; ++q) {
            const AttentionSpan span = attention_span(p, s.keys, s.first + wave_row + 32 * q + column);
            const bool sees = attention_sees(p, span, first + j);
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const float v = Traits<T>::load(value_rows + j * kValueRow, 32 * d + 8 * (r / 4) + 4 * half + r % 4);
                if (sees && !(fabsf(v) < INFINITY)) out[q][d][r] += v;
              }
              asm volatile("" : : : "memory");  // (a block of dims at a time: all at once would cost every step its registers)
            }
          }
        }
      }
      __syncthreads();
      for (int at = threadIdx.x; at < kKeys * kDepth; at += kThreads) {
        uint16_t *element = reinterpret_cast<uint16_t *>(value_rows + at / kDepth * kValueRow) + at % kDepth;
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
#pragma unroll
          for (int q = 0; q < kBlocks; ++q) out[q][d] = product<T>(value, weights[q][u], out[q][d]);
        }
    }
    if (step + 1 < steps) store(step + 1);
    __syncthreads();
  }

#pragma unroll
  for (int q = 0; q < kBlocks; ++q) {
    const int row = wave_row + 32 * q + column;
    const float total = other_half_sum(sum[q]);
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    if (row >= s.rows) continue;
    const int64_t at = (s.row + row) * p.queries + head;
    unsigned char *to = static_cast<unsigned char *>(b.out) + at * p.depth * 2;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int dim = 32 * d + 8 * (r / 4) + 4 * half;
        if (dim < p.depth) {
          uint2 w;
          w.x = pack2<T>(out[q][d][r] * inverse, out[q][d][r + 1] * inverse);
          w.y = pack2<T>(out[q][d][r + 2] * inverse, out[q][d][r + 3] * inverse);
          *reinterpret_cast<uint2 *>(to + dim * 2) = w;
        }
      }
    if (b.logs != nullptr && half == 0) b.logs[at] = total == 0.0f ? -INFINITY : (top[q] + __builtin_amdgcn_logf(total)) * kLn2;
  }
}

}  // namespace

template <int kDepth, int kWaves, int kBlocks, int kKeys> struct AttentionTilesTag {
  static std::string text() {
    return "attention_tiles/d" + std::to_string(kDepth) + "/" + std::to_string(kWaves * 32 * kBlocks) + "x" + std::to_string(kKeys);
  }
};

template <class T, int kDepth, int kWaves, int kBlocks, int kKeys>
static void start(const AttentionParams &p, const AttentionBuffers &b, hipStream_t stream) {
  constexpr int kRows = kWaves * 32 * kBlocks;
  note_variant<AttentionTilesTag<kDepth, kWaves, kBlocks, kKeys>>();
  const int tiles = (p.rows + kRows - 1) / kRows;
  const uint64_t slots = p.kind == AttentionKind::kPacked ? (uint64_t)p.rows / kRows + (uint64_t)p.sequences : (uint64_t)tiles * (uint64_t)p.sequences;
  hipLaunchKernelGGL((attention_tiles<T, kDepth, kWaves, kBlocks, kKeys>), dim3((uint32_t)(slots * (uint64_t)p.queries)), dim3(kWaves * kWaveLanes), 0,
                     stream, p, b, tiles);
}

bool attention_tiles_serves(Elem type, const AttentionParams &p, bool vector_aligned) {
  if (type == Elem::kF32 || p.kind == AttentionKind::kPaged || !vector_aligned || p.depth % 8 != 0) return false;
  return ((p.q_sequence | p.q_row | p.q_head | p.k_sequence | p.k_row | p.k_head | p.v_sequence | p.v_row | p.v_head) % 16) == 0;
}

hipError_t launch_attention_tiles(Elem type, const AttentionParams &p, const AttentionBuffers &b, hipStream_t stream) {
  auto typed = [&](auto tag) {
    using T = decltype(tag);
    if (p.depth <= 64) start<T, 64, 4, 1, 64>(p, b, stream);
    else if (p.depth <= 96) start<T, 96, 4, 1, 64>(p, b, stream);
    else if (p.depth <= 128) start<T, 128, 4, 1, 64>(p, b, stream);
    else start<T, 256, 4, 1, 32>(p, b, stream);
  };
  if (type == Elem::kF16) typed(F16{});
  else typed(BF16{});
  return hipGetLastError();
}

}  // namespace hyle_hip
