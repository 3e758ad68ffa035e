// paged_select.hip -- the pages of each sequence that a query's products can be largest in, for every key head.
//
// score of a page = max over the key head's query heads and the new rows of sum_d q_d (q_d >= 0 ? high_d : low_d)
// which no key of the page passes.  Products are exact in 64 bits (11 or 24 bits by 8); sums are kept there and rounded once to f32.  The kernels
// below add in orders of their own, which moves a sum by 2^-45 of its terms' magnitudes at most (256 of them): so two of them may give
// neighbouring f32 numbers for a sum that lies so close to the middle between them, or whose terms cancel, and the choice differs where
// that decides between two pages.  A score that is no number counts as the largest.  The
// first page and those of the newest tokens are always chosen, then the best, ties to the earlier, and written in their order.
// Two launches: scores to the workspace, and one block to a key head that finds the last chosen score digit by digit.
//
// Bound by the bytes of the bounds and, with many query rows, by the 64-bit products: 16 sequences of 20000 to 32768 keys in pages of 16, 8 key
// heads of 128 with four query heads each, 105 MB: scores 25.6 us (4.1 TB/s), choice 10.1, a launch and five latencies in a row (length, scores,
// what they begin with, some seven digits, the write).  One sequence of 131055 keys in pages of 32, 2 key heads of 256, 16 rows each: 8.5
// and 11 us.  Scores by the vector unit, a lane to eight channels, took 34 and 17 us (two conversions and two multiply-adds to a
// word and row, and sums across lanes); with the rows' parts in registers instead of LDS 36 and 6.5 (15 us of preparing them); with each lane's
// loads where the matrix unit wants them, four lanes to 64 bytes of a page, 30 (whole rows side by side through LDS: 25.6).
#include <algorithm>

#include "attention.h"

namespace hyle_hip {
namespace {

struct SelectSpan {
  uint32_t length, filled, newest;  // keys, pages that hold some, the first of those that hold the newest tokens
  uint32_t rows_before;             // new rows that stand before the sequence
};
__device__ __forceinline__ SelectSpan select_span(const PagedSelectParams &p, const int32_t *lengths, uint32_t sequence) {
  SelectSpan s;
  s.length = (uint32_t)max(lengths[sequence], 0);
  const uint64_t filled = s.length == 0 ? 0 : p.page.quotient(s.length - 1) + 1ull;
  s.filled = (uint32_t)min(filled, (uint64_t)p.columns);
  s.newest = min(p.page.quotient(s.length > p.rows ? s.length - p.rows : 0u), s.filled);
  s.rows_before = s.length < p.rows ? p.rows - s.length : 0u;
  return s;
}
// Only these are ranked: not the first page and not the newest tokens', and only where not all are chosen.
__device__ __forceinline__ bool ranked(const PagedSelectParams &p, const SelectSpan &s, uint32_t column) {
  return column >= 1 && column < s.newest && s.filled > p.count;
}
// f32 in the order of unsigned numbers; zeros are equal, what is no number is +inf.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t bits = x != x ? 0x7F800000u : f32_bits(x + 0.0f);
  return (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
}

// A page's score as it is defined, a lane to every 64th channel; the same in every lane.
template <class T>
__device__ __forceinline__ uint32_t page_score(const PagedSelectParams &p, const SelectSpan &s, const unsigned char *query, const unsigned char *bounds,
                                               uint32_t sequence, uint32_t head, int32_t page) {
  const unsigned char *low = bounds + page * p.b_page + head * p.b_head, *high = low + p.b_side;
  uint32_t best = ordered(-INFINITY);
#pragma unroll 1
  for (uint32_t r = s.rows_before; r < p.rows; ++r)
#pragma unroll 1
    for (uint32_t h = 0; h < p.shared.divisor; ++h) {
      const unsigned char *q = query + sequence * p.q_sequence + r * p.q_row + (head * p.shared.divisor + h) * p.q_head;
      double sum = 0.0;
      for (uint32_t d = threadIdx.x % kWaveLanes; d < p.depth; d += kWaveLanes) {
        const float x = Traits<T>::load(q, d);
        sum += (double)x * (double)Traits<BF16>::load(x >= 0.0f ? high : low, d);
      }
      best = max(best, ordered((float)wave_sum(sum)));
    }
  return best;
}

// Any depth and alignment: a wave to a page and key head.
template <class T>
__global__ __launch_bounds__(kBlockThreads) void paged_scores(PagedSelectParams p, const unsigned char *query, const unsigned char *bounds,
                                                              const int32_t *table, const int32_t *lengths, uint32_t *scores) {
  const uint64_t unit = (uint64_t)blockIdx.x * (kBlockThreads / kWaveLanes) + threadIdx.x / kWaveLanes;
  const uint32_t column = (uint32_t)(unit % p.columns);
  const uint64_t line = unit / p.columns;  // sequence and key head
  if (line >= (uint64_t)p.sequences * p.heads) return;
  const uint32_t sequence = (uint32_t)(line / p.heads), head = (uint32_t)(line - (uint64_t)sequence * p.heads);
  const SelectSpan s = select_span(p, lengths, sequence);
  if (!ranked(p, s, column)) return;
  const int32_t page = table[(int64_t)sequence * p.table_row + column];
  const uint32_t best = (uint32_t)page < p.pages ? page_score<T>(p, s, query, bounds, sequence, head, page) : ordered(-INFINITY);
  if (threadIdx.x % kWaveLanes == 0) scores[unit] = best;
}

// By the matrix unit in 64 bits: sixteen pages to a wave's tile, A their largest keys, then their least, B the query rows' positive and negative
// parts, which the block's waves read from LDS: sum_d q_d+ high_d + q_d- low_d.  Parts that are zero multiply a bound too, and an infinite one
// would make NaN of it: where a sum is no finite number, the page's score is taken again as it is defined.  (No bound is infinite where
// the sum is finite, so those are right.)  kRows: query rows of a step: 4 in four blocks of four pages, or 16.  A wave takes 64 or 128 channels;
// with more, kParts = 2 waves share a tile and join their sums in LDS.  A lane reads eight channels of a page, four lanes 64 bytes.
typedef double f64x4 __attribute__((ext_vector_type(4)));
// The words of a tile's next 32 channels are asked for as soon as those of this one's are converted.
template <class T, int kDepth, int kRows>
__global__ __launch_bounds__(kBlockThreads, kRows == 4 ? 4 : kDepth == 256 ? 1 : 2) void paged_scores_tiles(PagedSelectParams p, Divisor blocks, uint32_t tiles,
                                                                                        const unsigned char *query, const unsigned char *bounds,
                                                                                        const int32_t *table, const int32_t *lengths, uint32_t *scores) {
  constexpr int kWaves = kBlockThreads / kWaveLanes, kParts = kDepth == 256 ? 2 : 1, kMine = kDepth / kParts, kChunks = kMine / 32;
  constexpr int kItems = kRows == 4 ? 1 : 4, kVectors = 8 / Traits<T>::kVec;
  constexpr int kRowVectors = kMine / 8, kLoads = 16 * kRowVectors / kWaveLanes, kRow = kMine * 2 + 16;  // (bytes: 16 rows of 16 fill the banks)
  __shared__ double signs[kDepth / 4][2][4][kRows];  // a step's positive and negative parts: of four channels, eight apart
  __shared__ __attribute__((aligned(16))) unsigned char held[kWaves][16 * kRow];
  __shared__ double joined[2][kParts == 2 ? kWaves / 2 : 1][kItems][kParts == 2 ? kWaveLanes : 1];
  // (a page's heads stand behind one another in memory, so they are looked at at the same time)
  const uint32_t sequence = blocks.quotient(blockIdx.x), rest = blockIdx.x - sequence * blocks.divisor, block = rest / p.heads, head = rest - block * p.heads;
  const uint32_t line = sequence * p.heads + head;
  const uint32_t lane = threadIdx.x % kWaveLanes, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWaveLanes));
  const uint32_t tile_wave = wave / kParts, part = wave % kParts;
  const SelectSpan s = select_span(p, lengths, sequence);
  const uint32_t block_first = block * (kWaves / kParts) * 16 * tiles;
  if (s.filled <= p.count || block_first >= s.newest) return;
  // tiles of the block's waves in turn; all of them go as far as the first wave does
  const uint32_t first = block_first + tile_wave * 16, count = min(tiles, (s.newest - block_first + 16 * (kWaves / kParts) - 1) / (16 * (kWaves / kParts)));
  const uint32_t rows = (p.rows - s.rows_before) * p.shared.divisor, quarter = lane / 16;
  // (lanes past the depth read the row's first vector, times zeros)
  uint32_t vector = part * kRowVectors + lane % kRowVectors;
  if (vector >= p.depth / 8) vector = 0;
  auto page_of = [&](uint32_t t) {  // of the lane's column
    const uint32_t column = first + 16 * (kWaves / kParts) * t + lane % 16;
    return t < count && ranked(p, s, column) ? table[(int64_t)sequence * p.table_row + column] : -1;
  };
  // Whole rows side by side, low and high in turn; to the lanes that multiply them through LDS.
  u32x4 low[kLoads], high[kLoads];
  const unsigned char *from[kLoads];
  auto places = [&](int32_t page) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int32_t of = __shfl(page, k * (kWaveLanes / kRowVectors) + (int)(lane / kRowVectors), kWaveLanes);
      from[k] = bounds + ((uint32_t)of < p.pages ? of * p.b_page : 0) + head * p.b_head;
    }
  };
  auto ask = [&](u32x4 (&words)[kLoads], int64_t side) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) words[k] = load16_stream(from[k] + side, vector);
  };
  auto put = [&](const u32x4 (&words)[kLoads]) {
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses are in order)
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      *reinterpret_cast<u32x4 *>(held[wave] + (k * (kWaveLanes / kRowVectors) + lane / kRowVectors) * kRow + lane % kRowVectors * 16) = words[k];
    __builtin_amdgcn_wave_barrier();
  };
#pragma unroll 1
  for (uint32_t group = 0; group < rows; group += kRows) {
    int32_t page = page_of(0), next = page_of(1);
    places(page);
    ask(low, 0);
    ask(high, p.b_side);
    if (group != 0) __syncthreads();  // the rows before are read
    for (uint32_t i = threadIdx.x; i < kRows * kDepth / 8; i += kBlockThreads) {
      const uint32_t j = i % kRows, v = i / kRows, index = min(group + j, rows - 1), row = p.shared.quotient(index), shared = index - row * p.shared.divisor;
      const unsigned char *from = query + sequence * p.q_sequence + (s.rows_before + row) * p.q_row + (head * p.shared.divisor + shared) * p.q_head;
      float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (v < p.depth / 8) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
          float part_of[Traits<T>::kVec];
          Traits<T>::unpack(load16(from, v * kVectors + k), part_of);
#pragma unroll
          for (int e = 0; e < Traits<T>::kVec; ++e) x[k * Traits<T>::kVec + e] = part_of[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        signs[v / 4 * 8 + e][0][v % 4][j] = (double)(x[e] >= 0.0f ? x[e] : 0.0f);
        signs[v / 4 * 8 + e][1][v % 4][j] = (double)(x[e] >= 0.0f ? 0.0f : x[e]);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t t = 0; t < count; ++t) {
      using Sum = std::conditional_t<kRows == 4, double, f64x4>;
      Sum over{}, under{};
      auto product = [](double a, double b, Sum c) {
        if constexpr (kRows == 4) return __builtin_amdgcn_mfma_f64_4x4x4f64(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
      };
      const int32_t after = page_of(t + 2);
      auto products = [&](int sign, Sum sum) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const u32x4 words = *reinterpret_cast<const u32x4 *>(held[wave] + lane % 16 * kRow + (4 * c + quarter) * 16);
          const double(*q)[2][4][kRows] = signs + part * (kMine / 4) + 8 * c;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            sum = product((double)bf16_lo(words[w]), q[2 * w][sign][quarter][lane % kRows], sum);
            sum = product((double)bf16_hi(words[w]), q[2 * w + 1][sign][quarter][lane % kRows], sum);
          }
        }
        return sum;
      };
      put(low);
      if (t + 1 < count) {
        places(next);
        ask(low, 0);
      }
      under = products(1, under);
      put(high);
      if (t + 1 < count) ask(high, p.b_side);
      over = products(0, over);
      double sum[kItems];
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if constexpr (kRows == 4) sum[i] = over + under;
        else sum[i] = over[i] + under[i];
      }
      const uint32_t there = (uint32_t)__ballot((uint32_t)page < p.pages) & 0xFFFFu, tile_first = first + 16 * (kWaves / kParts) * t;
      const int32_t mine = page;
      page = next, next = after;
      if constexpr (kParts == 2) {
        if (part == 1) {
#pragma unroll
          for (int i = 0; i < kItems; ++i) joined[t % 2][tile_wave][i][lane] = sum[i];
        }
        __syncthreads();
        if (part == 1) continue;
#pragma unroll
        for (int i = 0; i < kItems; ++i) sum[i] += joined[t % 2][tile_wave][i][lane];
      }
      // an item is page 4 (lane % 16 / 4) + lane / 16 of the tile, or, of 16 rows, 4 item + lane / 16
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const uint32_t which = kRows == 4 ? lane % 16 / 4 * 4 + quarter : 4 * i + quarter;
        uint32_t most = ordered((float)sum[i]);
        most = max(most, (uint32_t)dpp_move<kDppSwap1>((int)most));
        most = max(most, (uint32_t)dpp_move<kDppSwap2>((int)most));
        if constexpr (kRows == 16) {
          most = max(most, (uint32_t)dpp_move<kDppHalfMirror>((int)most));
          most = max(most, (uint32_t)dpp_move<kDppRowMirror>((int)most));
        }
        if (((there >> which) & 1u) == 0) most = ordered(-INFINITY);
        uint64_t odd = __ballot(!(fabs(sum[i]) < (double)INFINITY) && ((there >> which) & 1u) != 0);
        while (odd != 0) {
          const int at = __builtin_ctzll(odd);
          const uint32_t odd_page = kRows == 4 ? (uint32_t)(at % 16 / 4 * 4 + at / 16) : (uint32_t)(4 * i + at / 16);
          odd &= ~((kRows == 4 ? 0xFull : 0xFFFFull) << (kRows == 4 ? at / 4 * 4 : at / 16 * 16));
          const uint32_t score = page_score<T>(p, s, query, bounds, sequence, head, __builtin_amdgcn_readlane(mine, (int)odd_page));
          if (which == odd_page) most = score;
        }
        const uint32_t column = tile_first + which;
        if (lane % kRows == 0 && ranked(p, s, column)) {
          uint32_t *to = scores + (uint64_t)line * p.columns + column;
          *to = group == 0 ? most : max(most, *to);  // (its own of the rows before)
        }
      }
    }
    if (kParts == 2) __syncthreads();  // the sums in LDS are read
  }
}

__device__ __forceinline__ uint32_t most_of_wave(uint32_t v) {
  v = max(v, (uint32_t)dpp_move<kDppSwap1>((int)v));
  v = max(v, (uint32_t)dpp_move<kDppSwap2>((int)v));
  v = max(v, (uint32_t)dpp_move<kDppHalfMirror>((int)v));
  v = max(v, (uint32_t)dpp_move<kDppRowMirror>((int)v));
  const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(rows[0], rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(halves[0], halves[1]);
}

// A block to a key head: the largest bound that `count` pages' scores are at or over, two bits at a time from where they differ until
// just so many are, then those over it and the first
// of those at it in order.  Pages that are always chosen count as over all scores.  kKeys: consecutive pages whose scores a thread keeps in
// registers, 0: any number, read again for every two bits.
constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / kWaveLanes;
template <int kKeys>
__global__ __launch_bounds__(kChooseThreads) void paged_choose(PagedSelectParams p, const int32_t *table, const int32_t *lengths,
                                                               const uint32_t *scores, int32_t *selected, int32_t *seen) {
  __shared__ uint32_t counts[16][3], ends[2];
  __shared__ uint32_t wave_more[kChooseWaves], wave_same[kChooseWaves];
  const uint32_t line = blockIdx.x, sequence = line / p.heads, thread = threadIdx.x, lane = thread % kWaveLanes, wave = thread / kWaveLanes;
  const SelectSpan s = select_span(p, lengths, sequence);
  const int32_t *pages = table + (int64_t)sequence * p.table_row;
  int32_t *out = selected + (uint64_t)line * p.count;
  const uint32_t kept = min(s.filled, p.count);
  if (thread == 0) seen[line] = (int32_t)(s.length - (s.filled - kept) * p.page.divisor);
  for (uint32_t i = kept + thread; i < p.count; i += kChooseThreads) out[i] = -1;
  if (s.filled <= p.count) {
    for (uint32_t i = thread; i < kept; i += kChooseThreads) out[i] = pages[i];
    return;
  }
  const uint32_t *mine = scores + (uint64_t)line * p.columns;
  auto key_of = [&](uint32_t i) { return i >= s.filled ? 0u : i == 0 || i >= s.newest ? 0xFFFFFFFFu : mine[i]; };
  uint32_t held[kKeys > 0 ? kKeys : 1];
  int32_t chosen[kKeys > 0 ? kKeys : 1];  // (asked for here, not one after another where they are written)
  const uint32_t each = kKeys > 0 ? (uint32_t)kKeys : (s.filled + kChooseThreads - 1) / kChooseThreads, first = thread * each;
#pragma unroll
  for (int k = 0; k < kKeys; ++k) {
    held[k] = key_of(first + k);
    chosen[k] = pages[min(first + k, s.filled - 1)];
  }
  if (thread < 48) counts[thread / 3][thread % 3] = 0;
  if (thread == 0) ends[0] = 0, ends[1] = 0xFFFFFFFFu;
  __syncthreads();
  // what all ranked scores begin with
  {
    uint32_t most = 0, least = 0xFFFFFFFFu;
    auto look = [&](uint32_t key) {
      if (key != 0 && key != 0xFFFFFFFFu) most = max(most, key), least = min(least, key);
    };
    if constexpr (kKeys > 0) {
#pragma unroll
      for (int k = 0; k < kKeys; ++k) look(held[k]);
    } else {
      for (uint32_t k = 0; k < each; ++k) look(key_of(first + k));
    }
    most = most_of_wave(most), least = ~most_of_wave(~least);
    if (lane == 0) atomicMax(&ends[0], most), atomicMin(&ends[1], least);
  }
  __syncthreads();
  const uint32_t differs = ends[0] > ends[1] ? ends[0] ^ ends[1] : 0u;
  const int from = differs == 0 ? -2 : (31 - __clz((int)differs)) / 2 * 2;
  uint32_t bound = ends[0] & (differs == 0 ? 0xFFFFFFFFu : from >= 30 ? 0u : 0xFFFFFFFCu << from);
  if (1 + s.filled - max(s.newest, 1u) >= p.count) bound = 0xFFFFFFFFu;  // (none of the ranked)
  for (int shift = bound == 0xFFFFFFFFu ? -2 : from; shift >= 0; shift -= 2) {
    const int step = 15 - shift / 2;
    uint32_t over[3] = {0, 0, 0};
    auto look = [&](uint32_t key) {
#pragma unroll
      for (uint32_t d = 0; d < 3; ++d) over[d] += (uint32_t)__popcll(__ballot(key >= (bound | (d + 1) << shift)));
    };
    if constexpr (kKeys > 0) {
#pragma unroll
      for (int k = 0; k < kKeys; ++k) look(held[k]);
    } else {
      for (uint32_t i = thread; i < each * kChooseThreads; i += kChooseThreads) look(key_of(i));  // (every lane of a wave takes part)
    }
    if (lane < 3) atomicAdd(&counts[step][lane], lane == 0 ? over[0] : lane == 1 ? over[1] : over[2]);
    __syncthreads();
    const uint32_t digit = (counts[step][0] >= p.count) + (counts[step][1] >= p.count) + (counts[step][2] >= p.count);
    bound |= digit << shift;
    if (digit > 0 && counts[step][digit - 1] == p.count) break;  // just those
  }
  // those over the bound are fewer than count (it would be a larger one otherwise); of those at it the first are taken
  uint32_t more = 0, same = 0;
  auto count = [&](uint32_t key) { more += key > bound, same += key == bound; };
  if constexpr (kKeys > 0) {
#pragma unroll
    for (int k = 0; k < kKeys; ++k) count(held[k]);
  } else {
    for (uint32_t k = 0; k < each; ++k) count(key_of(first + k));
  }
  auto through = [&](uint32_t v) {
    uint32_t up;
    up = lane_up<1>(v), v += lane >= 1 ? up : 0u;
    up = lane_up<2>(v), v += lane >= 2 ? up : 0u;
    up = lane_up<4>(v), v += lane >= 4 ? up : 0u;
    up = lane_up<8>(v), v += lane >= 8 ? up : 0u;
    up = lane_up<16>(v), v += lane >= 16 ? up : 0u;
    up = lane_up<32>(v), v += lane >= 32 ? up : 0u;
    return v;
  };
  uint32_t more_before = through(more), same_before = through(same);
  if (lane == kWaveLanes - 1) wave_more[wave] = more_before, wave_same[wave] = same_before;
  more_before -= more, same_before -= same;
  __syncthreads();
  uint32_t all_more = 0;
  for (uint32_t w = 0; w < kChooseWaves; ++w) {
    if (w < wave) more_before += wave_more[w], same_before += wave_same[w];
    all_more += wave_more[w];
  }
  const uint32_t left = p.count - all_more;
  auto write = [&](uint32_t key, int32_t page) {
    if (key > bound || (key == bound && same_before < left)) out[more_before + min(same_before, left)] = page;
    more_before += key > bound, same_before += key == bound;
  };
  if constexpr (kKeys > 0) {
#pragma unroll
    for (int k = 0; k < kKeys; ++k) write(held[k], chosen[k]);
  } else {
    for (uint32_t k = 0; k < each; ++k) {
      const uint32_t key = key_of(first + k);
      write(key, key >= bound ? pages[first + k] : -1);
    }
  }
}

}  // namespace

struct PagedScoresTag {
  static std::string text() { return "paged_scores/channels"; }
};
template <int kDepth, int kRows> struct PagedScoresTilesTag {
  static std::string text() { return "paged_scores/tiles-d" + std::to_string(kDepth) + "/" + std::to_string(kRows) + "-rows"; }
};
template <int kKeys> struct PagedChooseTag {
  static std::string text() { return "paged_choose/" + (kKeys > 0 ? std::to_string(kKeys) : std::string("any")); }
};

namespace {
struct SelectBuffers {
  const unsigned char *query, *bounds;
  const int32_t *table, *lengths;
  uint32_t *scores;
};
template <class T, int kDepth, int kRows>
void start_tiles(const PagedSelectParams &p, const SelectBuffers &b, int compute_units, hipStream_t stream) {
  note_variant<PagedScoresTilesTag<kDepth, kRows>>();
  // so many tiles to a wave that the blocks are two rounds of what the device holds (one and three: the same within 3 %)
  constexpr uint32_t kColumns = kBlockThreads / kWaveLanes / (kDepth == 256 ? 2 : 1) * 16;
  const uint64_t lines = (uint64_t)p.sequences * p.heads, most = (p.columns + kColumns - 1) / kColumns;
  const uint64_t wanted = 2 * (kRows == 4 ? 4 : 2) * (uint64_t)compute_units;
  const uint32_t tiles = (uint32_t)std::max<uint64_t>(1, std::min(most, lines * most / wanted));
  const uint32_t blocks = ((uint32_t)most + tiles - 1) / tiles;
  hipLaunchKernelGGL((paged_scores_tiles<T, kDepth, kRows>), dim3((uint32_t)lines * blocks), dim3(kBlockThreads), 0, stream, p, Divisor(blocks * p.heads), tiles,
                     b.query, b.bounds, b.table, b.lengths, b.scores);
}
template <class T, int kDepth> void tiles_by_rows(const PagedSelectParams &p, const SelectBuffers &b, int compute_units, hipStream_t stream) {
  if ((uint64_t)p.rows * p.shared.divisor <= 8) start_tiles<T, kDepth, 4>(p, b, compute_units, stream);
  else start_tiles<T, kDepth, 16>(p, b, compute_units, stream);
}
template <class T> void start_scores(const PagedSelectParams &p, const SelectBuffers &b, bool vectors, int compute_units, hipStream_t stream) {
  if (vectors) {
    if (p.depth <= 64) tiles_by_rows<T, 64>(p, b, compute_units, stream);
    else if (p.depth <= 128) tiles_by_rows<T, 128>(p, b, compute_units, stream);
    else tiles_by_rows<T, 256>(p, b, compute_units, stream);
    return;
  }
  const uint64_t units = (uint64_t)p.sequences * p.heads * p.columns;
  constexpr uint32_t kWaves = kBlockThreads / kWaveLanes;
  note_variant<PagedScoresTag>();
  hipLaunchKernelGGL((paged_scores<T>), dim3((uint32_t)((units + kWaves - 1) / kWaves)), dim3(kBlockThreads), 0, stream, p, b.query, b.bounds, b.table,
                     b.lengths, b.scores);
}
template <int kKeys>
void start_choose(const PagedSelectParams &p, const SelectBuffers &b, int32_t *selected, int32_t *seen, hipStream_t stream) {
  note_variant<PagedChooseTag<kKeys>>();
  hipLaunchKernelGGL((paged_choose<kKeys>), dim3(p.sequences * p.heads), dim3(kChooseThreads), 0, stream, p, b.table, b.lengths, b.scores, selected, seen);
}
}  // namespace

hipError_t launch_paged_select(Elem type, const PagedSelectParams &p, const void *query, const void *bounds, const int32_t *table,
                               const int32_t *lengths, int32_t *selected, int32_t *seen, void *workspace, bool vector_aligned,
                               int compute_units, hipStream_t stream) {
  const SelectBuffers b{static_cast<const unsigned char *>(query), static_cast<const unsigned char *>(bounds), table, lengths, static_cast<uint32_t *>(workspace)};
  if (p.columns > p.count) {
    // (lanes without a page read the first one's bounds, so there has to be one)
    const bool vectors = vector_aligned && p.pages != 0 && p.depth % 8 == 0 && (p.q_sequence | p.q_row | p.q_head | p.b_page | p.b_side | p.b_head) % 16 == 0;
    switch (type) {
      case Elem::kF32: start_scores<F32>(p, b, vectors, compute_units, stream); break;
      case Elem::kF16: start_scores<F16>(p, b, vectors, compute_units, stream); break;
      case Elem::kBF16: start_scores<BF16>(p, b, vectors, compute_units, stream); break;
    }
  }
  if (p.columns <= 4 * kChooseThreads) start_choose<4>(p, b, selected, seen, stream);
  else if (p.columns <= 16 * kChooseThreads) start_choose<16>(p, b, selected, seen, stream);
  else start_choose<0>(p, b, selected, seen, stream);
  return hipGetLastError();
}

}  // namespace hyle_hip
