// paged_select.hip -- the pages of each sequence that a query's products can be largest in, for every key head.
//
// score of a page = max over the key head's query heads and the new rows of sum_d q_d (q_d >= 0 ? high_d : low_d)
// which no key of the page passes.  Sums are kept in 64 bits and rounded once to f32, so that the order of pages does not depend on
// the order of additions; the products of f16 and bf16 numbers are exact.  A score that is no number counts as the largest.  The
// first page and those of the newest tokens are always chosen, then the best, ties to the earlier, and written in their order.
// Two launches: scores to the workspace, and one block to a key head that finds the last chosen score digit by digit.
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

// A wave to a page and key head, a lane to every 64th channel.
template <class T>
__global__ __launch_bounds__(kBlockThreads) void paged_scores(PagedSelectParams p, const unsigned char *query, const unsigned char *bounds,
                                                              const int32_t *table, const int32_t *lengths, uint32_t *scores) {
  const uint32_t lane = threadIdx.x % kWaveLanes;
  const uint64_t unit = (uint64_t)blockIdx.x * (kBlockThreads / kWaveLanes) + threadIdx.x / kWaveLanes;
  const uint32_t column = (uint32_t)(unit % p.columns);
  const uint64_t line = unit / p.columns;  // sequence and key head
  if (line >= (uint64_t)p.sequences * p.heads) return;
  const uint32_t sequence = (uint32_t)(line / p.heads), head = (uint32_t)(line - (uint64_t)sequence * p.heads);
  const SelectSpan s = select_span(p, lengths, sequence);
  if (!ranked(p, s, column)) return;
  const int32_t page = table[(int64_t)sequence * p.table_row + column];
  uint32_t best = ordered(-INFINITY);
  if ((uint32_t)page < p.pages) {
    const unsigned char *low = bounds + page * p.b_page + head * p.b_head, *high = low + p.b_side;
    for (uint32_t r = s.rows_before; r < p.rows; ++r)
      for (uint32_t h = 0; h < p.shared.divisor; ++h) {
        const unsigned char *q = query + sequence * p.q_sequence + r * p.q_row + (head * p.shared.divisor + h) * p.q_head;
        double sum = 0.0;
        for (uint32_t d = lane; d < p.depth; d += kWaveLanes) {
          const float x = Traits<T>::load(q, d);
          sum += (double)x * (double)Traits<BF16>::load(x >= 0.0f ? high : low, d);
        }
        best = max(best, ordered((float)wave_sum(sum)));
      }
  }
  if (lane == 0) scores[unit] = best;
}

constexpr int kChooseThreads = 1024;
__global__ __launch_bounds__(kChooseThreads) void paged_choose(PagedSelectParams p, const int32_t *table, const int32_t *lengths,
                                                               const uint32_t *scores, int32_t *selected, int32_t *seen) {
  __shared__ uint32_t counts[256];
  __shared__ uint32_t chosen_digit, chosen_left;
  __shared__ uint32_t wave_more[kChooseThreads / kWaveLanes], wave_same[kChooseThreads / kWaveLanes];
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
  // ranked columns are [1, newest); the first page and those from `newest` on are chosen: fewer than count, by the plan
  const uint32_t first = 1, last = max(s.newest, 1u), always = 1 + (s.filled - last);
  uint32_t left = p.count - always, bound = 0, mask = 0;  // of the ranked: those to choose, the last one's score so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (thread < 256) counts[thread] = 0;
    __syncthreads();
    for (uint32_t i = first + thread; i < last; i += kChooseThreads) {
      const uint32_t key = mine[i];
      if ((key & mask) == bound) atomicAdd(&counts[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (thread == 0) {
      uint32_t digit = 255, more = 0;
      while (digit > 0 && more + counts[digit] < left) more += counts[digit--];
      chosen_digit = digit, chosen_left = left - min(left, more);
    }
    __syncthreads();
    bound |= chosen_digit << shift, mask |= 255u << shift, left = chosen_left;
    __syncthreads();
  }
  // those over the bound, and of those at it the first `left`, in order
  if (thread == 0) out[0] = pages[0];
  uint32_t at = 1, same_before = 0;
  for (uint32_t base = first; base < last; base += kChooseThreads) {
    const uint32_t i = base + thread, key = i < last ? mine[i] : 0u;
    const bool more = i < last && key > bound, same = i < last && key == bound;
    const uint64_t more_lanes = __ballot(more), same_lanes = __ballot(same), below = (1ull << lane) - 1;
    if (lane == 0) wave_more[wave] = __popcll(more_lanes), wave_same[wave] = __popcll(same_lanes);
    __syncthreads();
    uint32_t more_before = 0, same_here = same_before, all_more = 0, all_same = 0;
    for (uint32_t w = 0; w < kChooseThreads / kWaveLanes; ++w) {
      if (w < wave) more_before += wave_more[w], same_here += wave_same[w];
      all_more += wave_more[w], all_same += wave_same[w];
    }
    more_before += __popcll(more_lanes & below), same_here += __popcll(same_lanes & below);
    // chosen before this one: those over the bound, and of those at it what is left
    const uint32_t place = at + more_before + (min(same_here, left) - min(same_before, left));
    if (more || (same && same_here < left)) out[place] = pages[i];
    at += all_more + (min(same_before + all_same, left) - min(same_before, left));
    same_before += all_same;
    __syncthreads();
  }
  for (uint32_t i = last + thread; i < s.filled; i += kChooseThreads) out[at + (i - last)] = pages[i];
}

}  // namespace

struct PagedScoresTag {
  static std::string text() { return "paged_scores/channels"; }
};
struct PagedChooseTag {
  static std::string text() { return "paged_choose"; }
};

hipError_t launch_paged_select(Elem type, const PagedSelectParams &p, const void *query, const void *bounds, const int32_t *table,
                               const int32_t *lengths, int32_t *selected, int32_t *seen, void *workspace, bool vector_aligned,
                               hipStream_t stream) {
  uint32_t *scores = static_cast<uint32_t *>(workspace);
  if (p.columns > p.count) {
    const uint64_t units = (uint64_t)p.sequences * p.heads * p.columns;
    constexpr uint32_t kWaves = kBlockThreads / kWaveLanes;
    auto typed = [&](auto tag) {
      using T = decltype(tag);
      note_variant<PagedScoresTag>();
      hipLaunchKernelGGL((paged_scores<T>), dim3((uint32_t)((units + kWaves - 1) / kWaves)), dim3(kBlockThreads), 0, stream, p,
                         static_cast<const unsigned char *>(query), static_cast<const unsigned char *>(bounds), table, lengths, scores);
    };
    switch (type) {
      case Elem::kF32: typed(F32{}); break;
      case Elem::kF16: typed(F16{}); break;
      case Elem::kBF16: typed(BF16{}); break;
    }
  }
  note_variant<PagedChooseTag>();
  hipLaunchKernelGGL(paged_choose, dim3(p.sequences * p.heads), dim3(kChooseThreads), 0, stream, p, table, lengths, scores, selected, seen);
  return hipGetLastError();
}

}  // namespace hyle_hip
