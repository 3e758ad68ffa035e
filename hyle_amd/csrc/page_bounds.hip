// page_bounds.hip -- the least and largest key of every channel of a cache's pages, [pages, 2, heads, depth] in bf16: what a page's
// products with a query cannot pass (PagedSelect's score).
//
// A number that bf16 does not have goes to the next one below or above, so the bounds stay bounds; elements that are no numbers have
// no part.  Of each sequence the pages that hold its newest tokens are written, from the keys that it has there.
#include "cache_types.h"

namespace hyle_hip {
namespace {

__device__ __forceinline__ uint16_t bf16_below(float x) {
  const uint32_t bits = f32_bits(x);
  return (uint16_t)((((bits & 0x80000000u) != 0 ? bits + 0xFFFFu : bits)) >> 16);
}
__device__ __forceinline__ uint16_t bf16_above(float x) {
  const uint32_t bits = f32_bits(x);
  return (uint16_t)((((bits & 0x80000000u) != 0 ? bits : bits + 0xFFFFu)) >> 16);
}

// The keys of a sequence that lie in a block's page; false where there is nothing to write.
struct BoundsPage {
  int32_t page;
  uint32_t keys;
};
__device__ __forceinline__ bool bounds_page(const PageBoundsParams &p, const int32_t *table, const int32_t *lengths, uint32_t block, BoundsPage *found) {
  const uint32_t sequence = block / p.span, step = block - sequence * p.span;
  const uint32_t length = (uint32_t)max(lengths[sequence], 0);
  const uint32_t since = p.newest != 0 && length > p.newest ? length - p.newest : 0u;
  const uint64_t column = (uint64_t)p.page.quotient(since) + step, first = column * p.page.divisor;
  if (first >= length || column >= p.columns) return false;
  found->page = table[(int64_t)sequence * p.table_row + (int64_t)column];
  found->keys = min(length - (uint32_t)first, p.page.divisor);
  return (uint32_t)found->page < p.pages;
}

// A thread to a channel, any type and alignment.
template <class C>
__global__ __launch_bounds__(kBlockThreads) void page_bounds_channels(PageBoundsParams p, const unsigned char *cache, const int32_t *table,
                                                                      const int32_t *lengths, uint16_t *bounds) {
  const uint32_t block = blockIdx.x / p.heads, head = blockIdx.x - block * p.heads;
  BoundsPage found;
  if (!bounds_page(p, table, lengths, block, &found)) return;
  const unsigned char *from = cache + found.page * p.page_bytes + head * p.head_bytes;
  uint16_t *low_to = bounds + ((uint64_t)found.page * 2 * p.heads + head) * p.depth, *high_to = low_to + (uint64_t)p.heads * p.depth;
  for (uint32_t d = threadIdx.x; d < p.depth; d += kBlockThreads) {
    float low = INFINITY, high = -INFINITY;
    for (uint32_t r = 0; r < found.keys; ++r) {
      float x;
      if constexpr (std::is_same<C, MX4>::value) x = mx4_element(from + r * p.row_bytes, from + p.scale_offset + r * (p.row_bytes / 16), (int)d);
      else x = Traits<C>::load(from + r * p.row_bytes, d);
      low = x < low ? x : low, high = x > high ? x : high;
    }
    low_to[d] = bf16_below(low);
    high_to[d] = bf16_above(high);
  }
}

}  // namespace

template <class C> struct BoundsChannelsTag {
  static std::string text() {
    return std::string("page_bounds_channels/") + (std::is_same<C, MX4>::value ? "mx4" : std::is_same<C, E4M3>::value ? "e4m3" :
                                                    std::is_same<C, F32>::value ? "f32" : std::is_same<C, F16>::value ? "f16" : "bf16");
  }
};

hipError_t launch_page_bounds(const PageBoundsParams &p, const void *cache, const int32_t *table, const int32_t *lengths, void *bounds,
                              bool vector_aligned, hipStream_t stream) {
  auto typed = [&](auto tag) {
    using C = decltype(tag);
    note_variant<BoundsChannelsTag<C>>();
    hipLaunchKernelGGL((page_bounds_channels<C>), dim3(p.sequences * p.span * p.heads), dim3(kBlockThreads), 0, stream, p,
                       static_cast<const unsigned char *>(cache), table, lengths, static_cast<uint16_t *>(bounds));
  };
  if (p.cache == CacheKind::kFourBits) typed(MX4{});
  else if (p.cache == CacheKind::kNarrow) typed(E4M3{});
  else if (p.type == Elem::kF32) typed(F32{});
  else if (p.type == Elem::kF16) typed(F16{});
  else typed(BF16{});
  return hipGetLastError();
}

}  // namespace hyle_hip
