// page_bounds.hip -- the least and largest key of every channel of a cache's pages, [pages, 2, heads, depth] in bf16: what a page's
// products with a query cannot pass (PagedSelect's score).
//
// A number that bf16 does not have goes to the next one below or above, so the bounds stay bounds; elements that are no numbers have
// no part.  Of each sequence the pages that hold its newest tokens are written, from the keys that it has there.
//
// 5 sequences of 9001 to 32768 keys, 8 key heads of 128 in e4m3, pages of 64, 118 MB: 24.8 us, 4.8 TB/s (the same with two, four and eight loads
// ahead; 38.7 with a block to a page, a thread to a channel 147).  Bound by memory and the waves' own work, which overlap only
// between waves (one asks for its vectors, folds them, asks again, and ends): of 103 MB in such pages, 22.7 us, a plain read of the same runs takes 16.3 (6.3
// TB/s, in any order of pages and with or without the values between them) and the kernel over one page again and again 14.1 (in bf16
// 39.4 and 27.8, in 4 bits 22.6 and 18.5).  The page that each of 64 streams wrote to, 16 keys of 8 heads in bf16: 3.2 us, a launch.
#include <algorithm>

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

// By whole vectors: kWaves waves to a page and key head, a lane to the same vector of every row that it reads; rows past the last key
// read it again.  Lanes that hold the same channels of different rows meet at the end: halves and rows of sixteen lanes trade half of their
// channels each, so that every lane goes on with fewer.
template <class C> constexpr int kElements = std::is_same<C, MX4>::value ? 32 : std::is_same<C, E4M3>::value ? 16 : std::is_same<C, F32>::value ? 4 : 8;
template <class C, int kDepth, int kWaves>
__global__ __launch_bounds__(kBlockThreads) void page_bounds_vectors(PageBoundsParams p, const unsigned char *cache, const int32_t *table,
                                                                     const int32_t *lengths, unsigned char *bounds) {
  constexpr int E = kElements<C>, kVectors = kDepth / E, kRows = kWaveLanes / kVectors, kAhead = 4, kBlockWaves = kBlockThreads / kWaveLanes;
  constexpr bool kFour = std::is_same<C, MX4>::value;
  const uint32_t lane = threadIdx.x % kWaveLanes, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWaveLanes));
  const uint32_t unit = kWaves == 1 ? blockIdx.x * kBlockWaves + wave : blockIdx.x, block = unit / p.heads, head = unit - block * p.heads;
  if (block >= p.sequences * p.span) return;  // (kWaves == 1: the last block's)
  BoundsPage found;
  if (!bounds_page(p, table, lengths, block, &found)) return;
  const unsigned char *from = cache + found.page * p.page_bytes + head * p.head_bytes;
  const uint32_t vectors = p.depth / E, own = lane % kVectors, vector = own < vectors ? own : 0u;  // (lanes past the depth write nothing)
  float low[E], high[E];
#pragma unroll
  for (int e = 0; e < E; ++e) low[e] = INFINITY, high[e] = -INFINITY;
  for (uint32_t first = kWaves == 1 ? 0u : wave * (kRows * kAhead); first < found.keys; first += kWaves * kRows * kAhead) {
    u32x4 words[kAhead];
    uint32_t scales[kFour ? kAhead : 1];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t row = min(first + k * kRows + lane / kVectors, found.keys - 1);
      const unsigned char *at = from + (int64_t)row * p.row_bytes;
      if constexpr (kFour) {
        words[k] = load16_words(at, vector);
        scales[k] = from[p.scale_offset + (int64_t)row * (p.row_bytes / 16) + vector];
      } else {
        words[k] = load16_stream(at, vector);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float x[E];
      if constexpr (kFour) {
        const float scale = bits_f32(scales[k] << 23);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(words[k][w], scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(words[k][w], scale, 1);
          const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(words[k][w], scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(words[k][w], scale, 3);
          x[8 * w] = a[0], x[8 * w + 1] = a[1], x[8 * w + 2] = b[0], x[8 * w + 3] = b[1];
          x[8 * w + 4] = c[0], x[8 * w + 5] = c[1], x[8 * w + 6] = d[0], x[8 * w + 7] = d[1];
        }
      } else if constexpr (std::is_same<C, E4M3>::value) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)words[k][w], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)words[k][w], true);
          x[4 * w] = a[0], x[4 * w + 1] = a[1], x[4 * w + 2] = b[0], x[4 * w + 3] = b[1];
        }
      } else {
        Traits<C>::unpack(words[k], x);
        if constexpr (!std::is_same<C, F16>::value) {  // (a signaling NaN would take the minimum's place; f16's are quiet after conversion)
#pragma unroll
          for (int e = 0; e < E; ++e) x[e] = __builtin_canonicalizef(x[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) low[e] = fminf(low[e], x[e]), high[e] = fmaxf(high[e], x[e]);  // (NaN has no part)
    }
  }
  constexpr int kHalved = kVectors <= 32 ? E / 2 : E, kKept = kVectors <= 16 ? kHalved / 2 : kHalved;
  uint32_t channel = own * E;
  if constexpr (kVectors <= 32) {
    channel += lane >= 32 ? kHalved : 0;
#pragma unroll
    for (int e = 0; e < kHalved; ++e) {
      const auto l = __builtin_amdgcn_permlane32_swap(f32_bits(low[e]), f32_bits(low[e + kHalved]), false, false);
      const auto h = __builtin_amdgcn_permlane32_swap(f32_bits(high[e]), f32_bits(high[e + kHalved]), false, false);
      low[e] = fminf(bits_f32(l[0]), bits_f32(l[1])), high[e] = fmaxf(bits_f32(h[0]), bits_f32(h[1]));
    }
  }
  if constexpr (kVectors <= 16) {
    channel += (lane & 16) != 0 ? kKept : 0;
#pragma unroll
    for (int e = 0; e < kKept; ++e) {
      const auto l = __builtin_amdgcn_permlane16_swap(f32_bits(low[e]), f32_bits(low[e + kKept]), false, false);
      const auto h = __builtin_amdgcn_permlane16_swap(f32_bits(high[e]), f32_bits(high[e + kKept]), false, false);
      low[e] = fminf(bits_f32(l[0]), bits_f32(l[1])), high[e] = fmaxf(bits_f32(h[0]), bits_f32(h[1]));
    }
  }
#pragma unroll
  for (int e = 0; e < kKept; ++e) {  // within rows of sixteen by turning them
    if constexpr (kVectors <= 8) low[e] = fminf(low[e], dpp_move<0x128>(low[e])), high[e] = fmaxf(high[e], dpp_move<0x128>(high[e]));
    if constexpr (kVectors <= 4) low[e] = fminf(low[e], dpp_move<0x124>(low[e])), high[e] = fmaxf(high[e], dpp_move<0x124>(high[e]));
    if constexpr (kVectors <= 2) low[e] = fminf(low[e], dpp_move<0x122>(low[e])), high[e] = fmaxf(high[e], dpp_move<0x122>(high[e]));
  }
  const bool writes = own < vectors && lane % 16 / kVectors == 0;
  if constexpr (kWaves > 1) {
    __shared__ float joined[kWaves][2][kDepth];
    if (writes) {
#pragma unroll
      for (int e = 0; e < kKept; ++e) joined[wave][0][channel + e] = low[e], joined[wave][1][channel + e] = high[e];
    }
    __syncthreads();
    uint16_t *to = reinterpret_cast<uint16_t *>(bounds) + ((uint64_t)found.page * 2 * p.heads + head) * p.depth;
    for (uint32_t i = threadIdx.x; i < 2 * kDepth; i += kBlockThreads) {
      const uint32_t side = i / kDepth, d = i % kDepth;
      if (d >= p.depth) continue;
      float edge = joined[0][side][d];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) edge = side == 0 ? fminf(edge, joined[w][0][d]) : fmaxf(edge, joined[w][1][d]);
      to[(uint64_t)side * p.heads * p.depth + d] = side == 0 ? bf16_below(edge) : bf16_above(edge);
    }
  } else if (writes) {
    uint16_t *low_to = reinterpret_cast<uint16_t *>(bounds) + ((uint64_t)found.page * 2 * p.heads + head) * p.depth + channel;
    uint16_t *high_to = low_to + (uint64_t)p.heads * p.depth;
    typedef uint16_t Kept __attribute__((ext_vector_type(kKept)));
    Kept l, h;
#pragma unroll
    for (int e = 0; e < kKept; ++e) l[e] = bf16_below(low[e]), h[e] = bf16_above(high[e]);
    *reinterpret_cast<Kept *>(low_to) = l;
    *reinterpret_cast<Kept *>(high_to) = h;
  }
}

}  // namespace

template <class C> static const char *bounds_type() {
  return std::is_same<C, MX4>::value ? "mx4" : std::is_same<C, E4M3>::value ? "e4m3" : std::is_same<C, F32>::value ? "f32" : std::is_same<C, F16>::value ? "f16" : "bf16";
}
template <class C> struct BoundsChannelsTag {
  static std::string text() { return std::string("page_bounds_channels/") + bounds_type<C>(); }
};
template <class C, int kDepth, int kWaves> struct BoundsVectorsTag {
  static std::string text() { return std::string("page_bounds_vectors/") + bounds_type<C>() + "/d" + std::to_string(kDepth) + (kWaves == 1 ? "/wave" : "/block"); }
};

template <class C, int kDepth>
static void start_vectors(const PageBoundsParams &p, const unsigned char *cache, const int32_t *table, const int32_t *lengths, void *bounds, hipStream_t stream) {
  constexpr uint32_t kRows = kWaveLanes / (kDepth / kElements<C>);
  const uint32_t units = p.sequences * p.span * p.heads;
  // (a wave's loads one after another: 16 steps of a page are shared by four)
  if (p.page.divisor >= 16 * kRows) {
    note_variant<BoundsVectorsTag<C, kDepth, 4>>();
    hipLaunchKernelGGL((page_bounds_vectors<C, kDepth, 4>), dim3(units), dim3(kBlockThreads), 0, stream, p, cache, table, lengths, static_cast<unsigned char *>(bounds));
  } else {
    note_variant<BoundsVectorsTag<C, kDepth, 1>>();
    hipLaunchKernelGGL((page_bounds_vectors<C, kDepth, 1>), dim3((units + 3) / 4), dim3(kBlockThreads), 0, stream, p, cache, table, lengths, static_cast<unsigned char *>(bounds));
  }
}

hipError_t launch_page_bounds(const PageBoundsParams &p, const void *cache, const int32_t *table, const int32_t *lengths, void *bounds,
                              hipStream_t stream) {
  const unsigned char *from = static_cast<const unsigned char *>(cache);
  const bool aligned16 = reinterpret_cast<uintptr_t>(bounds) % 16 == 0;
  auto typed = [&](auto tag) {
    using C = decltype(tag);
    const uintptr_t places = reinterpret_cast<uintptr_t>(cache) | (uintptr_t)p.page_bytes | (uintptr_t)p.head_bytes | (uintptr_t)p.row_bytes;
    const bool vectors = aligned16 && p.depth % std::max(kElements<C>, 8) == 0 && p.depth <= 256 &&
                         (std::is_same<C, MX4>::value ? (places % 4 == 0) : (places % 16 == 0));
    if (!vectors) {
      note_variant<BoundsChannelsTag<C>>();
      hipLaunchKernelGGL((page_bounds_channels<C>), dim3(p.sequences * p.span * p.heads), dim3(kBlockThreads), 0, stream, p, from, table, lengths,
                         static_cast<uint16_t *>(bounds));
    } else if (p.depth <= 64) {
      start_vectors<C, 64>(p, from, table, lengths, bounds, stream);
    } else if (p.depth <= 128) {
      start_vectors<C, 128>(p, from, table, lengths, bounds, stream);
    } else {
      start_vectors<C, 256>(p, from, table, lengths, bounds, stream);
    }
  };
  if (p.cache == CacheKind::kFourBits) typed(MX4{});
  else if (p.cache == CacheKind::kNarrow) typed(E4M3{});
  else if (p.type == Elem::kF32) typed(F32{});
  else if (p.type == Elem::kF16) typed(F16{});
  else typed(BF16{});
  return hipGetLastError();
}

}  // namespace hyle_hip
