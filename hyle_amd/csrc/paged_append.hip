// paged_append.hip -- keys and values of new tokens to their slots of a paged cache [pages, 2, heads, page, depth].
//
// A thread moves eight elements of a head (16 bytes of f16 / bf16), sixteen for a cache of e4m3 where the depth allows, or, where
// a row is not made of whole aligned vectors, one; into 4 bits eight, four threads to a scale, or all 32 of a scale.  Bound by bytes: every element is read once and written once (8192 tokens of 8
// heads of 128, bf16 to e4m3, 50 MB: 11.2 us, 4.5 TB/s where a large copy reaches 4.9; eight elements to a thread 14.1; to 4 bits,
// 42 MB, 11.8, 3.6 TB/s; 64 tokens kept as bf16, 3.2 us, a launch; 1037 to 4 bits 3.1).
// Threads, and so the vectors of a token, are in no order: a slot of several tokens holds a mix of their vectors (700 tokens of 8
// heads of 128 to one slot: 97 of 100 launches).  To have one token win, each block would look through the tokens after its own:
// 8192 tokens 14.9 us instead of 11.2, 65536 of one head 55 instead of 7; slots are a server's own and differ.
#include "cache_types.h"

namespace hyle_hip {
namespace {

struct AppendLayout {
  uint32_t units;      // of a token: 2 sides x heads x units of a head
  Divisor unit, head;  // by units of a token, by units of a head
  Divisor page;
  uint32_t heads, slots;
  uint64_t total;
  int64_t k_token, k_head, v_token, v_head;
  uint32_t depth;
};

// kElements: of a thread; in 4 bits eight are a lane's share of a scale's block, 32 the block read element by element
template <class T, CacheKind kKind, int kElements>
__global__ __launch_bounds__(kBlockThreads) void paged_append(AppendLayout p, const unsigned char *keys, const unsigned char *values,
                                                              const int32_t *slots, unsigned char *cache) {
  const uint64_t i = (uint64_t)blockIdx.x * kBlockThreads + threadIdx.x;
  if (i >= p.total) return;
  const uint32_t token = p.unit.quotient((uint32_t)i), rest = (uint32_t)i - token * p.units;
  const uint32_t row = p.head.quotient(rest), unit = rest - row * p.head.divisor;  // row: side * heads + head
  const uint32_t slot = (uint32_t)slots[token];
  if (slot >= p.slots) return;
  const bool value = row >= p.heads;
  const uint32_t head = value ? row - p.heads : row;
  const unsigned char *from = (value ? values : keys) + (int64_t)token * (value ? p.v_token : p.k_token) + (int64_t)head * (value ? p.v_head : p.k_head);
  const uint32_t page = p.page.quotient(slot), at = slot - page * p.page.divisor;
  constexpr bool kNarrow = kKind == CacheKind::kNarrow;
  if constexpr (kKind == CacheKind::kFourBits) {
    unsigned char *base = cache + ((uint64_t)page * 2 * p.heads + row) * (p.page.divisor * (uint64_t)(p.depth / kMx4Block * 17));
    unsigned char *codes = base + (uint64_t)at * (p.depth / 2) + (uint64_t)unit * (kElements / 2);
    unsigned char *scale = base + ((uint64_t)p.page.divisor * (p.depth / 2) + (uint64_t)at * (p.depth / kMx4Block)) + unit * kElements / kMx4Block;
    if constexpr (kElements == kMx4Block) {
      mx4_store_block<T>([&](int e) { return Traits<T>::load(from, (size_t)unit * kMx4Block + e); }, codes, scale);
    } else {
      float x[kElements];
#pragma unroll
      for (int v = 0; v < kElements / Traits<T>::kVec; ++v) {
        float part[Traits<T>::kVec];
        Traits<T>::unpack(load16_stream(from, (size_t)unit * (kElements / Traits<T>::kVec) + v), part);
#pragma unroll
        for (int e = 0; e < Traits<T>::kVec; ++e) x[v * Traits<T>::kVec + e] = part[e];
      }
      uint32_t byte;
      *reinterpret_cast<uint32_t *>(codes) = mx4_of_quad<T>(x, &byte);
      if (unit % 4 == 0) *scale = (unsigned char)byte;
    }
    return;
  }
  const uint64_t to = (((uint64_t)page * 2 * p.heads + row) * p.page.divisor + at) * p.depth + (uint64_t)unit * kElements;
  if constexpr (kKind == CacheKind::kFourBits) {
  } else if constexpr (kElements == 1) {
    const float x = Traits<T>::load(from, unit);
    if constexpr (kNarrow) cache[to] = (unsigned char)pack_e4m3(x, 0.0f, 0.0f, 0.0f);
    else if constexpr (Traits<T>::kSize == 4) reinterpret_cast<uint32_t *>(cache)[to] = reinterpret_cast<const uint32_t *>(from)[unit];
    else reinterpret_cast<uint16_t *>(cache)[to] = reinterpret_cast<const uint16_t *>(from)[unit];
  } else {
    constexpr int kVectors = kElements * Traits<T>::kSize / 16;
    u32x4 w[kVectors];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) w[v] = load16_stream(from, (size_t)unit * kVectors + v);
    if constexpr (kNarrow) {
      float x[kElements];
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        float part[Traits<T>::kVec];
        Traits<T>::unpack(w[v], part);
#pragma unroll
        for (int e = 0; e < Traits<T>::kVec; ++e) x[v * Traits<T>::kVec + e] = part[e];
      }
      uint32_t packed[kElements / 4];
#pragma unroll
      for (int e = 0; e < kElements / 4; ++e) packed[e] = pack_e4m3(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
      if constexpr (kElements == 16) store16(cache + to, 0, u32x4{packed[0], packed[1], packed[2], packed[3]});
      else *reinterpret_cast<uint2 *>(cache + to) = uint2{packed[0], packed[1]};
    } else {
#pragma unroll
      for (int v = 0; v < kVectors; ++v) store16(cache + to * Traits<T>::kSize, v, w[v]);
    }
  }
}

}  // namespace

template <CacheKind kKind, int kElements> struct AppendTag {
  static std::string text() {
    return std::string("paged_append/") + (kKind == CacheKind::kFourBits ? "mx4/" : kKind == CacheKind::kNarrow ? "e4m3/" : "kept/") + std::to_string(kElements);
  }
};

template <class T, CacheKind kKind, int kElements>
static void start(AppendLayout layout, const AppendParams &p, const void *keys, const void *values, const int32_t *slots, void *cache,
                  hipStream_t stream) {
  note_variant<AppendTag<kKind, kElements>>();
  const uint32_t units = p.depth / kElements;
  layout.units = 2 * p.heads * units;
  layout.unit = Divisor(layout.units);
  layout.head = Divisor(units);
  layout.total = (uint64_t)p.tokens * layout.units;
  hipLaunchKernelGGL((paged_append<T, kKind, kElements>), dim3((uint32_t)((layout.total + kBlockThreads - 1) / kBlockThreads)), dim3(kBlockThreads),
                     0, stream, layout, static_cast<const unsigned char *>(keys), static_cast<const unsigned char *>(values), slots,
                     static_cast<unsigned char *>(cache));
}

hipError_t launch_paged_append(Elem type, const AppendParams &p, const void *keys, const void *values, const int32_t *slots, void *cache,
                               bool vector_aligned, hipStream_t stream) {
  AppendLayout layout{};
  layout.page = p.page;
  layout.heads = p.heads;
  layout.depth = p.depth;
  layout.slots = p.pages * p.page.divisor;
  layout.k_token = p.k_token, layout.k_head = p.k_head, layout.v_token = p.v_token, layout.v_head = p.v_head;
  const bool vectors = vector_aligned && p.depth % 8 == 0 && (p.k_token | p.k_head | p.v_token | p.v_head) % 16 == 0;
  // (words of codes are written at addresses of whole words)
  const bool words = vectors && reinterpret_cast<uintptr_t>(cache) % 4 == 0 && p.page.divisor * (uint64_t)(p.depth / kMx4Block * 17) % 4 == 0;
  auto typed = [&](auto tag) {
    using T = decltype(tag);
    switch (p.cache) {
      case CacheKind::kKept:
        if (vectors) start<T, CacheKind::kKept, 8>(layout, p, keys, values, slots, cache, stream);
        else start<T, CacheKind::kKept, 1>(layout, p, keys, values, slots, cache, stream);
        break;
      case CacheKind::kNarrow:
        if (vectors && p.depth % 16 == 0) start<T, CacheKind::kNarrow, 16>(layout, p, keys, values, slots, cache, stream);
        else if (vectors) start<T, CacheKind::kNarrow, 8>(layout, p, keys, values, slots, cache, stream);
        else start<T, CacheKind::kNarrow, 1>(layout, p, keys, values, slots, cache, stream);
        break;
      case CacheKind::kFourBits:
        if (words) start<T, CacheKind::kFourBits, 8>(layout, p, keys, values, slots, cache, stream);
        else start<T, CacheKind::kFourBits, kMx4Block>(layout, p, keys, values, slots, cache, stream);
        break;
    }
  };
  switch (type) {
    case Elem::kF32: typed(F32{}); break;
    case Elem::kF16: typed(F16{}); break;
    case Elem::kBF16: typed(BF16{}); break;
  }
  return hipGetLastError();
}

}  // namespace hyle_hip
