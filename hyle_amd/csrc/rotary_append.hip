// rotary_append.hip -- the projected rows [tokens, queries + 2 heads, depth] of new tokens: queries and keys rotated by their positions, the
// queries to a tensor of their own, keys and values to their slots of a paged cache.
//
// The rotation is RoPE's (rope.hip): phase = frequency * position in f32, a' = a cos - b sin, b' = a sin + b cos with every product and sum
// rounded on its own.  cos and sin are those of the f32 phase in 64 bits, rounded to f32 once: they are then the nearest numbers, whoever
// computes them, and so is everything behind them, down to the codes of a cache in 4 bits.  A rotated element is rounded once, to what
// the cache keeps.
#include "cache_types.h"

namespace hyle_hip {
namespace {

constexpr int kWaves = kBlockThreads / kWaveLanes;
constexpr int kMostDepth = 1024;

struct Layout {
  RotaryAppendParams p;
  const unsigned char *projected;
  const void *positions;
  const float *frequencies;
  const int32_t *slots;
  unsigned char *cache, *rotated;
  uint32_t slot_count;
  uint64_t units;
};

__device__ __forceinline__ float position_of(const Layout &l, uint32_t token) {
  return l.p.wide_positions ? (float)static_cast<const int64_t *>(l.positions)[token] : (float)static_cast<const int32_t *>(l.positions)[token];
}
__device__ __forceinline__ void turn_of(const Layout &l, uint32_t token, uint32_t pair, float position, float *c, float *s) {
  const float phase = l.frequencies[(l.p.stepped_frequencies ? (uint64_t)token * (l.p.rotary / 2) : 0u) + pair] * position;
  double sine, cosine;
  sincos((double)phase, &sine, &cosine);
  *c = (float)cosine, *s = (float)sine;
}

// Any depth, rotary width and alignment: a wave to a row (one head of one token), rotated in LDS.
template <class T, CacheKind kKind>
__global__ __launch_bounds__(kBlockThreads) void rotary_append_rows(Layout l) {
  __shared__ float held[kWaves][kMostDepth];
  const RotaryAppendParams &p = l.p;
  const uint32_t wave = threadIdx.x / kWaveLanes, lane = threadIdx.x % kWaveLanes, rows = p.queries + 2 * p.heads;
  const uint64_t unit = (uint64_t)blockIdx.x * kWaves + wave;
  if (unit >= l.units) return;
  const uint32_t token = (uint32_t)(unit / rows), row = (uint32_t)(unit - (uint64_t)token * rows);
  const unsigned char *from = l.projected + (int64_t)token * p.token + (int64_t)row * p.head;
  const bool query = row < p.queries;
  const uint32_t slot = query ? 0u : (uint32_t)l.slots[token];
  if (!query && slot >= l.slot_count) return;
  const uint32_t rotary = row < p.queries + p.heads ? p.rotary : 0u, pairs = rotary / 2;
  float *to = held[wave];
  for (uint32_t i = lane; i < pairs; i += kWaveLanes) {
    const uint32_t first = p.half_split ? i : 2 * i, second = p.half_split ? i + pairs : 2 * i + 1;
    const float a = Traits<T>::load(from, first), b = Traits<T>::load(from, second);
    float c, s;
    turn_of(l, token, i, position_of(l, token), &c, &s);
    to[first] = a * c - b * s;
    to[second] = a * s + b * c;
  }
  for (uint32_t i = rotary + lane; i < p.depth; i += kWaveLanes) to[i] = Traits<T>::load(from, i);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  if (query || kKind == CacheKind::kKept) {
    const uint32_t page = query ? 0u : p.page.quotient(slot), at = slot - page * p.page.divisor;
    unsigned char *out = query ? l.rotated + ((uint64_t)token * p.queries + row) * p.depth * Traits<T>::kSize
                               : l.cache + ((((uint64_t)page * 2 * p.heads + row - p.queries) * p.page.divisor + at) * p.depth) * Traits<T>::kSize;
    for (uint32_t i = lane; i < p.depth; i += kWaveLanes) {
      if (i < rotary) {
        Traits<T>::store(out, i, to[i]);
      } else if constexpr (Traits<T>::kSize == 4) {  // what is not rotated keeps its bits
        reinterpret_cast<uint32_t *>(out)[i] = reinterpret_cast<const uint32_t *>(from)[i];
      } else {
        reinterpret_cast<uint16_t *>(out)[i] = reinterpret_cast<const uint16_t *>(from)[i];
      }
    }
  } else {
    const uint32_t page = p.page.quotient(slot), at = slot - page * p.page.divisor;
    const uint64_t line = (uint64_t)page * 2 * p.heads + row - p.queries;
    if constexpr (kKind == CacheKind::kNarrow) {
      unsigned char *out = l.cache + (line * p.page.divisor + at) * p.depth;
      for (uint32_t i = lane; i < p.depth; i += kWaveLanes) out[i] = (unsigned char)pack_e4m3(to[i], 0.0f, 0.0f, 0.0f);
    } else {
      const uint32_t blocks = p.depth / kMx4Block;
      unsigned char *base = l.cache + line * (p.page.divisor * (uint64_t)(blocks * 17));
      for (uint32_t i = lane; i < blocks; i += kWaveLanes)
        mx4_store_block<T>([&](int e) { return to[i * kMx4Block + e]; }, base + (uint64_t)at * (p.depth / 2) + i * 16,
                           base + (uint64_t)p.page.divisor * (p.depth / 2) + (uint64_t)at * blocks + i);
    }
  }
}

}  // namespace

template <CacheKind kKind> struct RotaryRowsTag {
  static std::string text() {
    return std::string("rotary_append_rows/") + (kKind == CacheKind::kFourBits ? "mx4" : kKind == CacheKind::kNarrow ? "e4m3" : "kept");
  }
};

template <class T, CacheKind kKind> static void start(Layout l, bool vector_aligned, hipStream_t stream) {
  l.units = (uint64_t)l.p.tokens * (l.p.queries + 2 * l.p.heads);
  note_variant<RotaryRowsTag<kKind>>();
  hipLaunchKernelGGL((rotary_append_rows<T, kKind>), dim3((uint32_t)((l.units + kWaves - 1) / kWaves)), dim3(kBlockThreads), 0, stream, l);
}

hipError_t launch_rotary_append(Elem type, const RotaryAppendParams &p, const void *projected, const void *positions, const void *frequencies,
                                const int32_t *slots, void *cache, void *rotated, bool vector_aligned, hipStream_t stream) {
  Layout l{};
  l.p = p;
  l.projected = static_cast<const unsigned char *>(projected);
  l.positions = positions;
  l.frequencies = static_cast<const float *>(frequencies);
  l.slots = slots;
  l.cache = static_cast<unsigned char *>(cache);
  l.rotated = static_cast<unsigned char *>(rotated);
  l.slot_count = p.pages * p.page.divisor;
  auto typed = [&](auto tag) {
    using T = decltype(tag);
    switch (p.cache) {
      case CacheKind::kKept: start<T, CacheKind::kKept>(l, vector_aligned, stream); break;
      case CacheKind::kNarrow: start<T, CacheKind::kNarrow>(l, vector_aligned, stream); break;
      case CacheKind::kFourBits: start<T, CacheKind::kFourBits>(l, vector_aligned, stream); break;
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
