// rotary_append.hip -- the projected rows [tokens, queries + 2 heads, depth] of new tokens: queries and keys rotated by their positions, the
// queries to a tensor of their own, keys and values to their slots of a paged cache.
//
// The rotation is RoPE's (rope.hip): phase = frequency * position in f32, a' = a cos - b sin, b' = a sin + b cos with every product and sum
// rounded on its own.  cos and sin are those of the f32 phase in 64 bits, rounded to f32 once: they are then the nearest numbers, whoever
// computes them, and so is everything behind them, down to the codes of a cache in 4 bits.  A rotated element is rounded once, to what
// the cache keeps.
//
// Bound by bytes: 8192 tokens of 32 query and 8 key heads of 128, bf16 to e4m3, 184 MB: 33.7 us, 5.5 TB/s (a wave to a row, which works out
// its own cos and sin, 162), to 4 bits 34.2; 64 tokens kept as bf16, 3.4 us, a launch; 1037 of 20 and 5 heads of 96 to 4 bits 6.7 us, launch, position,
// 64-bit cos and sin, rows and LDS one after another (half and four times the waves: the same).  Depths and rotary widths that are no multiples of
// 16 take a wave to a row: of the 8192 tokens, us as bf16 / e4m3 / 4 bits, width 128 37.3 / 34.3 / 34.2, 120 140 / 138 / 172, 40 162 / 157 / 197;
// depth 80, width 80 31.8, 40 142 (64 tokens 3.3 and 3.6).
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

// By whole vectors: a wave to a token (or to some of its rows, where tokens are few), whose cos and sin are worked out once, two times eight
// elements of a row to a lane: those that turn together, or neighbours where nothing turns.  Rows for a cache in 4 bits go through LDS to
// lanes of eight neighbours, four to a scale.
template <class T> struct Eight {
  static constexpr int kWords = 8 / Traits<T>::kVec;
  u32x4 words[kWords];
};
template <class T, CacheKind kKind, bool kHalf>
__global__ __launch_bounds__(kBlockThreads) void rotary_append_vectors(Layout l, Divisor splits, Divisor lanes, uint32_t rows_each) {
  constexpr int kWords = Eight<T>::kWords;
  constexpr bool kFour = kKind == CacheKind::kFourBits;
  __shared__ __attribute__((aligned(16))) float turns[kWaves][2][kMostDepth / 2];
  __shared__ __attribute__((aligned(16))) float staged[kFour ? kWaves : 1][kFour ? kWaveLanes * 16 : 1];
  const RotaryAppendParams &p = l.p;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWaveLanes)), lane = threadIdx.x % kWaveLanes;
  const uint32_t unit = blockIdx.x * kWaves + wave, token = splits.quotient(unit);
  if (token >= p.tokens) return;
  const uint32_t rows = p.queries + 2 * p.heads, first = (unit - token * splits.divisor) * rows_each, end = min(first + rows_each, rows);
  const uint32_t step = kWaveLanes / lanes.divisor, own = lanes.quotient(lane), part = lane - own * lanes.divisor;
  const bool turned = part < p.rotary / 16;
  const uint32_t near = kHalf && turned ? 8 * part : 16 * part, far = kHalf && turned ? p.rotary / 2 + near : near + 8;
  const uint32_t slot = (uint32_t)l.slots[token], page = p.page.quotient(slot), at = slot - page * p.page.divisor;
  const unsigned char *from = l.projected + (int64_t)token * p.token;
  // (a token without a slot has queries alone)
  const uint32_t last = slot < l.slot_count ? end : min(end, p.queries);
  auto ask = [&](uint32_t row, Eight<T> *a, Eight<T> *b) {
    const unsigned char *at = from + (int64_t)min(row, rows - 1) * p.head;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      a->words[w] = load16_stream(at, near / Traits<T>::kVec + w);
      b->words[w] = load16_stream(at, far / Traits<T>::kVec + w);
    }
  };
  auto unpacked = [](const Eight<T> &v, float (&x)[8]) {
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      float some[Traits<T>::kVec];
      Traits<T>::unpack(v.words[w], some);
#pragma unroll
      for (int e = 0; e < Traits<T>::kVec; ++e) x[w * Traits<T>::kVec + e] = some[e];
    }
  };
  auto packed = [](const float (&x)[8]) {
    Eight<T> v;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      float some[Traits<T>::kVec];
#pragma unroll
      for (int e = 0; e < Traits<T>::kVec; ++e) some[e] = x[w * Traits<T>::kVec + e];
      v.words[w] = Traits<T>::pack(some);
    }
    return v;
  };
  if (first >= last) return;
  Eight<T> a, b;
  ask(first + own, &a, &b);
  if (first < p.queries + p.heads) {
    const float position = position_of(l, token);
    for (uint32_t i = lane; i < p.rotary / 2; i += kWaveLanes) turn_of(l, token, i, position, &turns[wave][0][i], &turns[wave][1][i]);
  }
  __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses are in order)
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = turns[wave][0][turned ? 8 * part + e : 0], s[e] = turns[wave][1][turned ? 8 * part + e : 0];
  for (uint32_t base = first; base < last; base += step) {
    const uint32_t row = base + own;
    const bool mine = own < step && row < last, query = row < p.queries;
    float x[8], y[8];
    unpacked(a, x), unpacked(b, y);
    Eight<T> keep_a = a, keep_b = b;
    if (base + step < last) ask(row + step, &a, &b);
    if (turned && row < p.queries + p.heads) {
      if constexpr (kHalf) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = x[e], v = y[e];
          x[e] = u * c[e] - v * s[e];
          y[e] = u * s[e] + v * c[e];
        }
      } else {
        auto pairs = [&](float (&z)[8], int from) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = z[2 * e], v = z[2 * e + 1];
            z[2 * e] = u * c[from + e] - v * s[from + e];
            z[2 * e + 1] = u * s[from + e] + v * c[from + e];
          }
        };
        pairs(x, 0), pairs(y, 4);
      }
      if (query || kKind == CacheKind::kKept) keep_a = packed(x), keep_b = packed(y);
    }
    const uint64_t line = (uint64_t)page * 2 * p.heads + row - p.queries;
    if (mine && (query || kKind == CacheKind::kKept)) {  // what is not rotated keeps its bits
      unsigned char *out = query ? l.rotated + ((uint64_t)token * p.queries + row) * p.depth * Traits<T>::kSize
                                 : l.cache + (line * p.page.divisor + at) * p.depth * Traits<T>::kSize;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        store16(out, near / Traits<T>::kVec + w, keep_a.words[w]);
        store16(out, far / Traits<T>::kVec + w, keep_b.words[w]);
      }
    }
    if constexpr (kKind == CacheKind::kNarrow) {
      if (mine && !query) {
        unsigned char *out = l.cache + (line * p.page.divisor + at) * p.depth;
        *reinterpret_cast<uint2 *>(out + near) = uint2{pack_e4m3(x[0], x[1], x[2], x[3]), pack_e4m3(x[4], x[5], x[6], x[7])};
        *reinterpret_cast<uint2 *>(out + far) = uint2{pack_e4m3(y[0], y[1], y[2], y[3]), pack_e4m3(y[4], y[5], y[6], y[7])};
      }
    }
    if constexpr (kFour) {
      if (base + step > p.queries) {  // some of these rows are the cache's
        float *to = staged[wave];
        __builtin_amdgcn_wave_barrier();
        if (own < step) {
          f32x4 *near_to = reinterpret_cast<f32x4 *>(to + own * p.depth + near), *far_to = reinterpret_cast<f32x4 *>(to + own * p.depth + far);
          near_to[0] = f32x4{x[0], x[1], x[2], x[3]}, near_to[1] = f32x4{x[4], x[5], x[6], x[7]};
          far_to[0] = f32x4{y[0], y[1], y[2], y[3]}, far_to[1] = f32x4{y[4], y[5], y[6], y[7]};
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
          // (a quad of lanes is one block of one row: all of it is here or none)
          const uint32_t eight = half * kWaveLanes + lane, of = lanes.quotient(eight / 2), row_of = base + of;
          if (of >= step || row_of < p.queries || row_of >= last) continue;
          const uint32_t d = (eight - of * 2 * lanes.divisor) * 8;
          const f32x4 *in = reinterpret_cast<const f32x4 *>(to + of * p.depth + d);
          const f32x4 some = in[0], more = in[1];
          const float z[8] = {some[0], some[1], some[2], some[3], more[0], more[1], more[2], more[3]};
          uint32_t byte;
          const uint32_t codes = mx4_of_quad<T>(z, &byte);
          unsigned char *side = l.cache + ((uint64_t)page * 2 * p.heads + row_of - p.queries) * (p.page.divisor * (uint64_t)(p.depth / kMx4Block * 17));
          *reinterpret_cast<uint32_t *>(side + (uint64_t)at * (p.depth / 2) + d / 2) = codes;
          if (lane % 4 == 0) side[(uint64_t)p.page.divisor * (p.depth / 2) + (uint64_t)at * (p.depth / kMx4Block) + d / kMx4Block] = (unsigned char)byte;
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
}

}  // namespace

static const char *kind_name(CacheKind kind) { return kind == CacheKind::kFourBits ? "mx4" : kind == CacheKind::kNarrow ? "e4m3" : "kept"; }
template <CacheKind kKind> struct RotaryRowsTag {
  static std::string text() { return std::string("rotary_append_rows/") + kind_name(kKind); }
};
template <CacheKind kKind, bool kHalf> struct RotaryVectorsTag {
  static std::string text() { return std::string("rotary_append_vectors/") + kind_name(kKind) + (kHalf ? "/half-split" : "/interleaved"); }
};

template <class T, CacheKind kKind, bool kHalf> static void start_vectors(const Layout &l, int compute_units, hipStream_t stream) {
  note_variant<RotaryVectorsTag<kKind, kHalf>>();
  const uint32_t rows = l.p.queries + 2 * l.p.heads, step = kWaveLanes / (l.p.depth / 16), steps = (rows + step - 1) / step;
  // a token's rows are split where its tokens alone are few waves to each unit
  const uint32_t wanted = 16 * (uint32_t)compute_units / l.p.tokens, most = wanted < 1 ? 1 : wanted < steps ? wanted : steps;
  const uint32_t rows_each = (steps + most - 1) / most * step, splits = (rows + rows_each - 1) / rows_each;
  const uint64_t waves = (uint64_t)l.p.tokens * splits;
  hipLaunchKernelGGL((rotary_append_vectors<T, kKind, kHalf>), dim3((uint32_t)((waves + kWaves - 1) / kWaves)), dim3(kBlockThreads), 0, stream, l,
                     Divisor(splits), Divisor(l.p.depth / 16), rows_each);
}
template <class T, CacheKind kKind> static void start(Layout l, bool vector_aligned, int compute_units, hipStream_t stream) {
  // (words of codes are written at addresses of whole words)
  const bool cache_aligned = kKind == CacheKind::kFourBits
                                 ? reinterpret_cast<uintptr_t>(l.cache) % 4 == 0 && l.p.page.divisor * (uint64_t)(l.p.depth / kMx4Block * 17) % 4 == 0
                                 : reinterpret_cast<uintptr_t>(l.cache) % 16 == 0;
  if (vector_aligned && cache_aligned && l.p.depth % 16 == 0 && l.p.rotary % 16 == 0 && (l.p.token | l.p.head) % 16 == 0) {
    if (l.p.half_split) start_vectors<T, kKind, true>(l, compute_units, stream);
    else start_vectors<T, kKind, false>(l, compute_units, stream);
    return;
  }
  l.units = (uint64_t)l.p.tokens * (l.p.queries + 2 * l.p.heads);
  note_variant<RotaryRowsTag<kKind>>();
  hipLaunchKernelGGL((rotary_append_rows<T, kKind>), dim3((uint32_t)((l.units + kWaves - 1) / kWaves)), dim3(kBlockThreads), 0, stream, l);
}

// vector_aligned: the rows and the rotated queries
hipError_t launch_rotary_append(Elem type, const RotaryAppendParams &p, const void *projected, const void *positions, const void *frequencies,
                                const int32_t *slots, void *cache, void *rotated, bool vector_aligned, int compute_units, hipStream_t stream) {
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
      case CacheKind::kKept: start<T, CacheKind::kKept>(l, vector_aligned, compute_units, stream); break;
      case CacheKind::kNarrow: start<T, CacheKind::kNarrow>(l, vector_aligned, compute_units, stream); break;
      case CacheKind::kFourBits: start<T, CacheKind::kFourBits>(l, vector_aligned, compute_units, stream); break;
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
