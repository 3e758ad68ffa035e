// attention_general.hip -- attention of any type, depth and alignment: one block per query row and head.
//
// Each of the block's waves takes every kWaves-th group of 64 keys: a lane's product of the query (in LDS, f32) with one key,
// the running maximum m and sum l of the softmax, then the 64 weights over the values with a lane per dim:
//   o <- o * exp(m - m') + sum_j exp(s_j - m') v_j,   l <- l * exp(m - m') + sum_j exp(s_j - m').
// The waves' (m, l, o) are joined through LDS by the same rule.  Weights and sums stay in f32 throughout.
// For f32, and for depths and addresses that are no whole vectors; bound by its scalar loads and multiply-adds (8192 causal tokens
// of 16 heads of 128 took 60.8 ms here, 4.5 TFLOP/s).  The waves split the keys, so that one row over many keys is not one wave's.
#include "attention.h"

namespace hyle_hip {
namespace {

constexpr int kWaves = 8;
constexpr int kMaxDepth = 256;
constexpr int kDims = kMaxDepth / kWaveLanes;  // of a lane
constexpr uint32_t kAcross = 1u << 22;  // blocks along x, whose threads are counted in 32 bits; further ones lie along y

__host__ __device__ inline uint32_t blocks_of(const AttentionParams &p) {  // (no more than there are query elements)
  return (uint32_t)p.rows * (p.kind == AttentionKind::kPacked ? 1u : (uint32_t)p.sequences / p.apart.divisor) * (uint32_t)p.queries;
}

// Element d of a key or value at its codes' address; `scales`, of a cache in 4 bits.
template <class C> __device__ __forceinline__ float element(const unsigned char *at, const unsigned char *scales, int d) {
  if constexpr (std::is_same<C, MX4>::value) return mx4_element(at, scales, d);
  else return Traits<C>::load(at, d);
}

template <class T, class C>
__global__ __launch_bounds__(kWaves * kWaveLanes) void attention_rows(AttentionParams p, AttentionBuffers b) {
  __shared__ float query[kMaxDepth], weights[kWaves][kWaveLanes], joined[kWaves][kMaxDepth], tops[kWaves], sums[kWaves];
  const uint32_t block = blockIdx.y * kAcross + blockIdx.x;
  if (block >= blocks_of(p)) return;
  const int head = (int)(block % (uint32_t)p.queries);
  int row = (int)(block / (uint32_t)p.queries), index;
  if (p.kind == AttentionKind::kPacked) {
    // the last sequence that begins at or before the row
    int low = 0, high = p.sequences - 1;
    while (low < high) {
      const int middle = (low + high + 1) / 2;
      if (b.marks[middle] <= row) low = middle;
      else high = middle - 1;
    }
    index = low;
    const AttentionSequence s = attention_sequence(p, b.marks, index);
    if (row < s.row || row >= s.row + s.rows) return;  // a row of no sequence
    row -= (int)s.row;
  } else {
    index = row / p.rows;
    row -= index * p.rows;
  }
  const int group = (int)p.shared.quotient((uint32_t)head);
  if (p.apart.divisor != 1) index = index * (int)p.apart.divisor + group;  // a sequence of its own
  const AttentionSequence s = attention_sequence(p, b.marks, index);
  const AttentionSpan span = attention_span(p, s.keys, s.first + row);
  const unsigned char *q = attention_query(p, b, s, row, head);
  const int wave = (int)threadIdx.x / kWaveLanes, lane = (int)threadIdx.x % kWaveLanes;
  for (int d = threadIdx.x; d < p.depth; d += kWaves * kWaveLanes) query[d] = Traits<T>::load(q, d);
  __syncthreads();

  float top = -INFINITY, sum = 0.0f, out[kDims] = {};
  // groups of keys: those of the sinks before the window first, then the window's
  const int sinks = min(min(p.sinks, span.low), span.high);
  const int before = (sinks + kWaveLanes - 1) / kWaveLanes, low = max(0, span.low);
  const int groups = before + (span.high > low ? (span.high - low + kWaveLanes - 1) / kWaveLanes : 0);
  for (int g = wave; g < groups; g += kWaves) {
    const int first = g < before ? g * kWaveLanes : low + (g - before) * kWaveLanes;
    const int end = g < before ? sinks : span.high;
    AttentionPlace place{0, 0, 0};
    bool seen = first + lane < end;
    if (seen) seen = attention_place(p, b.table, s, index, first + lane, &place);
    float score = -INFINITY;
    if (seen) {
      const unsigned char *k = static_cast<const unsigned char *>(b.key) + place.key + (int64_t)group * p.k_head;
      const unsigned char *k_scales = static_cast<const unsigned char *>(b.key) + place.scale + (int64_t)group * p.k_head;
      score = 0.0f;
      for (int d = 0; d < p.depth; ++d) score = fmaf(query[d], element<C>(k, k_scales, d), score);
      score *= p.scale;  // (a query times the scale may pass f32's range where the product does not)
    }
    const float next = fmaxf(top, group_max<kWaveLanes>(score));
    const float shift = next == -INFINITY ? 0.0f : next;
    const float weight = seen ? expf(score - shift) : 0.0f;
    const float keep = expf(top - shift);
    top = next;
    sum = sum * keep + group_sum<kWaveLanes>(weight);
    weights[wave][lane] = weight;
#pragma unroll
    for (int i = 0; i < kDims; ++i) out[i] *= keep;
    uint64_t lanes = __ballot(seen);  // a wave's own LDS writes and reads are in order
    while (lanes != 0) {
      const int j = __builtin_ctzll(lanes);
      lanes &= lanes - 1;
      const float w = weights[wave][j];
      const int64_t at = ((int64_t)__builtin_amdgcn_readlane((int)(place.value >> 32), j) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)place.value, j);
      const unsigned char *v = static_cast<const unsigned char *>(b.value) + at + (int64_t)group * p.v_head, *v_scales = v;
      if constexpr (std::is_same<C, MX4>::value) {
        const int64_t scale_at = ((int64_t)__builtin_amdgcn_readlane((int)(place.scale >> 32), j) << 32) |
                                 (uint32_t)__builtin_amdgcn_readlane((int)place.scale, j);
        v_scales = static_cast<const unsigned char *>(b.value) + scale_at + (int64_t)group * p.v_head;
      }
#pragma unroll
      for (int i = 0; i < kDims; ++i) {
        const int d = lane + i * kWaveLanes;
        if (d < p.depth) out[i] = fmaf(w, element<C>(v, v_scales, d), out[i]);
      }
    }
  }
  if (lane == 0) tops[wave] = top, sums[wave] = sum;
#pragma unroll
  for (int i = 0; i < kDims; ++i) joined[wave][lane + i * kWaveLanes] = out[i];
  __syncthreads();
  float most = tops[0];
  for (int w = 1; w < kWaves; ++w) most = fmaxf(most, tops[w]);
  const float shift = most == -INFINITY ? 0.0f : most;
  float total = 0.0f;
  for (int w = 0; w < kWaves; ++w) total += sums[w] * expf(tops[w] - shift);
  const int64_t at = (s.row + row) * p.queries + head;
  for (int d = threadIdx.x; d < p.depth; d += kWaves * kWaveLanes) {
    float o = 0.0f;
    for (int w = 0; w < kWaves; ++w) o += joined[w][d] * expf(tops[w] - shift);
    Traits<T>::store(b.out, (size_t)(at * p.depth + d), total == 0.0f ? 0.0f : o / total);
  }
  if (b.logs != nullptr && threadIdx.x == 0) b.logs[at] = total == 0.0f ? -INFINITY : shift + logf(total);
}

}  // namespace

struct AttentionGeneralTag {
  static std::string text() { return "attention_rows"; }
};

template <class T, class C> static void start(const AttentionParams &p, const AttentionBuffers &b, hipStream_t stream) {
  const uint32_t blocks = blocks_of(p);
  const dim3 grid(blocks < kAcross ? blocks : kAcross, (blocks + kAcross - 1) / kAcross);
  hipLaunchKernelGGL((attention_rows<T, C>), grid, dim3(kWaves * kWaveLanes), 0, stream, p, b);
}

hipError_t launch_attention_general(Elem type, const AttentionParams &p, const AttentionBuffers &b, hipStream_t stream) {
  note_variant<AttentionGeneralTag>();
  switch (type) {
    case Elem::kF32: p.four_bits ? start<F32, MX4>(p, b, stream) : p.narrow_cache ? start<F32, E4M3>(p, b, stream) : start<F32, F32>(p, b, stream); break;
    case Elem::kF16: p.four_bits ? start<F16, MX4>(p, b, stream) : p.narrow_cache ? start<F16, E4M3>(p, b, stream) : start<F16, F16>(p, b, stream); break;
    case Elem::kBF16: p.four_bits ? start<BF16, MX4>(p, b, stream) : p.narrow_cache ? start<BF16, E4M3>(p, b, stream) : start<BF16, BF16>(p, b, stream); break;
  }
  return hipGetLastError();
}

}  // namespace hyle_hip
