// attention.h -- what the attention kernels share: which rows and keys a sequence has, where a key stands, which keys a
// query sees, and the decoder of e4m3 caches.
#pragma once

#include "device_common.h"
#include "kernels.h"

namespace hyle_hip {

struct E4M3 {};
template <> struct Traits<E4M3> {
  static constexpr int kSize = 1;
  static __device__ __forceinline__ float load(const void *p, size_t i) {
    return __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t *>(p)[i], 0);
  }
};

// One sequence of a launch.  `first` is the position of its first query; its queries are rows `row` on of the output.
struct AttentionSequence {
  int rows, keys, first;
  int64_t row;
};

// Marks are clamped to what the operands hold, so no value of theirs leads outside.
__device__ __forceinline__ int attention_mark(const AttentionParams &p, const int32_t *marks, int index) {
  return marks != nullptr ? max(marks[index], 0) : p.keys;
}
// A sequence of a batch or a paged cache, by its mark.
__device__ __forceinline__ AttentionSequence attention_sequence_of(const AttentionParams &p, int index, int mark) {
  AttentionSequence s;
  s.rows = p.rows;
  s.keys = min(mark, p.keys);
  s.first = (p.kind == AttentionKind::kPaged ? mark : p.keys) - p.rows;
  s.row = (int64_t)index * p.rows;
  return s;
}
__device__ __forceinline__ AttentionSequence attention_sequence(const AttentionParams &p, const int32_t *marks, int index) {
  if (p.kind != AttentionKind::kPacked) return attention_sequence_of(p, index, attention_mark(p, marks, index));
  AttentionSequence s;
  const int begin = min(max(marks[index], 0), p.rows), end = min(max(marks[index + 1], begin), p.rows);
  s.rows = s.keys = end - begin;
  s.first = 0;
  s.row = begin;
  return s;
}

// The keys that a query at `position` sees: [low, high), and of those before low the first `sinks`.
struct AttentionSpan {
  int low, high;
};
__device__ __forceinline__ AttentionSpan attention_span(const AttentionParams &p, int keys, int position) {
  AttentionSpan s{0, keys};
  if (p.causal) {
    s.high = max(0, min(keys, position + 1));  // (positions are below 2^31 - 1: lengths count from one)
    if (p.window != 0 && position >= p.window) s.low = position - p.window + 1;
  }
  return s;
}
__device__ __forceinline__ bool attention_sees(const AttentionParams &p, const AttentionSpan &s, int key) {
  return key < s.high && (key >= s.low || key < p.sinks);
}

__device__ __forceinline__ const unsigned char *attention_query(const AttentionParams &p, const AttentionBuffers &b, const AttentionSequence &s,
                                                                int index, int row, int head) {
  const int64_t at = p.kind == AttentionKind::kPacked ? (s.row + row) * p.q_row : (int64_t)index * p.q_sequence + (int64_t)row * p.q_row;
  return static_cast<const unsigned char *>(b.query) + at + (int64_t)head * p.q_head;
}

// Byte offsets of key `key` of head 0 from the operands' first bytes; false where a paged key has no page in the cache.
struct AttentionPlace {
  int64_t key, value;
};
__device__ __forceinline__ bool attention_place(const AttentionParams &p, const int32_t *table, const AttentionSequence &s, int index, int key,
                                                AttentionPlace *place) {
  if (p.kind == AttentionKind::kPaged) {
    const uint32_t column = p.page.quotient((uint32_t)key), at = (uint32_t)key - column * p.page.divisor;
    const int32_t page = table[(int64_t)index * p.table_row + column];
    place->key = place->value = (int64_t)page * p.k_sequence + (int64_t)at * p.k_row;
    return (uint32_t)page < (uint32_t)p.pages;
  }
  const int64_t row = p.kind == AttentionKind::kPacked ? s.row + key : key;
  const int64_t sequence = p.kind == AttentionKind::kPacked ? 0 : index;
  place->key = sequence * p.k_sequence + row * p.k_row;
  place->value = sequence * p.v_sequence + row * p.v_row;
  return true;
}

}  // namespace hyle_hip
