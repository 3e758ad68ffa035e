"""Attention, PagedAttention and PagedAppend without a device: inferred outputs, refusals and declines."""
from __future__ import annotations

import math

import pytest

from hyle_amd import compute as hc

DT, D = hc.DataType, hc.TensorDesc.dense
CTX = hc.Context.planning_only()
BF16, F32, I32, E4M3 = DT.kBFloat16, DT.kFloat32, DT.kInt32, DT.kFloat8E4M3FN


def test_attention_outputs_follow_the_queries():
    q, k = D(BF16, [2, 5, 8, 64]), D(BF16, [2, 9, 4, 64])
    assert hc.infer_output_descriptions(hc.Attention(), [q, k, k]) == [q]
    assert hc.infer_output_descriptions(hc.Attention(0.125, False, return_log_sum=True), [q, k, k, D(I32, [2])]) == [q, D(F32, [2, 5, 8])]
    t = D(DT.kFloat16, [7, 6, 80])
    assert hc.infer_output_descriptions(hc.Attention(window=3, sinks=1), [t, D(DT.kFloat16, [7, 2, 80]), D(DT.kFloat16, [7, 2, 80]), D(I32, [4])]) == [t]
    cache, table, lengths = D(E4M3, [10, 2, 4, 16, 64]), D(I32, [2, 3]), D(I32, [2])
    assert hc.infer_output_descriptions(hc.PagedAttention(return_log_sum=True), [q, cache, table, lengths]) == [q, D(F32, [2, 5, 8])]
    one = D(BF16, [2, 8, 64])
    assert hc.infer_output_descriptions(hc.PagedAttention(), [one, D(BF16, [10, 2, 4, 16, 64]), table, lengths]) == [one]
    keys = D(BF16, [3, 4, 64])
    assert hc.infer_output_descriptions(hc.PagedAppend(10, 16, E4M3), [keys, keys, D(I32, [3])]) == [cache]


def _refused(operation, inputs, code=hc.StatusCode.kInvalidArgument):
    with pytest.raises(hc.StatusError) as refused:
        hc.prepare(CTX, operation, *inputs)
    assert refused.value.code == code, refused.value


Q, K, MARKS = D(BF16, [2, 5, 8, 64]), D(BF16, [2, 9, 4, 64]), D(I32, [2])


@pytest.mark.parametrize("operation,inputs", [
    (hc.Attention(), [Q, K]),                                                   # values are missing
    (hc.Attention(), [Q, K, K, MARKS, MARKS]),                                  # one input too many
    (hc.Attention(), [D(I32, [2, 5, 8, 64]), K, K]),                            # queries that are not floating
    (hc.Attention(), [D(BF16, [8, 64]), D(BF16, [4, 64]), D(BF16, [4, 64])]),   # no row axis
    (hc.Attention(), [Q, D(DT.kFloat16, [2, 9, 4, 64]), K]),                    # types differ
    (hc.Attention(), [Q, K, D(BF16, [2, 8, 4, 64])]),                           # values of another number
    (hc.Attention(), [Q, D(BF16, [2, 9, 4, 32]), D(BF16, [2, 9, 4, 32])]),      # depths differ
    (hc.Attention(), [Q, D(BF16, [3, 9, 4, 64]), D(BF16, [3, 9, 4, 64])]),      # batches differ
    (hc.Attention(), [Q, D(BF16, [2, 9, 3, 64]), D(BF16, [2, 9, 3, 64])]),      # 8 query heads over 3
    (hc.Attention(), [Q, D(BF16, [2, 9, 0, 64]), D(BF16, [2, 9, 0, 64])]),      # no key heads
    (hc.Attention(), [D(BF16, [2, 5, 8, 0]), D(BF16, [2, 9, 4, 0]), D(BF16, [2, 9, 4, 0])]),  # no depth
    (hc.Attention(), [Q, K, K, D(DT.kInt64, [2])]),                             # marks of another type
    (hc.Attention(), [Q, K, K, D(I32, [3])]),                                   # marks of another batch
    (hc.Attention(), [D(BF16, [5, 8, 64]), D(BF16, [9, 4, 64]), D(BF16, [9, 4, 64]), D(I32, [2])]),  # packed rows differ
    (hc.Attention(), [D(BF16, [5, 8, 64]), D(BF16, [5, 4, 64]), D(BF16, [5, 4, 64]), D(I32, [0])]),  # not even an end
    (hc.Attention(scale=math.nan), [Q, K, K]),
    (hc.Attention(scale=math.inf), [Q, K, K]),
    (hc.Attention(causal=False, window=4), [Q, K, K]),                          # a window without an order
    (hc.Attention(sinks=4), [Q, K, K]),                                         # sinks without a window
    (hc.Attention(window=-1), [Q, K, K]),
    (hc.Attention(window=2 ** 31), [Q, K, K]),
    (hc.Attention(window=4, sinks=-1), [Q, K, K]),
    (hc.PagedAttention(), [Q, D(BF16, [10, 2, 4, 16, 64]), D(I32, [2, 3])]),    # lengths are missing
    (hc.PagedAttention(), [Q, D(BF16, [10, 1, 4, 16, 64]), D(I32, [2, 3]), MARKS]),
    (hc.PagedAttention(), [Q, D(BF16, [10, 2, 4, 16, 32]), D(I32, [2, 3]), MARKS]),
    (hc.PagedAttention(), [Q, D(DT.kFloat16, [10, 2, 4, 16, 64]), D(I32, [2, 3]), MARKS]),
    (hc.PagedAttention(), [Q, D(DT.kFloat8E5M2, [10, 2, 4, 16, 64]), D(I32, [2, 3]), MARKS]),
    (hc.PagedAttention(), [Q, D(BF16, [10, 2, 4, 16, 64]), D(I32, [3, 3]), MARKS]),
    (hc.PagedAttention(), [Q, D(BF16, [10, 2, 4, 16, 64]), D(DT.kInt64, [2, 3]), MARKS]),
    (hc.PagedAttention(sinks=1), [Q, D(BF16, [10, 2, 4, 16, 64]), D(I32, [2, 3]), MARKS]),
    (hc.PagedAppend(10, 16, BF16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 32]), D(I32, [3])]),
    (hc.PagedAppend(10, 16, BF16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [2])]),
    (hc.PagedAppend(10, 16, BF16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(DT.kInt64, [3])]),
    (hc.PagedAppend(10, 16, DT.kFloat16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3])]),
    (hc.PagedAppend(10, 16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3])]),
    (hc.PagedAppend(10, 0, BF16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3])]),
    (hc.PagedAppend(-1, 16, BF16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3])]),
    (hc.PagedAppend(2 ** 28, 16, BF16), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3])]),  # slots past int32
])
def test_operands_that_do_not_fit_are_refused(operation, inputs):
    _refused(operation, inputs)


def _strided(dtype, dims, strides):
    return hc.TensorDesc.strided_bytes(dtype, dims, strides)


@pytest.mark.parametrize("operation,inputs", [
    (hc.Attention(), [D(DT.kFloat64, [5, 4, 64])] * 3),                                          # a type that the kernels do not compute in
    (hc.Attention(), [D(BF16, [5, 4, 264])] * 3),                                                # deeper than served
    (hc.Attention(), [D(BF16, [5, 4, 64]), _strided(BF16, (5, 4, 64), (4, 1280, 20)), D(BF16, [5, 4, 64])]),  # heads that are no runs
    (hc.Attention(), [D(BF16, [5, 4, 64]), _strided(BF16, (5, 4, 64), (513, 128, 2)), D(BF16, [5, 4, 64])]),  # rows between elements
    (hc.Attention(), [D(BF16, [5, 4, 64])] * 3 + [_strided(I32, (3,), (8,))]),                   # marks that are no run
    (hc.PagedAttention(), [D(BF16, [1, 4, 64]), D(BF16, [4, 2, 4, 2 ** 16, 64]), D(I32, [1, 2 ** 15]), D(I32, [1])]),  # positions past int32
    (hc.PagedAppend(10, 16, BF16), [_strided(BF16, (3, 4, 64), (512, 2, 8)), D(BF16, [3, 4, 64]), D(I32, [3])]),
])
def test_operands_that_no_kernel_takes_are_declined(operation, inputs):
    _refused(operation, inputs, hc.StatusCode.kUnimplemented)


def test_empty_operands_are_no_work():
    assert hc.prepare(CTX, hc.Attention(), *[D(BF16, [0, 4, 64])] * 3).dispatch_count() == 0
    assert hc.prepare(CTX, hc.Attention(), *[D(BF16, [5, 4, 64])] * 3, D(I32, [1])).dispatch_count() == 0  # no sequence
    assert hc.prepare(CTX, hc.PagedAttention(), D(BF16, [0, 4, 64]), D(BF16, [4, 2, 4, 16, 64]), D(I32, [0, 2]), D(I32, [0])).dispatch_count() == 0
    assert hc.prepare(CTX, hc.PagedAppend(0, 16, BF16), D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3])).dispatch_count() == 0
    # queries without a key still have rows to write
    assert hc.prepare(CTX, hc.Attention(), D(BF16, [5, 4, 64]), D(BF16, [0, 4, 64]), D(BF16, [0, 4, 64])).dispatch_count() > 0


def test_no_operand_may_be_an_output():
    q = D(BF16, [5, 4, 64])
    plan = hc.prepare(CTX, hc.Attention(), q, q, q)
    assert not any(plan.alias_support(0, i) for i in range(3))
    append = hc.prepare(CTX, hc.PagedAppend(10, 16, BF16), D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), D(I32, [3]))
    assert not any(append.alias_support(0, i) for i in range(3))


def test_workspaces_hold_what_split_keys_leave():
    def plan(sequences, columns, window=0, depth=128):
        return hc.prepare(CTX, hc.PagedAttention(window=window), D(BF16, [sequences, 8, depth]), D(BF16, [64, 2, 2, 16, depth]), D(I32, [sequences, columns]),
                          D(I32, [sequences]))
    short = plan(4, 32)                       # 512 keys: a block to a sequence and key head
    assert short.dispatch_count() == 1 and short.workspace_requirement().size == 0
    long = plan(4, 33)
    assert long.dispatch_count() == 2 and long.workspace_requirement().alignment == 256
    assert plan(1, 4096, window=300).dispatch_count() == 1  # a window of few tiles, whatever lies before it
    assert plan(64, 4096).workspace_requirement().size < 64 << 20
    assert hc.prepare(CTX, hc.PagedAttention(), D(BF16, [2, 8, 60]), D(BF16, [64, 2, 2, 16, 60]), D(I32, [2, 4096]), D(I32, [2])).dispatch_count() == 1
