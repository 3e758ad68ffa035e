"""RotaryAppend, PageBounds, PagedSelect and caches of 4 bits without a device: inferred outputs, refusals and declines."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc

import cache_support as cs

DT, D = hc.DataType, hc.TensorDesc.dense
CTX = hc.Context.planning_only()
BF16, F16, F32, I32, I64, U8, E4M3 = DT.kBFloat16, DT.kFloat16, DT.kFloat32, DT.kInt32, DT.kInt64, DT.kUInt8, DT.kFloat8E4M3FN
HALF = hc.RopeLayout.kHalfSplit


def test_outputs_follow_the_operands():
    rows = D(BF16, [3, 16, 64])
    rest = [D(I32, [3]), D(F32, [16]), D(I32, [3])]
    assert hc.infer_output_descriptions(hc.RotaryAppend(10, 16, BF16, 4), [rows, *rest]) == [D(BF16, [10, 2, 4, 16, 64]), D(BF16, [3, 8, 64])]
    assert hc.infer_output_descriptions(hc.RotaryAppend(10, 16, U8, 4, HALF), [rows, D(I64, [3]), D(F32, [3, 32]), rest[2]]) == [
        D(U8, [10, 2, 4, 16, 34]), D(BF16, [3, 8, 64])]
    assert hc.infer_output_descriptions(hc.RotaryAppend(10, 16, E4M3, 8), [rows, *rest]) == [D(E4M3, [10, 2, 8, 16, 64])]  # keys and values alone
    keys = D(F16, [3, 4, 96])
    assert hc.infer_output_descriptions(hc.PagedAppend(10, 16, U8), [keys, keys, D(I32, [3])]) == [D(U8, [10, 2, 4, 16, 51])]
    q, four = D(F16, [2, 5, 8, 96]), D(U8, [10, 2, 4, 16, 51])
    assert hc.infer_output_descriptions(hc.PagedAttention(return_log_sum=True), [q, four, D(I32, [2, 3]), D(I32, [2])]) == [q, D(F32, [2, 5, 8])]
    assert hc.infer_output_descriptions(hc.PagedAttention(), [q, four, D(I32, [2, 4, 3]), D(I32, [2, 4])]) == [q]
    for cache in (four, D(F32, [10, 2, 4, 16, 96]), D(E4M3, [10, 2, 4, 16, 96])):
        assert hc.infer_output_descriptions(hc.PageBounds(3), [cache, D(I32, [2, 3]), D(I32, [2])]) == [D(BF16, [10, 2, 4, 96])]
    assert hc.infer_output_descriptions(hc.PagedSelect(7, 16), [q, D(BF16, [10, 2, 4, 96]), D(I32, [2, 3]), D(I32, [2])]) == [
        D(I32, [2, 4, 7]), D(I32, [2, 4])]


ROWS, AT, TURNS = D(BF16, [3, 16, 64]), D(I32, [3]), D(F32, [32])
Q, BOUNDS, TABLE, LENGTHS = D(BF16, [2, 5, 8, 64]), D(BF16, [10, 2, 4, 64]), D(I32, [2, 9]), D(I32, [2])
CACHE, FOUR = D(BF16, [10, 2, 4, 16, 64]), D(U8, [10, 2, 4, 16, 34])


@pytest.mark.parametrize("operation,inputs", [
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, TURNS]),                            # slots are missing
    (hc.RotaryAppend(10, 16, BF16, 9), [ROWS, AT, TURNS, AT]),                        # 18 heads of keys and values in 16
    (hc.RotaryAppend(10, 16, BF16, 0), [ROWS, AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, -1), [ROWS, AT, TURNS, AT]),
    (hc.RotaryAppend(10, 0, BF16, 4), [ROWS, AT, TURNS, AT]),
    (hc.RotaryAppend(-1, 16, BF16, 4), [ROWS, AT, TURNS, AT]),
    (hc.RotaryAppend(2 ** 28, 16, BF16, 4), [ROWS, AT, TURNS, AT]),                   # slots past int32
    (hc.RotaryAppend(10, 16, F16, 4), [ROWS, AT, TURNS, AT]),                         # a cache of another 16-bit type
    (hc.RotaryAppend(10, 16, DT.kFloat8E5M2, 4), [ROWS, AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, U8, 4), [D(BF16, [3, 16, 80]), AT, TURNS, AT]),          # no whole blocks of 32
    (hc.RotaryAppend(10, 16, BF16, 4), [D(I32, [3, 16, 64]), AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [D(BF16, [48, 64]), AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, D(F32, [3]), TURNS, AT]),               # positions that are no whole numbers
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, D(I32, [2]), TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, D(F32, [33]), AT]),                 # more pairs than the depth has
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, D(F32, [0]), AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, D(F32, [2, 32]), AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, D(BF16, [32]), AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, TURNS, D(I64, [3])]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, TURNS, D(I32, [4])]),
    (hc.PagedAppend(10, 16, U8), [D(BF16, [3, 4, 80]), D(BF16, [3, 4, 80]), AT]),
    (hc.PagedAppend(10, 16, DT.kInt8), [D(BF16, [3, 4, 64]), D(BF16, [3, 4, 64]), AT]),
    (hc.PagedAttention(), [Q, D(U8, [10, 2, 4, 16, 64]), D(I32, [2, 3]), LENGTHS]),   # bytes that are no blocks
    (hc.PagedAttention(), [Q, D(U8, [10, 2, 4, 16, 51]), D(I32, [2, 3]), LENGTHS]),   # blocks of another depth
    (hc.PagedAttention(), [Q, FOUR, D(I32, [2, 4, 3]), LENGTHS]),                     # lengths of sequences, pages of key heads
    (hc.PagedAttention(), [Q, FOUR, D(I32, [2, 8, 3]), D(I32, [2, 8])]),              # pages of query heads
    (hc.PagedAttention(), [Q, FOUR, D(I32, [2, 3]), D(I32, [2, 4])]),
    (hc.PageBounds(), [CACHE, TABLE]),
    (hc.PageBounds(), [BOUNDS, TABLE, LENGTHS]),                                      # no cache
    (hc.PageBounds(), [D(U8, [10, 2, 4, 16, 64]), TABLE, LENGTHS]),
    (hc.PageBounds(), [CACHE, TABLE, D(I32, [3])]),
    (hc.PageBounds(), [CACHE, D(I64, [2, 9]), LENGTHS]),
    (hc.PageBounds(-1), [CACHE, TABLE, LENGTHS]),
    (hc.PagedSelect(7, 16), [Q, BOUNDS, TABLE]),
    (hc.PagedSelect(7, 16), [Q, D(F16, [10, 2, 4, 64]), TABLE, LENGTHS]),             # bounds of another type
    (hc.PagedSelect(7, 16), [Q, D(BF16, [10, 2, 3, 64]), TABLE, LENGTHS]),            # 8 query heads over 3
    (hc.PagedSelect(7, 16), [Q, D(BF16, [10, 2, 4, 32]), TABLE, LENGTHS]),
    (hc.PagedSelect(7, 16), [Q, BOUNDS, D(I32, [3, 9]), LENGTHS]),
    (hc.PagedSelect(7, 0), [Q, BOUNDS, TABLE, LENGTHS]),
    (hc.PagedSelect(-1, 16), [Q, BOUNDS, TABLE, LENGTHS]),
    (hc.PagedSelect(2, 16), [Q, BOUNDS, TABLE, LENGTHS]),                             # five tokens can lie in two pages behind the first
    (hc.PagedSelect(5, 1), [Q, BOUNDS, TABLE, LENGTHS]),
    (hc.PagedSelect(1, 16), [D(BF16, [2, 8, 64]), BOUNDS, TABLE, LENGTHS]),
])
def test_operands_that_do_not_fit_are_refused(operation, inputs):
    with pytest.raises(hc.StatusError) as refused:
        hc.prepare(CTX, operation, *inputs)
    assert refused.value.is_invalid_argument(), refused.value


def _strided(dtype, dims, strides):
    return hc.TensorDesc.strided_bytes(dtype, dims, strides)


@pytest.mark.parametrize("operation,inputs", [
    (hc.RotaryAppend(10, 16, DT.kFloat64, 4), [D(DT.kFloat64, [3, 16, 64]), AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [_strided(BF16, (3, 16, 64), (4096, 256, 4)), AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 4), [ROWS, _strided(I32, (3,), (8,)), TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 1), [D(BF16, [3, 3, 1056]), AT, TURNS, AT]),
    (hc.RotaryAppend(10, 16, BF16, 1), [D(BF16, [2 ** 25, 8, 4]), D(I32, [2 ** 25]), D(F32, [2]), D(I32, [2 ** 25])]),  # 2^28 heads of tokens
    (hc.PagedAttention(), [Q, _strided(U8, (10, 2, 4, 16, 34), (4608, 2304, 576, 36, 1)), D(I32, [2, 3]), LENGTHS]),    # gaps between rows
    (hc.PagedAttention(), [Q, FOUR, _strided(I32, (2, 4, 3), (64, 12, 4)), D(I32, [2, 4])]),                              # a gap between sequences
    (hc.PagedAttention(), [Q, FOUR, D(I32, [2, 4, 3]), _strided(I32, (2, 4), (32, 4))]),
    (hc.PageBounds(), [D(DT.kFloat64, [10, 2, 4, 16, 64]), TABLE, LENGTHS]),
    (hc.PageBounds(), [_strided(U8, (10, 2, 4, 16, 34), (4608, 2304, 576, 36, 1)), TABLE, LENGTHS]),
    (hc.PageBounds(), [CACHE, D(I32, [2 ** 12, 2 ** 12]), D(I32, [2 ** 12])]),                                            # 2^26 pages of heads
    (hc.PagedSelect(7, 16), [D(DT.kFloat64, [2, 5, 8, 64]), BOUNDS, TABLE, LENGTHS]),
    (hc.PagedSelect(7, 16), [D(BF16, [2, 5, 8, 264]), D(BF16, [10, 2, 4, 264]), TABLE, LENGTHS]),
    (hc.PagedSelect(7, 2 ** 20), [Q, BOUNDS, D(I32, [2, 2 ** 12]), LENGTHS]),                                             # positions past int32
])
def test_operands_that_no_kernel_takes_are_declined(operation, inputs):
    with pytest.raises(hc.StatusError) as refused:
        hc.prepare(CTX, operation, *inputs)
    assert refused.value.code == hc.StatusCode.kUnimplemented, refused.value


def test_empty_operands_are_no_work():
    none = [D(I32, [0]), TURNS, D(I32, [0])]
    assert hc.prepare(CTX, hc.RotaryAppend(10, 16, BF16, 4), D(BF16, [0, 16, 64]), *none).dispatch_count() == 0
    assert hc.prepare(CTX, hc.RotaryAppend(0, 16, BF16, 8), ROWS, AT, TURNS, AT).dispatch_count() == 0
    assert hc.prepare(CTX, hc.RotaryAppend(0, 16, BF16, 4), ROWS, AT, TURNS, AT).dispatch_count() == 1  # queries are still rotated
    assert hc.prepare(CTX, hc.PageBounds(), CACHE, D(I32, [2, 0]), LENGTHS).dispatch_count() == 0
    assert hc.prepare(CTX, hc.PageBounds(), D(BF16, [0, 2, 4, 16, 64]), TABLE, LENGTHS).dispatch_count() == 0
    assert hc.prepare(CTX, hc.PagedSelect(7, 16), D(BF16, [0, 8, 64]), BOUNDS, D(I32, [0, 9]), D(I32, [0])).dispatch_count() == 0
    assert hc.prepare(CTX, hc.PagedSelect(7, 16), Q, BOUNDS, D(I32, [2, 0]), LENGTHS).dispatch_count() == 1  # lengths are still written


def test_a_choice_of_all_pages_needs_no_scores():
    few, many = (hc.prepare(CTX, hc.PagedSelect(count, 16), Q, BOUNDS, TABLE, LENGTHS) for count in (9, 8))
    assert few.dispatch_count() == 1 and few.workspace_requirement().size == 0
    assert many.dispatch_count() == 2 and many.workspace_requirement().size == 2 * 4 * 9 * 4


def test_no_operand_may_be_an_output():
    for operation, inputs in ((hc.RotaryAppend(10, 16, BF16, 4), [ROWS, AT, TURNS, AT]), (hc.PageBounds(), [CACHE, TABLE, LENGTHS]),
                              (hc.PagedSelect(7, 16), [Q, BOUNDS, TABLE, LENGTHS])):
        plan = hc.prepare(CTX, operation, *inputs)
        assert not any(plan.alias_support(o, i) for o in range(len(plan.output_descriptions())) for i in range(len(inputs)))


def test_blocks_of_four_bits_by_hand():
    """The checker's own codec at the places where its rules turn."""
    x = np.zeros((9, 32))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]   # ties, at a scale of one
    x[1, :3] = [7.0, 0.25, -5.0]                              # 1.75 * 4: no doubling
    x[2, :3] = [7.03125, 0.5, 1.5]                            # over it: scale two
    x[3, 0] = 2.0 ** -130
    x[4, 0] = -1.9 * 2.0 ** 127                               # beyond six of the largest scale
    x[5, 3] = np.nan
    x[6, 3] = -np.inf
    x[7, :2] = [-0.0, 4.0]
    codes, scales = cs.mx4_encode(x)
    assert scales[:, 0].tolist() == [127, 127, 128, 0, 252, 255, 255, 127, 0]
    nibbles = np.stack((codes & 15, codes >> 4), -1).reshape(9, 32)
    assert nibbles[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7]
    assert nibbles[1, :3].tolist() == [7, 0, 14] and nibbles[2, :3].tolist() == [6, 0, 2]
    assert nibbles[3, 0] == 0 and nibbles[4, 0] == 15 and nibbles[7, :2].tolist() == [8, 6]
    assert cs.mx4_encode(np.full((1, 32), 65504.0), torch.float16)[1][0, 0] == 140
    assert cs.mx4_decode(*cs.mx4_encode(np.full((1, 32), 65504.0), torch.float16))[0, 0] == 6 * 2.0 ** 13
    values = cs.mx4_decode(codes, scales)
    assert values[2, 0] == 8.0 and np.isnan(values[5]).all() and np.signbit(values[7, 0])
    joined = cs.mx4_join(codes.reshape(3, 3, 16), scales.reshape(3, 3, 1))
    assert joined.shape == (3, 3, 17)
    again = cs.mx4_split(joined)
    assert np.array_equal(again[0], codes.reshape(3, 3, 16)) and np.array_equal(again[1], scales.reshape(3, 3, 1))


@pytest.mark.parametrize("cache", [CACHE, FOUR])
@pytest.mark.parametrize("strides", [(0, 4), (32, 4), (4, 8)])
def test_lengths_of_key_heads_are_dense_also_where_the_table_is_empty(cache, strides):
    """The kernels read a length of every sequence and key head, pages or not: those of one sequence for all would be read past their end."""
    for columns in (3, 0):
        table = D(I32, [2, 4, columns])
        with pytest.raises(hc.StatusError) as refused:
            hc.prepare(CTX, hc.PagedAttention(), Q, cache, table, _strided(I32, (2, 4), strides))
        assert refused.value.code == hc.StatusCode.kUnimplemented, refused.value
        assert hc.prepare(CTX, hc.PagedAttention(), Q, cache, table, D(I32, [2, 4])).dispatch_count() >= 1
