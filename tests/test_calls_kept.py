"""Calls of the 16-bit paths that took more than the package's own records and integers keep doing so (no GPU needed)."""

import numpy
import pytest
import torch

import streamattn_b200 as sa


def paged_fields(**over):
    fields = dict(key=torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16), value=torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16),
                  page_table=torch.arange(6, dtype=torch.int32).view(2, 3), sequence_lengths=torch.tensor([5, 40], dtype=torch.int32))
    return {**fields, **over}


Q = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)


class Lookalike:
    """Not a PagedKVCache: another package's record with the same fields and checks."""

    def __init__(self, record):
        self.record, self.validated = record, 0

    def __getattr__(self, name):
        return getattr(self.record, name)

    def validate(self, query, *, validate_metadata=True):
        self.validated += 1
        self.record.validate(query, validate_metadata=validate_metadata)


def test_exact_plans_take_any_record_with_the_fields_of_a_paged_cache():
    cache = Lookalike(sa.PagedKVCache(**paged_fields()))
    with pytest.raises(RuntimeError, match="no CPU fallback"):             # every check is passed; there is no GPU here
        sa.PagedExactDecodePlan.build(Q, cache)
    assert cache.validated == 1
    with pytest.raises(ValueError, match="multiple of KV heads"):          # and the record's own checks decide
        sa.PagedExactDecodePlan.build(Q[:, :, :3], cache)


@pytest.mark.parametrize("one", [numpy.int64(1), numpy.int32(1), torch.tensor(1), True], ids=["int64", "int32", "tensor", "bool"])
def test_pages_are_reserved_for_any_whole_number(one):
    cache = sa.PagedKVCache(**paged_fields(sequence_lengths=torch.tensor([16, 31], dtype=torch.int32)))
    writer = sa.PagedKVWriter.attach(cache)
    assert writer.reserve(one) == 1                                        # row 0 starts a page, row 1 does not
    assert writer.pages == [[0, 1], [3, 4]]
    assert writer.reserve(17 * one) == 2 and [len(p) for p in writer.pages] == [3, 3]
    assert writer.reserve(-one) == 0                                       # nothing to do, as ever
    assert writer.lengths == [16, 31]


def test_pages_are_reserved_for_a_number_each():
    cache = sa.PagedKVCache(**paged_fields(sequence_lengths=torch.tensor([16, 31], dtype=torch.int32)))
    for each in ([0, 2], (0, 2), numpy.array([0, 2]), torch.tensor([0, 2])):
        writer = sa.PagedKVWriter.attach(cache)
        assert writer.reserve(each) == 1 and [len(p) for p in writer.pages] == [1, 3]
    for bad in ([1], [1, 2, 3], [-1, 2], [[1, 2]], ["x", 1], 1.5, None):
        with pytest.raises((ValueError, TypeError)):
            writer.reserve(bad)
    assert [len(p) for p in writer.pages] == [1, 3]
