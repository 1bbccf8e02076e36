"""The paged decode's page pool and refusals (no GPU)."""

from __future__ import annotations

import pytest
import torch

from uma_qmoe_amd.formats import ContractError
from uma_qmoe_amd.paged_decode import PagedDecodeGraph, PagePool


def test_pool_gives_pages_as_sequences_grow():
    pool = PagePool(6, 16, 3)
    assert pool.reserve([(0, 17), (2, 16)]) == [(0, 0, 0), (0, 1, 1), (2, 0, 2)]
    assert pool.reserve([(0, 32), (2, 16)]) == []
    assert pool.reserve([(0, 33), (1, 1)]) == [(0, 2, 3), (1, 0, 4)]
    assert pool.owned == [[0, 1, 3], [4], [2]] and pool.free == [5]


def test_pool_refuses_with_nothing_given():
    pool = PagePool(2, 32, 2)
    pool.reserve([(0, 1)])
    with pytest.raises(ContractError, match="1 free pages, 2 are needed"):
        pool.reserve([(0, 33), (1, 5)])
    assert pool.owned == [[0], []] and pool.free == [1]
    assert pool.reserve([(1, 5)]) == [(1, 0, 1)]


def test_pool_takes_pages_back():
    pool = PagePool(4, 16, 2)
    pool.reserve([(0, 40), (1, 3)])
    pool.release(0)
    pool.release(0)
    assert pool.reserve([(1, 60)]) == [(1, 1, 0), (1, 2, 1), (1, 3, 2)]
    assert pool.free == []


def test_a_model_on_the_host_is_refused():
    with pytest.raises(ContractError, match="HIP device"):
        PagedDecodeGraph(torch.nn.Linear(2, 2), batch=1, max_len=8)


def test_pool_takes_back_what_it_gave_last():
    pool = PagePool(8, 16, 2)
    pool.reserve([(0, 20), (1, 3)])
    before = ([list(o) for o in pool.owned], list(pool.free))
    given = pool.reserve([(0, 50), (1, 17)])
    assert given == [(0, 2, 3), (0, 3, 4), (1, 1, 5)]
    pool.give_back(given)
    assert (pool.owned, pool.free) == before
    pool.give_back([])
    assert (pool.owned, pool.free) == before
