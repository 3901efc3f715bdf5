"""The page bookkeeping of the serving example, without a GPU."""
import pytest

from npu_amd.serving import Pages


def test_pages_grow_by_need_and_are_given_back():
    p = Pages(pages=5, page=16, slots=2, max_pages=3)
    assert [at for at, _ in p.grow(0, 1)] == [0] and p.grow(0, 16) == []
    assert [at for at, _ in p.grow(0, 33)] == [1, 2]
    assert [at for at, _ in p.grow(1, 17)] == [0, 1]
    assert sorted(p.owned[0] + p.owned[1]) == list(range(5)) and not p.free
    with pytest.raises(RuntimeError, match="table holds 3"):
        p.grow(0, 49)
    with pytest.raises(RuntimeError, match="0 free pages, 1 are needed"):
        p.grow(1, 33)
    assert len(p.owned[1]) == 2
    p.release(0)
    assert len(p.free) == 3 and p.owned[0] == []
    assert [at for at, _ in p.grow(1, 48)] == [2]
