"""The operators for several answers at the edges of what their calls allow."""
import pytest
import torch

from test_gpu_kvcache import _i32, kv  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [4, 8])
def test_slopes_that_want_a_gradient(kv, heads):  # noqa: F811
    """Attention depends on its slopes: a backward pass to them alone raises, of results and log-sums."""
    c = kv.new(4, 2, 64, 16)
    t, n = _i32([[0], [1], [2]]), _i32([16] * 3)
    q = torch.ones((3, heads, 64), dtype=torch.bfloat16, device="cuda")
    slopes = torch.ones(heads, device="cuda").requires_grad_()
    plain = kv.attention(q, c, t, n, slopes=slopes.detach(), return_lse=True)
    for want, got in zip(plain, kv.attention(q, c, t, n, slopes=slopes, return_lse=True)):
        assert not want.requires_grad and got.requires_grad and torch.equal(want, got)
        with pytest.raises(NotImplementedError, match="attention"):
            got.float().sum().backward()
    with torch.no_grad():
        assert not kv.attention(q, c, t, n, slopes=slopes).requires_grad


@pytest.mark.parametrize("rows", [0, 3])
@pytest.mark.parametrize("apart", [None, True], ids=["rule", "apart"])
def test_common_pages_of_an_empty_batch(kv, monkeypatch, apart, rows):  # noqa: F811
    """A step without sequences, of any number of groups: what the call without common pages gives."""
    if apart:
        monkeypatch.setattr(kv, "_front_pays", lambda *a: True)
    c = kv.new(4, 2, 64, 16)
    q = torch.ones((rows, 8, 64), dtype=torch.bfloat16, device="cuda")
    table, lens = torch.empty((0, 5), dtype=torch.int32, device="cuda"), _i32([])
    for offsets in (_i32([0]), None) if rows == 0 else (_i32([0]),):
        for groups in (0, 1, 3):
            for more in (dict(), dict(softcap=5.0), dict(window=9)):
                out, lse = kv.attention(q, c, table, lens, offsets, return_lse=True, shared=_i32([1] * groups), **more)
                assert out.shape == q.shape and not out.any() and lse.shape == (rows, 8) and torch.isneginf(lse).all()
    # sequences, but no rows of theirs
    out = kv.attention(q[:0], c, _i32([[0], [1]]), _i32([9, 9]), _i32([0, 0, 0]), shared=_i32([1]))
    assert out.shape == (0, 8, 64)
    with pytest.raises(ValueError, match="groups"):
        kv.attention(q[:0], c, _i32([[0], [1]]), _i32([9, 9]), _i32([0, 0, 0]), shared=_i32([]))


@pytest.mark.parametrize("pages", [1, 2, 3, 2000])
@pytest.mark.parametrize("width", [1, 5])
def test_compaction_under_a_table_of_no_rows(pages, width):
    """Holders that no table names (another's, or none): pages in use move all the same."""
    from perm_amd import kvpages
    table = torch.empty((0, width), dtype=torch.int32, device="cuda")
    for held in ([], [pages - 1], list(range(0, pages, 2))):
        refs = kvpages.new(pages)
        refs[held] = 1
        src, dst, used = kvpages.compact(refs, table)
        n = len(held)
        assert used.tolist() == [n] and refs.tolist() == [1] * n + [0] * (pages - n)
        moved, free = [p for p in held if p >= n], [p for p in range(n) if p not in held]
        assert src.tolist() == moved + [-1] * (pages // 2 - len(moved))
        assert dst.tolist() == free + [-1] * (pages // 2 - len(moved))
