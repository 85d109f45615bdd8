"""The rule by which attention reads pages in common apart, as far as it can be asked without a GPU."""
from types import SimpleNamespace

import pytest

from perm_amd import kvcache

DESC = SimpleNamespace(heads=8, head_dim=128, block=16)


@pytest.mark.parametrize("rows,batch,groups", [(0, 0, 0), (0, 0, 1), (0, 0, 3), (5, 0, 1), (0, 4, 1), (0, 4, 2)])
def test_a_call_without_rows_or_sequences_has_no_front(rows, batch, groups):
    assert kvcache._front_pays(DESC, rows, 16, batch, groups, 4096) is False
