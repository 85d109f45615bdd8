"""Tensors of another device than the current one are refused before anything runs on its stream."""
from types import SimpleNamespace

import pytest
import torch

from perm_amd import _lib, kvcache, kvpages


class On(torch.Tensor):
    """A tensor of device ``at`` as far as the checks ask."""

    at = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.at))

    def get_device(self):
        return self.at


def _on(shape, dtype, at=0):
    t = torch.zeros(shape, dtype=dtype).as_subclass(On)
    t.at = at
    return t


I32, B = torch.int32, torch.bfloat16
ARGS = ("k", "v", "k_scale", "v_scale", "rows", "table", "lens", "offsets")


def _args(elsewhere):
    at = {n: int(n == elsewhere) for n in ARGS}
    cache = kvcache.KvCache(_on((4, 2, 16, 64), torch.uint8, at["k"]), _on((4, 2, 64, 16), torch.uint8, at["v"]),
                            _on((4, 2), torch.float32, at["k_scale"]), _on((4, 2), torch.float32, at["v_scale"]))
    return (cache, _on((3, 2, 64), B, at["rows"]), _on((3, 5), I32, at["table"]), _on((3,), I32, at["lens"]),
            _on((4,), I32, at["offsets"]))


@pytest.fixture(autouse=True)
def _no_gpu(monkeypatch):
    """One device, number 0, and a library that nothing may be launched of."""
    monkeypatch.setattr(_lib, "load", lambda *a: SimpleNamespace())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


@pytest.mark.parametrize("elsewhere", ARGS)
def test_cache_calls(elsewhere):
    cache, rows, table, lens, offsets = _args(elsewhere)
    calls = {"write": lambda: kvcache.write(cache, rows, rows, table, lens, offsets),
             "attention": lambda: kvcache.attention(rows, cache, table, lens, offsets),
             "more": lambda: kvcache.attention(rows, cache, table, lens, offsets, softcap=3.0)}
    if elsewhere not in ("rows", "lens"):
        calls["read"] = lambda: kvcache.read(cache, table, offsets, 3)
    for name, call in calls.items():
        with pytest.raises(ValueError, match="current device|buffers"):
            call()
            pytest.fail(name)


@pytest.mark.parametrize("elsewhere", ARGS[:4])
@pytest.mark.parametrize("into", [False, True])
def test_page_copies(elsewhere, into):
    bad, fine = _args(elsewhere)[0], _args(None)[0]
    pages = _on((2,), I32)
    with pytest.raises(ValueError, match="current device|buffers"):
        kvpages.copy(fine if into else bad, pages, pages, into=bad if into else None)


def test_here():
    _lib.here(_on((1,), I32), None, _on((1,), I32))
    with pytest.raises(ValueError, match="cuda:1, but the current device is cuda:0"):
        _lib.here(_on((1,), I32), None, _on((1,), I32, 1))
