"""Further refusals of the 8-bit cache's wrappers, without a GPU."""
from types import SimpleNamespace

import pytest
import torch

from test_kv8_cpu import _calls, ext  # noqa: F401


def test_streams_of_another_device(ext, monkeypatch):  # noqa: F811
    """A stream of another device than the tensors': the call would run on some other stream than the one given."""
    from mserve_b200 import ops
    entered = []
    monkeypatch.setattr(torch.cuda, "stream", lambda s: entered.append(s))
    pages, table = ops.kv8_pages(4, 2, 128, device="cpu"), torch.zeros(1, 5, dtype=torch.int32)
    for call in _calls(pages, table):
        with pytest.raises(ValueError, match="stream of cuda:1"):
            call(stream=SimpleNamespace(device=torch.device("cuda", 1)))
    assert not entered
