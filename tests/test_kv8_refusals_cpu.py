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


def test_c_refuses_unaligned_words(built_lib):
    """Lengths, counts, lists, scores and the status word at addresses that a 32-bit access would fault on."""
    import ctypes as C
    from mserve_b200 import _lib
    from test_kv8_cpu import _append, _attn, _score
    lib = _lib.lib()
    for make, fn, names in ((_append, lib.mskv_kv8_append, ("tok0", "counts", "status")),
                            (_score, lib.mskv_kv8_block_score, ("lens", "scores", "status")),
                            (_attn, lib.mskv_kv8_attention, ("lens", "blocks", "counts", "status"))):
        for name in names:
            for off in (1, 2, 3):
                d = make()
                setattr(d, name, (20 << 20) + off)
                assert fn(C.byref(d), None) == _lib.MSKV_ERR_ARG, (fn, name)
                assert b"aligned" in lib.mskv_last_error()


def test_expanded_outputs(ext):  # noqa: F811
    """Outputs whose elements share memory: several blocks would write them at once."""
    from mserve_b200 import ops
    pages, table = ops.kv8_pages(4, 2, 128, device="cpu"), torch.zeros(3, 5, dtype=torch.int32)
    append, score, attend = _calls(pages, table, B=3)
    one = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    for out in (one.expand(3, 6, 1, 128), torch.zeros(3, 1, 1, 128, dtype=torch.bfloat16).expand(3, 6, 1, 128),
                torch.zeros(1, 6, 1, 128, dtype=torch.bfloat16).expand(3, 6, 1, 128)):
        with pytest.raises(ValueError, match="expanded"):
            attend(out=out)
    with pytest.raises(ValueError, match="must"):
        score(out=torch.zeros(1, 1, 4).expand(3, 2, 4))
    with pytest.raises(ValueError, match="expanded"):
        append(pages=pages._replace(k=pages.k[:1].expand(4, 2, 16, 128), v=pages.v[:1].expand(4, 2, 16, 128)))
