"""PagedKV8's selection of pages: several positions across a page's border."""
import pytest
import torch

from oracle import kv8_oracle as k8
from test_kv8_gpu import _bits, _close, _host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,lens,Q", [(16, [65, 49], 4), (16, [16, 33], 2), (16, [79, 200], 16), (32, [33, 95], 5),
                                         (16, [3, 64], 4)])
def test_positions_attend_to_themselves(built_lib, page, lens, Q):
    """One best page and one last page asked for: the lists hold every position's own page, and the result is the
    attention over them."""
    from mserve_b200 import ops
    from mserve_b200.kv8_cache import PagedKV8
    B, Hq, H, D = len(lens), 6, 2, 64
    g = torch.Generator().manual_seed(page + Q)
    eng = PagedKV8(1, B, Hq, H, D, 256, top_blocks=1, recent_blocks=1, page_size=page)
    host = _host(ops.kv8_pages(eng.num_pages, H, D, page_size=page))
    before = [0] * B
    for n_new in ([max(n - Q, 0) for n in lens], [n - max(n - Q, 0) for n in lens]):
        k, v = (torch.randn(B, H, max(n_new), D, generator=g).to(torch.bfloat16) for _ in range(2))
        # keys of the early pages are large, so that the one best page is not the positions' own
        if before == [0] * B:
            k[:, :, :page] *= 30
        eng.begin_step(n_new)
        eng.append_layer(0, k.cuda(), v.cuda())
        host = k8.append(host, torch.from_numpy(eng.page_table_h), k.double(), v.double(), before, n_new, torch.float8_e4m3fn)
        before = [a + b for a, b in zip(before, n_new)]
    q = torch.randn(B, Hq, Q, D, generator=g).to(torch.bfloat16)
    idx, counts = (t.cpu() for t in eng.select(0, q.cuda()))
    for b in range(B):
        own = {t // page for t in range(max(lens[b] - Q, 0), lens[b])}
        for h in range(H):
            listed = idx[b, h, :int(counts[b, h])].tolist()
            assert own <= set(listed) and len(set(listed)) == len(listed) and listed == sorted(listed), (b, h, listed, own)
    out = eng.decode_layer(0, q.cuda())
    want, bound = k8.attention(q.double(), host, torch.from_numpy(eng.page_table_h), lens, blocks=idx, counts=counts,
                               weight_bits=_bits(torch.bfloat16))
    _close(out, want, bound)
    ops.check_status(eng.device)
