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


def test_selections_are_the_callers_own(built_lib):
    """A later selection, of another layer, another query or on another stream at the same time, leaves an earlier one as it is."""
    from mserve_b200 import ops
    from mserve_b200.kv8_cache import PagedKV8
    B, Hq, H, D, layers = 2, 8, 2, 128, 4
    g = torch.Generator().manual_seed(3)
    eng = PagedKV8(layers, B, Hq, H, D, 2000, top_blocks=5)
    eng.begin_step([2000, 700])
    for layer in range(layers):
        k, v = (torch.randn(B, H, 2000, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        eng.append_layer(layer, k, v)
    qs = torch.randn(layers, B, Hq, D, generator=g).to(torch.bfloat16).cuda()
    want = [[t.clone() for t in eng.select(layer, qs[layer])] for layer in range(layers)]
    assert not torch.equal(want[0][0], want[1][0])
    held = [eng.select(layer, qs[layer]) for layer in range(layers)]
    eng.select(0, qs[1])
    for a, b in zip(held, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    streams = [torch.cuda.Stream() for _ in range(layers)]
    torch.cuda.synchronize()
    both = []
    for _ in range(10):
        for layer, st in enumerate(streams):
            with torch.cuda.stream(st):
                both.append((layer, eng.select(layer, qs[layer])))
    torch.cuda.synchronize()
    for layer, (idx, counts) in both:
        assert torch.equal(idx, want[layer][0]) and torch.equal(counts, want[layer][1])
    ops.check_status(eng.device)


def test_steps_do_not_wait_for_the_device(built_lib):
    """reset and begin_step return while earlier work of the stream still runs, and each sends its own lengths."""
    from mserve_b200 import ops
    from mserve_b200.kv8_cache import PagedKV8
    eng = PagedKV8(1, 3, 4, 2, 64, 100)
    for _ in range(6):                              # the staging memory exists
        eng.begin_step(1)
        eng.reset(0)
    eng.reset(1), eng.reset(2)
    torch.cuda.synchronize()
    torch.cuda._sleep(800_000_000)                  # four tenths of a second
    busy = torch.cuda.Event()
    busy.record()
    eng.begin_step([20, 5, 0])
    seen = [(eng.lens.clone(), eng.tok0.clone(), eng.held.clone(), eng.page_table.clone(), eng.page_table_h.copy())]
    for call in (lambda: eng.begin_step(1), lambda: eng.reset(0), lambda: eng.begin_step([40, 0, 1])):
        call()
        seen.append((eng.lens.clone(), eng.tok0.clone(), eng.held.clone(), eng.page_table.clone(), eng.page_table_h.copy()))
    assert not busy.query(), "a call waited for the stream"
    torch.cuda.synchronize()
    assert [s[0].tolist() for s in seen] == [[20, 5, 0], [21, 6, 1], [0, 6, 1], [40, 6, 2]]
    assert [s[1].tolist() for s in seen] == [[0, 0, 0], [20, 5, 0], [0, 6, 1], [0, 6, 1]]
    assert [s[2].tolist() for s in seen] == [[2, 1, 0], [2, 1, 1], [0, 1, 1], [3, 1, 1]]
    for s in seen:
        assert s[3].tolist() == s[4].tolist()
    ops.check_status(eng.device)


def test_begin_step_in_a_capture_is_refused(built_lib):
    from mserve_b200.kv8_cache import PagedKV8
    eng = PagedKV8(1, 1, 4, 2, 64, 100)
    eng.begin_step(3)
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x += 1
        for call in (eng.begin_step, lambda: eng.reset(0)):
            with pytest.raises(RuntimeError, match="captur"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1] * 4 and eng.len_h.tolist() == [3] and eng.lens.tolist() == [3]
    del graph


def test_more_blocks_than_there_are(built_lib):
    """top_blocks beyond the pages that a sequence has, or can have: the whole cache; short and empty sequences among them."""
    from mserve_b200 import ops
    from mserve_b200.kv8_cache import PagedKV8
    g = torch.Generator().manual_seed(8)
    lens = [200, 16, 17, 1, 0]
    x = torch.randn(2, 5, 2, 200, 64, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(5, 6, 3, 64, generator=g).to(torch.bfloat16).cuda()
    outs = []
    for top, recent in ((0, 1), (1000, 1), (5, 50), (1, 12)):
        eng = PagedKV8(1, 5, 6, 2, 64, 200, top_blocks=top, recent_blocks=recent)
        eng.begin_step(lens)
        eng.append_layer(0, x[0], x[1])
        outs.append(eng.decode_layer(0, q))
        if top:
            counts = eng.select(0, q)[1].cpu()
            assert counts.tolist() == [[min(-(-n // 16), top + max(recent, 2))] * 2 for n in lens]
    # the same tokens in the same order, split otherwise: the sums' rounding, then the output's
    whole = outs[0].double()
    for out in outs[1:]:
        assert ((out.double() - whole).abs() <= 2.0 ** -7 * whole.abs() + 2.0 ** -10).all()
    assert (whole[4] == 0).all() and (whole[3, :, :2] == 0).all()
    ops.check_status(torch.device("cuda"))
