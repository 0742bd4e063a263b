"""PagedKV8: decode steps over an 8-bit cache against the 64-bit oracle, captured and eager, whole and selected."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as k8
from test_kv8_gpu import _bits, _close, _host

pytestmark = pytest.mark.gpu


def _steps(eng, g, plan, dtype, Q=1, oracle=True):
    """Runs the plan's steps (tokens per sequence), checking every layer of every step against the oracle's cache."""
    from mserve_b200 import ops
    empty = [_host(ops.kv8_pages(eng.num_pages, eng.Hkv, eng.D, page_size=eng.page_size, dtype=eng.pages[0].k.dtype,
                                 bounds=True)) for _ in range(eng.L)]
    for n_new in plan:
        before = eng.len_h.copy()
        eng.begin_step(n_new)
        n = max(n_new)
        for layer in range(eng.L):
            k = torch.randn(eng.B, eng.Hkv, n, eng.D, generator=g).to(dtype)
            v = torch.randn(eng.B, eng.Hkv, n, eng.D, generator=g).to(dtype)
            q = torch.randn(eng.B, eng.Hq, Q, eng.D, generator=g).to(dtype)
            out = eng.step_layer(layer, q.cuda(), k.cuda(), v.cuda())
            table = torch.from_numpy(eng.page_table_h)
            empty[layer] = k8.append(empty[layer], table, k.double(), v.double(), before, n_new, eng.pages[0].k.dtype)
            blocks = counts = None
            if eng.top_blocks:
                blocks, counts = eng._idx.view(eng.B, eng.Hkv, -1).cpu(), eng._counts.view(eng.B, eng.Hkv).cpu()
                held = -(-eng.len_h // eng.page_size)
                for b in range(eng.B):
                    assert (counts[b] == min(eng.top_blocks, max(held[b] - eng.recent_blocks, 0))
                            + min(eng.recent_blocks, held[b])).all()
            want, bound = k8.attention(q.double(), empty[layer], table, eng.len_h, blocks=blocks, counts=counts,
                                       weight_bits=_bits(dtype))
            _close(out, want, bound)
    ops.check_status(eng.device)


@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("top", [0, 3])
def test_steps(built_lib, cache, top):
    from mserve_b200.kv8_cache import PagedKV8
    g = torch.Generator().manual_seed(top)
    eng = PagedKV8(2, 3, 14, 2, 128, 300, top_blocks=top, recent_blocks=2 if top else 1, cache_dtype=cache)
    _steps(eng, g, [[100, 17, 0], [1, 1, 1], [1, 0, 1], [5, 130, 20], [1, 1, 1]], torch.bfloat16)


def test_steps_of_several_positions(built_lib):
    from mserve_b200.kv8_cache import PagedKV8
    g = torch.Generator().manual_seed(9)
    eng = PagedKV8(1, 2, 8, 2, 64, 200, top_blocks=2, recent_blocks=2, page_size=32)
    _steps(eng, g, [[90, 3], [4, 4], [4, 4]], torch.float16, Q=4)


def test_captured_step_grows(built_lib):
    """A step captured once and replayed after begin_step: the same bits as eager steps on another cache."""
    from mserve_b200 import ops
    from mserve_b200.kv8_cache import PagedKV8
    g = torch.Generator().manual_seed(4)
    for top in (0, 4):
        engs = [PagedKV8(2, 2, 14, 2, 128, 700, top_blocks=top, recent_blocks=1) for _ in range(2)]
        prompt = torch.randn(2, 2, 2, 2, 600, 128, generator=g).to(torch.bfloat16).cuda()
        for eng in engs:
            eng.begin_step([600, 333])
            for layer in range(2):
                eng.append_layer(layer, prompt[layer, 0], prompt[layer, 1])
        q = torch.zeros(2, 2, 14, 128, dtype=torch.bfloat16, device="cuda")
        kv = torch.zeros(2, 2, 2, 2, 1, 128, dtype=torch.bfloat16, device="cuda")
        out = torch.zeros(2, 2, 14, 1, 128, dtype=torch.bfloat16, device="cuda")

        def step(eng, out):
            for layer in range(2):
                eng.step_layer(layer, q[layer], kv[layer, 0], kv[layer, 1], out=out[layer])

        graph = None
        for i in range(40):
            q.copy_(torch.randn(q.shape, generator=g))
            kv.copy_(torch.randn(kv.shape, generator=g))
            engs[0].begin_step()
            want = torch.zeros_like(out)
            step(engs[0], want)
            engs[1].begin_step()
            if graph is None:
                step(engs[1], out)              # warm-up; appending the same token again changes nothing
                graph = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    step(engs[1], out)
            graph.replay()
            assert torch.equal(out, want), i
        ops.check_status(engs[0].device)
        del graph


def test_reset_and_limits(built_lib):
    from mserve_b200 import ops
    from mserve_b200.kv8_cache import PagedKV8
    g = torch.Generator().manual_seed(6)
    eng = PagedKV8(1, 2, 4, 2, 64, 64)
    x = torch.randn(2, 2, 64, 64, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(2, 4, 64, generator=g).to(torch.bfloat16).cuda()
    eng.begin_step([64, 40])
    eng.append_layer(0, x, x)
    with pytest.raises(ValueError, match="capacity"):
        eng.begin_step([1, 0])
    with pytest.raises(ValueError, match="negative"):
        eng.begin_step([-1, 0])
    first = eng.decode_layer(0, q)
    eng.reset(0)
    out = eng.decode_layer(0, q)
    assert (out[0] == 0).all() and torch.equal(out[1], first[1])
    eng.begin_step([10, 0])
    with pytest.raises(ValueError, match="appends up to 10"):
        eng.append_layer(0, x[:, :, :9], x[:, :, :9])
    eng.append_layer(0, x[:, :, :10], x[:, :, :10])
    out = eng.decode_layer(0, q)
    assert torch.equal(out[1], first[1])
    fresh = PagedKV8(1, 2, 4, 2, 64, 64)
    fresh.begin_step([10, 40])
    fresh.append_layer(0, x, x)
    assert torch.equal(fresh.decode_layer(0, q), out)
    assert sorted(eng._free + eng.page_table_h[eng.page_table_h >= 0].tolist()) == list(range(eng.num_pages))
    ops.check_status(eng.device)
    for kw in (dict(q_heads=5), dict(capacity=0), dict(top_blocks=-1), dict(top_blocks=2, recent_blocks=0), dict(batch=0)):
        with pytest.raises(ValueError):
            PagedKV8(**{**dict(num_layers=1, batch=2, q_heads=4, kv_heads=2, head_dim=64, capacity=64), **kw})
