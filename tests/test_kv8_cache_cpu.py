"""PagedKV8's host side without a GPU: the calls that a step makes, on stand-ins for the operators."""
import contextlib

import pytest
import torch


@pytest.fixture
def engine(monkeypatch, built_lib):
    """make(...): a PagedKV8 on CPU tensors whose operator calls are recorded in make.calls as (name, device that is
    current, arguments)."""
    from mserve_b200 import kv8_cache, ops
    calls, current, pinned, capturing = [], [None], [], [False]

    @contextlib.contextmanager
    def on(device):
        was, current[0] = current[0], device
        yield
        current[0] = was

    def record(name, result=None):
        def call(*args, **kw):
            calls.append((name, current[0], args, kw))
            return result(*args, **kw) if result else None
        return call

    def topk(scores, *, top_k, recent=0, out=None, counts=None, **kw):
        n = scores.shape[0]
        return (torch.zeros(n, top_k + recent, dtype=torch.int32) if out is None else out,
                torch.zeros(n, dtype=torch.int32) if counts is None else counts)

    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t, *a: pinned.append(t) or t)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(ops, "kv8_append", record("append"))
    monkeypatch.setattr(ops, "kv8_block_score", record("score"))
    monkeypatch.setattr(ops, "topk", record("topk", topk))
    monkeypatch.setattr(ops, "kv8_attention", record("attention", lambda q, *a, **kw: torch.zeros_like(q)))

    def make(*args, **kw):
        return kv8_cache.PagedKV8(*args, device=torch.device("cpu"), **kw)
    make.calls, make.pinned, make.capturing = calls, pinned, capturing
    return make


def test_selection_runs_on_the_caches_device(engine):
    """The top-k call, which launches on the current device, is made with the cache's device current."""
    eng = engine(1, 2, 4, 2, 64, 100, top_blocks=2)
    eng.device = torch.device("cpu", 3)
    eng.decode_layer(0, torch.zeros(2, 4, 64, dtype=torch.bfloat16))
    assert [c[0] for c in engine.calls] == ["score", "topk", "attention"]
    assert engine.calls[1][1] == eng.device.index == 3


@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("recent", [1, 2, 5])
def test_recent_window_holds_the_positions_own_pages(engine, page, recent):
    """Whatever the length: the pages of the last Q tokens are among the last pages that the selection always takes."""
    eng = engine(1, 2, 4, 2, 64, 1000, top_blocks=3, recent_blocks=recent, page_size=page)
    for Q in (1, 2, 3, 4, 15, 16):
        engine.calls.clear()
        q = torch.zeros(2, 4, Q, 64, dtype=torch.bfloat16)
        eng.decode_layer(0, q)
        window = next(c[3]["recent"] for c in engine.calls if c[0] == "topk")
        assert window >= recent and (Q > 1 or window == recent)
        for n in range(Q, 3 * page + 20):
            assert (n - 1) // page - (n - Q) // page < window, (Q, n)
        assert window == recent or any((n - 1) // page - (n - Q) // page == window - 1 for n in range(Q, 3 * page)), "wider than needed"
    engine.calls.clear()
    eng.decode_layer(0, torch.zeros(2, 4, 64, dtype=torch.bfloat16))
    assert next(c[3]["recent"] for c in engine.calls if c[0] == "topk") == recent


def test_selections_share_nothing(engine):
    """Scores, indices and counts of two selections, of one layer or two, are memory of their own."""
    eng = engine(2, 2, 4, 2, 64, 1000, top_blocks=3)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    held = [eng.select(layer, q) for layer in (0, 1, 0)]
    scores = [c[3]["out"] for c in engine.calls if c[0] == "score"]
    for tensors in (scores, [s[0] for s in held], [s[1] for s in held]):
        assert len({t.data_ptr() for t in tensors}) == 3
    assert [c[2][0].data_ptr() for c in engine.calls if c[0] == "topk"] == [t.data_ptr() for t in scores]
    assert held[0][0].shape == (2, 2, 4) and held[0][1].shape == (2, 2)


def test_staging_is_of_each_send(engine):
    """Every send stages through memory of its own that nothing writes again: earlier copies may still be under way."""
    eng = engine(1, 2, 4, 2, 64, 1000)
    engine.pinned.clear()
    eng.begin_step([17, 3])
    eng.begin_step([0, 2])
    eng.reset(0)
    eng.begin_step(1)
    states = [t for t in engine.pinned if t.shape == (4, 2)]
    tables = [t for t in engine.pinned if t.shape == (2, 63)]
    assert len({t.data_ptr() for t in engine.pinned}) == len(engine.pinned) == len(states) + len(tables)
    assert [s.tolist() for s in states] == [[[0, 0], [17, 3], [17, 3], [2, 1]], [[17, 3], [0, 2], [17, 5], [2, 1]],
                                            [[0, 5], [0, 0], [0, 5], [0, 1]], [[0, 5], [1, 1], [1, 6], [1, 1]]]
    assert [(t >= 0).sum(dim=1).tolist() for t in tables] == [[2, 1], [0, 1], [1, 1]]
    assert eng.page_table.tolist() == eng.page_table_h.tolist()


def test_steps_are_not_captured(engine):
    eng = engine(1, 2, 4, 2, 64, 1000)
    eng.begin_step([17, 3])
    engine.capturing[0] = True
    for call in (eng.begin_step, lambda: eng.reset(1)):
        with pytest.raises(RuntimeError, match="captur"):
            call()
    engine.capturing[0] = False
    assert eng.len_h.tolist() == [17, 3] and eng.page_table_h[1, 0] >= 0
    eng.append_layer(0, torch.zeros(2, 2, 17, 64), torch.zeros(2, 2, 17, 64))
    with pytest.raises(ValueError, match="up to 17"):
        eng.append_layer(0, torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 16, 64))


@pytest.mark.parametrize("top", [0, 2])
def test_t_bound_covers_the_lengths(engine, top):
    """A bound below a sequence's length would leave tokens out, and shift what each position sees: refused."""
    eng = engine(1, 2, 4, 2, 64, 100, top_blocks=top)
    eng.begin_step([40, 7])
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16)
    for bad in (39, 0, -1, 101, 112):
        with pytest.raises(ValueError, match="t_bound"):
            eng.decode_layer(0, q, t_bound=bad)
    assert not engine.calls
    for good in (40, 77, 100, None):
        eng.decode_layer(0, q, t_bound=good)
    if not top:
        assert [c[3]["max_tokens"] for c in engine.calls] == [40, 77, 100, 100]


def test_arguments(engine):
    """Sizes that no cache has are refused as such, token counts that are no integers too: nothing is rounded or divided by."""
    make = dict(num_layers=1, batch=2, q_heads=4, kv_heads=2, head_dim=64, capacity=64)
    for kw in (dict(page_size=0), dict(page_size=-16), dict(page_size=24), dict(head_dim=96), dict(num_layers=0)):
        with pytest.raises(ValueError, match="page_size|head_dim|num_layers"):
            engine(**{**make, **kw})
    with pytest.raises(TypeError):
        engine(**make, cache_dtype=torch.float16)
    eng = engine(**make)
    for bad in (1.5, [1.0, 2.0], [1, 2, 3], [[1, 1]], [3], "1"):
        with pytest.raises(ValueError, match="n_new"):
            eng.begin_step(bad)
    assert eng.len_h.tolist() == [0, 0] and (eng.page_table_h < 0).all()
    for good in (3, [1, 0], (0, 2), torch.tensor([2, 2]), torch.tensor(1)):
        eng.begin_step(good)
    assert eng.len_h.tolist() == [7, 8]


@pytest.mark.parametrize("top", [0, 2])
def test_queries_of_another_model(engine, top):
    """Query heads that are not the cache's would be grouped otherwise without a word."""
    eng = engine(1, 2, 4, 2, 64, 100, top_blocks=top)
    eng.begin_step(5)
    for shape in ((2, 8, 64), (2, 2, 1, 64), (1, 4, 64), (2, 4, 32), (2, 4), (2, 4, 1, 1, 64)):
        with pytest.raises(ValueError, match="Hq=4"):
            eng.decode_layer(0, torch.zeros(shape, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="Hq=4"):
            eng.select(0, torch.zeros(shape, dtype=torch.bfloat16))
    assert not engine.calls
